"""Which arithmetic the 4-bit formats mean, on stand-ins for the kernels: the place (prefill or decode step) decides, not the number of rows."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import mx_ref  # noqa: E402
from test_engine_cpu import _model  # noqa: E402
from test_mxfp4_model_cpu import install, snap  # noqa: E402

BF16 = torch.bfloat16


def installed(monkeypatch):
    """The stand-ins, with the streaming product's refusal and its `out`; returns the calls made."""
    from hvlm import ops
    calls = install(monkeypatch)
    plain = ops.gemm_w4a16_nt

    def gemm_w4a16_nt(a, b4, residual=None, out=None):
        assert a.shape[0] <= 32
        y = plain(a, b4, residual=residual)
        return y if out is None else out.copy_(y)

    monkeypatch.setattr(ops, "gemm_w4a16_nt", gemm_w4a16_nt)
    return calls


@pytest.mark.parametrize("B", [1, 32, 33, 70])
def test_decode_steps_keep_their_activations(monkeypatch, B):
    calls = installed(monkeypatch)
    st = _model().stack
    snap(st)
    g = torch.Generator().manual_seed(B)
    x = torch.randn(B, st.D, generator=g).to(BF16)
    lens = torch.arange(B, dtype=torch.int32) % 5
    st.mxfp4_prepare()
    outs = []
    for kw in (dict(), dict(mxfp4=True)):
        cache = [torch.randn(B, 6, 3 * st.D, generator=torch.Generator().manual_seed(i)).to(BF16) for i in range(st.L)]
        del calls[:]
        outs.append(st.decode_step_batched(x, lens, cache, **kw).double())
    assert calls == ["stream"] * (4 * st.L * ((B + 31) // 32))
    # on weights that the format holds exactly, a step is the bf16 step but for the order of sums: nine roundings to bf16 a layer and the last norm's
    assert (outs[0] - outs[1]).norm() <= (9 * st.L + 1) * 2.0 ** -8 * outs[0].norm()


@pytest.mark.parametrize("B,S", [(1, 1), (1, 20), (2, 16), (3, 20)])
def test_prefill_quantises_its_activations(monkeypatch, B, S):
    calls = installed(monkeypatch)
    st = _model().stack
    st.mxfp4_prepare()
    del calls[:]
    x = torch.randn(S, st.D, generator=torch.Generator().manual_seed(S)).to(BF16)
    got = st.forward(x.repeat(B, 1), B, S, save=False, mxfp4=True).double()
    assert calls == ["quantize", "gemm"] * (4 * st.L)
    alone = st.forward(x, 1, S, save=False, mxfp4=True).double().repeat(B, 1)
    assert (got - alone).norm() <= (9 * st.L + 1) * 2.0 ** -8 * alone.norm()


def test_one_batched_cache_is_kept(monkeypatch):
    """The cache of the other format, and what was captured on it, does not stay beside the new one."""
    import gc
    import weakref
    installed(monkeypatch)
    st = _model().stack
    for first in (False, True, False):
        cache = st.new_cache(8, batch=2, kv4=first)
        assert st.new_cache(6, batch=2, kv4=first) is cache
        st._dec_graphs_b = {"captured": cache}
        seen = [weakref.ref(t) for layer in cache for t in (layer if first else [layer])]
        del cache
        st.new_cache(8, batch=2, kv4=not first)
        gc.collect()
        assert "_dec_graphs_b" not in st.__dict__ and not any(r() is not None for r in seen)
