"""The 4-bit formats through the model, on stand-ins for the kernels: generation with MXFP4 weights and cache, the evaluation's flags, refusals."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import cpu_ops  # noqa: E402
import mx_ref  # noqa: E402
from test_engine_cpu import _model  # noqa: E402

BF16 = torch.bfloat16


def install(monkeypatch):
    """Stand-ins for every operator the model calls, the 4-bit ones from their definition; returns the calls made of those."""
    from hvlm import ops
    cpu_ops.install(monkeypatch)
    calls = []

    def quantize_mxfp4(x):
        calls.append("quantize")
        return mx_ref.quantise(x)

    def product(name):
        def run(a, b4, residual=None):
            calls.append(name)
            a = mx_ref.values(a) if isinstance(a, tuple) else a.double()
            y = a @ mx_ref.values(b4).t()
            return (y if residual is None else y + residual.double()).to(BF16)
        return run

    def kv4_append(qkv, cache, start, H):
        calls.append("append")
        B, Hkv, n, dh = cache.checked("kv4_append")
        rows = qkv.view(B, -1, 3 * H * dh)
        for b in range(B):
            at = 0 if start is None else int(start[b])
            for col, codes, scales in ((1, cache.k, cache.k_scale), (2, cache.v, cache.v_scale)):
                for s in range(rows.shape[1]):
                    c, e = mx_ref.quantise(rows[b, s, col * H * dh:(col + 1) * H * dh].reshape(H, dh))
                    codes[b, :, at + s], scales[b, :, at + s] = c, e

    def attn_decode_kv4(q, cache, lens, H, scale):
        calls.append("attention")
        out = torch.zeros(q.shape[0], H * cache.k.shape[3] * 2, dtype=torch.float64)
        for b in range(q.shape[0]):
            n = int(lens[b])
            k, v = mx_ref.values((cache.k[b, :, :n], cache.k_scale[b, :, :n])), mx_ref.values((cache.v[b, :, :n], cache.v_scale[b, :, :n]))
            p = torch.softmax(q[b, :out.shape[1]].double().view(H, 1, -1) @ k.transpose(1, 2) * scale, -1)
            out[b] = (p @ v).reshape(-1)
        return out.to(BF16)

    for name, f in (("quantize_mxfp4", quantize_mxfp4), ("gemm_mxfp4_nt", product("gemm")), ("gemm_w4a16_nt", product("stream")),
                    ("kv4_append", kv4_append), ("attn_decode_kv4", attn_decode_kv4)):
        monkeypatch.setattr(ops, name, f)
    return calls


def snap(stack):
    """Every GEMM weight to the nearest MXFP4 value (which the format then holds exactly)."""
    for lp in stack.layers:
        for k in ("qkv", "o", "gu", "down"):
            lp.w[k].copy_(mx_ref.values(mx_ref.quantise(lp.w[k])).to(BF16))
    stack.invalidate_fp8()


def test_a_snapped_weight_quantises_to_itself():
    g = torch.Generator().manual_seed(0)
    v = mx_ref.values(mx_ref.quantise(torch.randn(64, 256, generator=g)))
    assert torch.equal(mx_ref.values(mx_ref.quantise(v)), v)


def test_decode_with_4_bit_weights_and_cache(monkeypatch):
    """On weights that MXFP4 holds exactly, decode steps with 4-bit weights are those of the bf16 weights; with the 4-bit cache they are those
    of a bf16 cache holding the cache's values."""
    calls = install(monkeypatch)
    m = _model()
    st = m.stack
    snap(st)
    g = torch.Generator().manual_seed(1)
    B, n = 3, 12
    x = torch.randn(B, st.D, generator=g).to(BF16)
    lens = torch.tensor([4, 0, 11], dtype=torch.int32)
    # roundings to bf16 of one layer in which the two sides may differ by a step: norm, qkv, RoPE, attention, o, norm, gate|up, SwiGLU, down
    tol = (9 * st.L + 1) * 2.0 ** -8
    outs = []
    for kw in (dict(), dict(mxfp4=True)):
        cache = [torch.zeros(B, n, 3 * st.D, dtype=BF16) for _ in range(st.L)]
        for c in cache:
            c.copy_(torch.randn(c.shape, generator=torch.Generator().manual_seed(2)).to(BF16))
        outs.append(st.decode_step_batched(x, lens, cache, **kw).double())
    assert calls.count("stream") == 4 * st.L and "gemm" not in calls
    assert (outs[0] - outs[1]).norm() <= tol * outs[0].norm()
    from hvlm import ops
    kv = st.new_cache(n, batch=B, kv4=True)
    assert kv is st.new_cache(n - 1, batch=B, kv4=True) and isinstance(kv[0], ops.KV4Cache)
    filled = torch.randn(B * n, 3 * st.D, generator=g).to(BF16)
    for c in kv:
        ops.kv4_append(filled, c, None, st.H)
    out = st.decode_step_batched(x, lens, kv, mxfp4=True).double()
    plain = []
    for c in kv:                                                                  # what the 4-bit cache holds after the step, the new token's row included
        t = torch.zeros(B, n, 3, st.H, st.dh, dtype=BF16)
        t[:, :, 1], t[:, :, 2] = (mx_ref.values(p).to(BF16).transpose(1, 2) for p in ((c.k, c.k_scale), (c.v, c.v_scale)))
        plain.append(t.view(B, n, 3 * st.D))
    monkeypatch.setattr(ops, "kv4_append", lambda *a: None)
    monkeypatch.setattr(ops, "attn_decode_kv4", lambda q, c, le, H, s: cpu_ops.attn_decode_batched(q, plain[[id(t) for t in kv].index(id(c))], le, H, st.dh, s))
    ref = st.decode_step_batched(x, lens, kv, mxfp4=True).double()
    assert (out - ref).norm() <= tol * ref.norm()


def test_copies_go_with_the_weights(monkeypatch):
    calls = install(monkeypatch)
    m = _model()
    st = m.stack
    x = torch.randn(40, st.D, generator=torch.Generator().manual_seed(3)).to(BF16)
    a = st.forward(x, 1, 40, save=False, mxfp4=True)
    assert calls.count("gemm") == 4 * st.L and calls.count("quantize") == 8 * st.L and len(st._mxfp4_w) == st.L
    assert torch.equal(a, st.forward(x, 1, 40, save=False, mxfp4=True)) and calls.count("quantize") == 12 * st.L
    st.init_random(seed=9)
    assert st._mxfp4_w is None and not torch.equal(a, st.forward(x, 1, 40, save=False, mxfp4=True))


def test_refusals(monkeypatch):
    install(monkeypatch)
    m = _model()
    st = m.stack
    x = torch.zeros(4, st.D, dtype=BF16)
    with pytest.raises(AssertionError, match="inference"):
        st.forward(x, 1, 4, save=True, mxfp4=True)
    with pytest.raises(AssertionError, match="inference"):
        st.forward(x, 1, 4, save=False, mxfp4=True, fp8=True)
    with pytest.raises(AssertionError, match="batch"):
        st.new_cache(8, kv4=True)
    with pytest.raises(AssertionError, match="padded"):
        st.forward(x, 1, 4, save=False, cache=st.new_cache(8, batch=1, kv4=True), cu_seqlens=torch.tensor([0, 4], dtype=torch.int32), pos=torch.arange(4, dtype=torch.int32))
    with pytest.raises(AssertionError, match="not both"):
        st.decode_step_batched(x[:1], torch.zeros(1, dtype=torch.int32), st.new_cache(8, batch=1), fp8=True, mxfp4=True)
    for kw in (dict(fp8=True, mxfp4=True), dict(fp8_decode=True, mxfp4_decode=True)):
        with pytest.raises(AssertionError, match="not both"):
            m.sample_batch(torch.zeros(1, 4, dtype=torch.long), **kw)


@pytest.mark.parametrize("flags,want", [([], {}), (["--mxfp4"], dict(mxfp4=True, mxfp4_decode=True)), (["--kv4"], dict(kv4=True)),
                                        (["--fp8", "--kv4"], dict(fp8=True, fp8_decode=True, kv4=True))])
def test_evaluation_flags(monkeypatch, flags, want):
    """`python -m hvlm.evaluate` hands the formats through to model.generate_batch."""
    from types import SimpleNamespace
    from hvlm import checkpoint, evaluate
    from hvlm.model import SampleDecoderOnlyOutput
    seen = []

    class Model:
        config = SimpleNamespace(vision=SimpleNamespace(hidden_size=64, intermediate_size=256, image_size=224))

        def eval(self):
            return self

        def generate_batch(self, ids, **kw):
            seen.append(kw)
            out = SampleDecoderOnlyOutput(sequences=ids, pred_hands=torch.zeros(len(ids), 2, 4, 2))
            out.num_hands = [4] * len(ids)
            return out

    monkeypatch.setattr(checkpoint, "from_pretrained", lambda *a, **k: Model())
    sample = dict(input_ids=torch.ones(1, 4, dtype=torch.long), image=torch.zeros(1, 1), future_hands=torch.zeros(1, 2, 5, 2), future_valid=torch.ones(1, 2))
    base = ["--model-path", "none", "--device", "cpu"]
    assert evaluate.main(base + ["--batch-size", "2"] + flags, samples=[sample] * 2)["n"] == 2
    names = ("fp8", "fp8_decode", "mxfp4", "mxfp4_decode", "kv4")
    assert {n: seen[0][n] for n in names} == {n: want.get(n, False) for n in names}
    if flags:
        with pytest.raises(AssertionError, match="batched"):
            evaluate.main(base + flags, samples=[sample])
    with pytest.raises(AssertionError, match="two formats"):
        evaluate.main(base + ["--batch-size", "2", "--fp8", "--mxfp4"], samples=[sample])
