"""Decode steps of more than 32 samples and short prefills in 4 bits on the GPU: the place decides the arithmetic, not the number of rows."""
import pytest
import torch

from test_gpu_mxfp4_model import BF16, DEV, filled, model, near, plain, snap, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [33, 64, 70])
def test_decode_weights_against_the_bf16_step(B, monkeypatch):
    """On weights that MXFP4 holds exactly, a step with 4-bit weights is the bf16 step, whatever the batch; a sample's result is that of a smaller batch."""
    from hvlm import ops
    st = model().stack
    snap(st)
    n = 40
    g = torch.Generator(device=DEV).manual_seed(B)
    x = torch.randn(B, st.D, device=DEV, generator=g).to(BF16)
    lens = (torch.arange(B, dtype=torch.int32, device=DEV) * 13) % n
    cache = filled(st, B, n, 7)
    base = st._decode_step_batched_eager(x, lens, plain(st, cache))
    st.mxfp4_prepare()
    with monkeypatch.context() as mp:
        mp.setattr(ops, "quantize_mxfp4", None)                                   # (activations stay as they are)
        got = st._decode_step_batched_eager(x, lens, plain(st, cache), mxfp4=True)
        near(got, base, tolerance(st))
        on4 = st._decode_step_batched_eager(x, lens, cache, mxfp4=True)
        part = [ops.KV4Cache(*(t[29:36].contiguous() for t in c)) for c in cache]
        near(on4[29:36], st._decode_step_batched_eager(x[29:36].contiguous(), lens[29:36].contiguous(), part, mxfp4=True), tolerance(st))
        assert torch.equal(st.decode_step_batched(x, lens, cache, mxfp4=True), on4)


@pytest.mark.parametrize("S", [1, 5, 32])
def test_a_short_prompt_is_prefilled_as_in_a_batch(S):
    st = model().stack
    x = torch.randn(S, st.D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(S)).to(BF16)
    alone = st.forward(x, 1, S, save=False, mxfp4=True)
    many = st.forward(x.repeat(40, 1), 40, S, save=False, mxfp4=True)
    for b in (0, 17, 39):
        near(many[b * S:(b + 1) * S], alone, tolerance(st))


@pytest.mark.parametrize("kv4", [False, True])
def test_a_cache_lives_as_long_as_the_graph_captured_on_it(kv4):
    """A graph is found again by its cache's address, so the address is not given to another cache while the graph is there."""
    import gc
    import weakref
    st = model().stack
    cache = st.new_cache(24, batch=2, kv4=kv4)
    other = st.new_cache(24, batch=2, kv4=not kv4)                                # lets go of the first one
    x = torch.zeros(2, st.D, dtype=BF16, device=DEV)
    st.decode_step_batched(x, torch.zeros(2, dtype=torch.int32, device=DEV), cache)
    seen = [weakref.ref(t) for layer in cache for t in (layer if kv4 else [layer])]
    del cache
    gc.collect()
    assert len(st._dec_graphs_b) == 1 and all(r() is not None for r in seen)
    assert st.new_cache(24, batch=2, kv4=not kv4) is other and all(r() is not None for r in seen)
    st.invalidate_fp8()
    gc.collect()
    assert all(r() is None for r in seen)
