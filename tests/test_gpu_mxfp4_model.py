"""The 4-bit formats through the model on the GPU: prefill, lock-step decode (eager and from its graph) and whole generations."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from oracle import synth  # noqa: E402

BF16 = torch.bfloat16
DEV = "cuda:0"


def model():
    from test_gpu_model import tiny_model
    return tiny_model(training=False)[0]


def snap(stack):
    """Every GEMM weight to an MXFP4 value, which the format then holds exactly."""
    from hvlm import ops
    for lp in stack.layers:
        for k in ("qkv", "o", "gu", "down"):
            lp.w[k].copy_(ops.dequantize_mxfp4(ops.quantize_mxfp4(lp.w[k])))
    stack.invalidate_fp8()


def tolerance(stack):
    """Two evaluations that differ in the order of sums: each of the nine roundings to bf16 of a layer (norm, qkv, RoPE, attention, o, norm, gate|up,
    SwiGLU, down) and the last norm's may fall to neighbouring values, one step or 2^-8 of the value's norm apart."""
    return (9 * stack.L + 1) * 2.0 ** -8


def near(a, b, tol):
    a, b = a.double(), b.double()
    assert torch.isfinite(a).all() and float((a - b).norm()) <= tol * float(b.norm())


def filled(st, B, n, seed):
    """A 4-bit cache with n random rows everywhere."""
    from hvlm import ops
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache = [ops.KV4Cache.empty(B, n, st.H, st.dh, DEV) for _ in range(st.L)]
    for c in cache:
        ops.kv4_append((torch.randn(B * n, 3 * st.D, device=DEV, generator=g) * 0.3).to(BF16), c, None, st.H)
    return cache


def plain(st, cache):
    """The bf16 cache that holds a 4-bit cache's values."""
    from hvlm import ops
    out = []
    for c in cache:
        B, H, n, dh = c.checked("plain")
        t = torch.zeros(B, n, 3, H, dh, dtype=BF16, device=DEV)
        for i, (codes, scales) in ((1, (c.k, c.k_scale)), (2, (c.v, c.v_scale))):
            v = ops.dequantize_mxfp4((codes.reshape(-1, dh // 2), scales.reshape(-1, dh // 32)))
            t[:, :, i] = v.view(B, H, n, dh).transpose(1, 2)
        out.append(t.view(B, n, 3 * H * dh))
    return out


@pytest.mark.parametrize("kw,kv4", [(dict(mxfp4=True), False), (dict(mxfp4=True), True), (dict(), True), (dict(fp8=True), True)])
@pytest.mark.parametrize("B", [3, 33])
def test_decode_graph_is_bit_identical_to_eager(kw, kv4, B, monkeypatch):
    """Several tokens in a row, and two caches of one shape in turn, replayed and issued eagerly."""
    st = model().stack
    n, got = 24, {}
    for mode in ("1", "0"):
        monkeypatch.setenv("HVLM_DECODE_BATCH_GRAPH", mode)
        g = torch.Generator(device=DEV).manual_seed(5)
        caches = [filled(st, B, n, s) for s in (1, 2)]
        if not kv4:
            caches = [plain(st, c) for c in caches]
        lens = (torch.arange(B, dtype=torch.int32, device=DEV) * 5) % 17
        hs = []
        for step in range(4):
            x = (torch.randn(B, st.D, device=DEV, generator=g) * 0.5).to(BF16)
            hs += [st.decode_step_batched(x, lens, c, **kw).clone() for c in caches]
            lens = lens + 1
        got[mode] = hs + [t.clone() for c in caches for layer in c for t in (layer if kv4 else [layer[:, :, st.D:]])]
    assert all(torch.equal(a, b) for a, b in zip(got["1"], got["0"]))
    assert not torch.equal(got["1"][0], got["1"][1]) and all(torch.isfinite(h.float()).all() for h in got["1"][:8])


@pytest.mark.parametrize("B", [1, 5, 32])
def test_decode_weights_and_cache_against_the_bf16_step(B):
    """On weights that MXFP4 holds exactly, a step with 4-bit weights is the bf16 step; a step on the 4-bit cache is the bf16 step on a cache that
    holds its values (the new token's row among them)."""
    from hvlm import ops
    st = model().stack
    snap(st)
    n = 40
    g = torch.Generator(device=DEV).manual_seed(B)
    x = torch.randn(B, st.D, device=DEV, generator=g).to(BF16)
    lens = (torch.arange(B, dtype=torch.int32, device=DEV) * 13) % n
    cache = filled(st, B, n, 7)
    base = st._decode_step_batched_eager(x, lens, plain(st, cache))
    near(st._decode_step_batched_eager(x, lens, plain(st, cache), mxfp4=True), base, tolerance(st))
    got = st._decode_step_batched_eager(x, lens, cache, mxfp4=True)
    held = {id(c): p for c, p in zip(cache, plain(st, cache))}
    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(ops, "kv4_append", lambda *a: None)
        mp.setattr(ops, "attn_decode_kv4", lambda q, c, le, H, s: ops.attn_decode_batched(q, held[id(c)], le, H, st.dh, s))
        ref = st._decode_step_batched_eager(x, lens, cache, mxfp4=True)
    near(got, ref, tolerance(st))


@pytest.mark.parametrize("B,S", [(1, 33), (2, 17), (3, 70), (1, 20)])
def test_prefill_against_products_of_the_same_values(B, S):
    """The 4-bit prefill = the bf16 GEMM on the values of both 4-bit operands (all exact in bf16); up to 32 rows keep their activations in bf16."""
    from hvlm import ops
    st = model().stack
    x = torch.randn(B * S, st.D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(S)).to(BF16)
    cache = st.new_cache(S + 3, batch=B, kv4=True)
    got = st.forward(x, B, S, save=False, cache=cache, mxfp4=True)
    held = [t.clone() for t in cache[0]]
    back = ops.dequantize_mxfp4
    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(ops, "gemm_mxfp4_nt", lambda a, w, residual=None: ops.gemm_nt(back(a), back(w), residual=residual))
        mp.setattr(ops, "gemm_w4a16_nt", lambda a, w, residual=None: ops.gemm_nt(a, back(w), residual=residual))
        ref = st.forward(x, B, S, save=False, cache=cache, mxfp4=True)
    near(got, ref, tolerance(st))
    for a, b in zip(held, cache[0]):                                              # the first layer's rows: the same codes but for ties that a bf16 step moves
        assert float((a[:, :, :S] != b[:, :, :S]).float().mean()) < 0.02


def test_generation_with_every_switch():
    """sample_batch with 4-bit prefill, decode weights and cache: the forced tokens, hand counts, repeatable to the bit, and the hands of a run whose
    products and attention see the same values in bf16."""
    from hvlm import ops
    m = model()
    st = m.stack
    B, T = 3, 16
    c = synth.TINY
    ids, _, mask = synth.make_text_batch(B, T, seed=8, n_hand=(0, 0, 0), pad_tail=(0, 5, 2))
    images = synth.make_images(B, c["frames"], 2, c["image"], seed=12).to(BF16)
    forced = [[512, 32100, 32100, 77, 2], [32100, 9, 32100, 32100, 2], [600, 601, 2, 2, 2]]
    g = torch.Generator().manual_seed(4)
    noise = [[2.0 * torch.randn(2, 256, generator=g) for _ in range(4)] for _ in range(B)]

    def force(cur, scores):
        out = torch.full_like(scores, -1e9)
        for b in range(B):
            out[b, forced[b][min(cur.shape[1] - T, 4)]] = 0.0
        return out

    run = lambda **kw: m.sample_batch(ids, logits_processor=[force], max_length=T + 5, eos_token_id=2, attention_mask=mask, image=images,  # noqa: E731
                                      hand_noise=noise, **kw)
    every = dict(mxfp4=True, mxfp4_decode=True, kv4=True)
    base = run()
    outs = [run(**every), run(**every)]
    for o in outs + [run(kv4=True), run(fp8=True, fp8_decode=True, kv4=True), run(mxfp4_decode=True)]:
        assert torch.equal(o.sequences, base.sequences) and o.num_hands == base.num_hands == [2, 3, 0] and o.lengths == base.lengths
        assert torch.isfinite(o.pred_hands).all()
    assert torch.equal(outs[0].pred_hands, outs[1].pred_hands)
    assert torch.equal(run().pred_hands, base.pred_hands)                         # the bf16 run is what it was before the 4-bit ones
    back = ops.dequantize_mxfp4
    with pytest.MonkeyPatch.context() as mp:
        mp.setenv("HVLM_DECODE_BATCH_GRAPH", "0")
        mp.setattr(ops, "gemm_mxfp4_nt", lambda a, w, residual=None: ops.gemm_nt(back(a), back(w), residual=residual))
        mp.setattr(ops, "gemm_w4a16_nt", lambda a, w, residual=None: ops.gemm_nt(a, back(w), residual=residual))
        mp.setattr(ops, "attn_decode_kv4", lambda q, kv, le, H, s: ops.attn_decode_batched(q, plain(st, [kv])[0], le, H, st.dh, s))
        ref = run(**every)
    for b in range(B):
        if ref.num_hands[b]:
            near(outs[0].pred_hands[b, :, : ref.num_hands[b]], ref.pred_hands[b, :, : ref.num_hands[b]], tolerance(st))
