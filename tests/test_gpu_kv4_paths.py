"""Single-token attention over the 4-bit cache in every launch shape that it chooses between, against the definition in 64 bits: rings of tiles that
wrap, splits of several rounds, more than 256 (sample, KV head) pairs on either side of 2048 keys."""
import math

import pytest
import torch

from test_gpu_mxfp4 import HALF_STEP, attn_ref, check_attn, gen, make_cache, ops  # noqa: F401

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


# A wave takes 32 keys at a time and holds four such tiles in its ring: the lengths end its first wave's work behind 1, 3, 4, 5, 8 and 9 tiles.
PATHS = [  # B, H, Hkv, dh, max_len, lens, splits
    # 288 pairs, up to 2048 keys: four waves a head, no split
    (9, 32, 32, 128, 1200, [1200, 512, 513, 1024, 1025, 384, 385, 1, 0], 1),
    (9, 32, 32, 64, 1200, [0, 33, 511, 512, 640, 1023, 1152, 1153, 1200], 1),
    (5, 64, 64, 128, 700, [700, 513, 512, 31, 128], 1),
    # beyond 2048 keys: 4 and 2 splits of several rounds
    (9, 32, 32, 128, 4700, [4700, 2049, 2048, 513, 4096, 4097, 1, 0, 3000], 4),
    (9, 32, 32, 64, 4700, [100, 4608, 4609, 2304, 0, 1024, 4700, 2500, 5], 4),
    (16, 64, 32, 128, 2300, [2300, 2299, 2048, 2049, 1024, 1025, 0, 1, 512, 513, 128, 129, 700, 1800, 2177, 2176], 2),
    # 128 pairs, one workgroup of eight waves a head, up to ten tiles a wave
    (4, 32, 32, 128, 2500, [2500, 1280, 1281, 2304], 1),
    (4, 32, 32, 64, 2500, [2305, 2500, 1024, 1025], 1),
    # 64 pairs with shared heads and long caches: 16 splits of up to ten rounds
    (8, 32, 8, 128, 20000, [20000, 8192, 8193, 16384, 1, 0, 10241, 19999], 16),
    (8, 32, 8, 64, 20000, [16385, 20000, 4096, 129, 10240, 0, 18432, 7], 16),
    # one sample, 32 heads, 16 splits
    (1, 32, 32, 128, 12000, [11999], 16),
    # 12 and 16 heads on one KV head
    (2, 24, 2, 128, 1500, [1500, 1281], 12),
    (2, 32, 2, 64, 1500, [1407, 1500], 12),
]


@pytest.mark.parametrize("B,H,Hkv,dh,n,lens,splits", PATHS)
def test_attention_launch_shapes(ops, B, H, Hkv, dh, n, lens, splits):  # noqa: F811
    from hvlm import _lib
    assert _lib.load().hvlm_attn_decode_kv4_ws_bytes(B, H, Hkv, dh, n) == (0 if splits == 1 else B * H * splits * (dh + 2) * 4)
    g = gen(B * 101 + H * 11 + n + dh)
    cache = make_cache(ops, B, Hkv, n, dh, g)
    q = torch.randn(B, H * dh, device="cuda", generator=g).to(BF16)
    out = check_attn(ops, q, cache, torch.tensor(lens, dtype=torch.int32, device="cuda"), H, dh ** -0.5)
    for b, m in enumerate(lens):
        assert (out[b] == 0).all() == (m == 0)


@pytest.mark.parametrize("B,H,Hkv,dh,n", [(2, 4, 2, 128, 300), (9, 32, 32, 64, 700), (2, 8, 8, 128, 3000)])
def test_scores_that_are_not_finite(ops, B, H, Hkv, dh, n):  # noqa: F811
    """What softmax makes of them: a head whose scores are all -inf has no result (0 / 0), no more than one with +inf or NaN among its scores.  The
    other heads and samples keep their bits, and no keys still give zeros."""
    g = gen(n)
    cache = make_cache(ops, B, Hkv, n, dh, g)
    G = H // Hkv
    lens = torch.tensor([n, n - 37][:B] + [0] * (B - 2), dtype=torch.int32, device="cuda")
    q = torch.randn(B, H * dh, device="cuda", generator=g).to(BF16)
    want = check_attn(ops, q, cache, lens, H, dh ** -0.5)
    h0 = G                                                                     # a query head on KV head 1, whose element 3 gets one sign in every key
    nan = torch.zeros_like(want, dtype=torch.bool)
    for code, bad in ((0x9, float("inf")), (0x2, float("-inf")), (0x2, float("inf")), (0x2, float("nan"))):
        c, x = ops.KV4Cache(*(t.clone() for t in cache)), q.clone()
        c.k[0, 1, :, 1] = (c.k[0, 1, :, 1] & 0x0F) | (code << 4)              # -0.5 or 1
        x[0, h0 * dh + 3] = bad
        got = ops.attn_decode_kv4(x, c, lens, H, dh ** -0.5)
        nan[:] = False
        nan[0, h0 * dh:(h0 + 1) * dh] = True
        assert torch.equal(torch.isnan(got), nan), (code, bad)
        keep = ~nan
        keep[0, G * dh:2 * G * dh] = False                                     # (KV head 1's other heads see other keys)
        assert torch.equal(got[keep], want[keep])


PRECISE = [(1, 32, 32, 128, 967, [967]), (9, 32, 32, 64, 700, [700, 513, 31] * 3), (2, 8, 1, 128, 3000, [3000, 1111]), (2, 18, 2, 128, 500, [500, 77]),
           (2, 16, 1, 64, 1500, [1500, 1281]), (9, 64, 32, 128, 2500, [2500, 2049, 1000] * 3)]


@pytest.mark.parametrize("B,H,Hkv,dh,n,lens", PRECISE)
def test_equal_scores_leave_a_constant_value_as_it_is(ops, B, H, Hkv, dh, n, lens):  # noqa: F811
    """Every value row is 1, so every result is 1.  One key in 32 scores 0.6916.. above the others, whose probability 0.5 (1 + 2^-8 - 2^-12) lies
    just short of half a bf16 step above 0.5: rounded there and not in their sum, they would lose 2^-8 of it together.  What 32 bits lose, (n + 8) 2^-23, and what two bf16 terms lose,
    2^-16, is far from half a step below 1, which is 2^-9."""
    cache = ops.KV4Cache(*(torch.full(t.shape, fill, dtype=torch.uint8, device="cuda")
                           for t, fill in zip(ops.KV4Cache.empty(B, n, Hkv, dh, "cuda"), (0x00, 127, 0x22, 127))))
    cache.k[..., 0] = 0x01                                                     # 0.5 in element 0,
    cache.k[:, :, ::32, 0] = 0x02                                              # 1 in every 32nd row
    q = torch.zeros(B, H, dh, dtype=BF16, device="cuda")
    q[:, :, 0] = 1.0
    scale = -2.0 * math.log(0.5 * (1 + 2.0 ** -8 - 2.0 ** -12))
    out = ops.attn_decode_kv4(q.view(B, H * dh), cache, torch.tensor(lens, dtype=torch.int32, device="cuda"), H, scale)
    assert (out == 1).all(), out.unique()


@pytest.mark.parametrize("B,H,Hkv,dh,n,lens", PRECISE)
def test_probabilities_are_not_rounded_to_bf16(ops, B, H, Hkv, dh, n, lens):  # noqa: F811
    """The bound of test_attention_shapes with 2^-16 of p |v| for the two terms of P in the place of 2^-8 for a single one."""
    g = gen(B + H + n)
    cache = make_cache(ops, B, Hkv, n, dh, g)
    q = torch.randn(B, H * dh, device="cuda", generator=g).to(BF16)
    got = ops.attn_decode_kv4(q, cache, torch.tensor(lens, dtype=torch.int32, device="cuda"), H, dh ** -0.5)
    want, tol = attn_ref(q, cache, lens, H, dh ** -0.5)
    mean, _ = attn_ref(q, cache._replace(v=cache.v & 0x77), lens, H, dh ** -0.5)           # p |v|: codes without their signs
    tol = tol - (HALF_STEP - 2.0 ** -16) * mean
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("B,H,Hkv,dh,n", [(9, 32, 32, 128, 700), (9, 32, 32, 64, 4700), (4, 32, 32, 128, 2500), (2, 24, 2, 128, 1500), (8, 32, 8, 128, 20000)])
def test_streams_and_graphs_at_once(ops, B, H, Hkv, dh, n):  # noqa: F811
    """Append and attention of two caches on two streams at once, then from two graphs replayed with eager work between: the bits of one call by itself."""
    g = gen(B + n)
    caches = [make_cache(ops, B, Hkv, n, dh, g) for _ in range(2)]
    qkv = [torch.randn(B, (H + 2 * Hkv) * dh, device="cuda", generator=g).to(BF16) for _ in range(2)]
    lens = [torch.randint(0, n, (B,), device="cuda", generator=g).to(torch.int32) for _ in range(2)]
    lens1 = [t + 1 for t in lens]

    def step(i):
        ops.kv4_append(qkv[i], caches[i], lens[i], H)
        return ops.attn_decode_kv4(qkv[i], caches[i], lens1[i], H, dh ** -0.5)

    want = [step(0), step(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            outs.append(step(i))
    for r in range(3):
        for i in range(2):
            qkv[i].copy_(torch.randn(qkv[i].shape, device="cuda", generator=g))
            lens[i].copy_((lens[i] + 17 * r) % n)
            lens1[i].copy_(lens[i] + 1)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        first = [o.clone() for o in outs]
        assert all(torch.equal(step(i), first[i]) for i in range(2))
