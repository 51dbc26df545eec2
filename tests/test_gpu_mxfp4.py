"""4-bit operators on the GPU against their definition in 64 bits (mx_ref): quantisation bit for bit, products and attention within bounds
derived from the roundings they make."""
import itertools

import pytest
import torch

import mx_ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HALF_STEP = torch.finfo(BF16).eps / 2                 # 2^-8: one rounding to bf16
U32 = torch.finfo(torch.float32).eps                  # 2^-23: one fp32 operation, truncation allowed for (the matrix pipe does not say how it rounds)


@pytest.fixture(scope="module")
def ops():
    from hvlm import ops
    return ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def same(a, b):
    assert a.dtype == b.dtype and a.shape == b.shape
    assert torch.equal(a, b), f"{int((a != b).sum())} of {a.numel()} differ"


# ---------------------------------------------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", [BF16, torch.float16])
def test_every_finite_value_at_every_scale(ops, dtype):
    """All 65536 bit patterns, each in a block whose maximum sits in turn 0 .. 7 binades above it, plus the patterns by themselves."""
    bits = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16)
    v = bits.view(dtype)
    x = torch.zeros(65536 * 9, 32, dtype=dtype, device="cuda")
    x[:, 5] = v.repeat(9)
    top = torch.where(torch.isfinite(v), v.float().abs(), torch.ones(65536, device="cuda"))
    for j in range(8):
        x[(j + 1) * 65536:(j + 2) * 65536, 31] = (top * 2.0 ** j).to(dtype)       # (overflow to infinity included: a NaN block)
    got, want = ops.quantize_mxfp4(x), mx_ref.quantise(x)
    same(got[1], want[1])
    same(got[0], want[0])


@pytest.mark.parametrize("dtype", [BF16, torch.float16])
def test_dequantise_every_code_and_scale(ops, dtype):
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(256, 1).view(256 * 16, 16)
    scales = torch.arange(256, dtype=torch.uint8, device="cuda").repeat_interleave(16).view(-1, 1)
    got = ops.dequantize_mxfp4((codes, scales), out_dtype=dtype)
    want = mx_ref.values((codes, scales)).to(torch.float32).to(dtype)             # (fp32 holds every value: one rounding, to fp16 only)
    same(got.view(torch.int16)[~torch.isnan(want)], want.view(torch.int16)[~torch.isnan(want)])
    assert torch.equal(torch.isnan(got), torch.isnan(want))


@pytest.mark.parametrize("rows,K", [(1, 32), (1, 4096), (3, 96), (867, 4096), (130, 13824), (65, 32 * 33)])
@pytest.mark.parametrize("dtype", [BF16, torch.float16])
def test_quantise_shapes_and_strides(ops, rows, K, dtype):
    g = gen(rows * 7 + K)
    wide = (torch.randn(rows, K + 40, device="cuda", generator=g) * torch.exp2(torch.randint(-6, 6, (rows, 1), device="cuda", generator=g).float())).to(dtype)
    for x in (wide[:, 8:8 + K], wide[:, 8:8 + K].contiguous()):                   # rows K + 40 apart and dense
        got, want = ops.quantize_mxfp4(x), mx_ref.quantise(x)
        same(got[0], want[0])
        same(got[1], want[1])
    buf = (torch.full((rows, K // 2 + 16), 77, dtype=torch.uint8, device="cuda"), torch.full((rows, K // 32 + 3), 77, dtype=torch.uint8, device="cuda"))
    out = (buf[0][:, 4:4 + K // 2], buf[1][:, 1:1 + K // 32])
    ops.quantize_mxfp4(wide[:, 8:8 + K], out=out)
    same(out[0].contiguous(), want[0])
    same(out[1].contiguous(), want[1])
    assert (buf[0][:, :4] == 77).all() and (buf[0][:, 4 + K // 2:] == 77).all() and (buf[1][:, 0] == 77).all() and (buf[1][:, 1 + K // 32:] == 77).all()
    same(ops.dequantize_mxfp4(out), mx_ref.values(want).to(BF16))


def test_quantise_special_blocks(ops):
    x = torch.randn(8, 32, device="cuda", generator=gen(1)).to(BF16)
    x[0], x[1, 3], x[2, 31], x[3, 0] = 0, float("nan"), float("inf"), float("-inf")
    x[4] = -0.0
    x[5] = 1e-40                                                                  # bf16 subnormals
    x[6, 7] = 3e38
    got, want = ops.quantize_mxfp4(x), mx_ref.quantise(x)
    same(got[0], want[0])
    same(got[1], want[1])
    assert got[1].flatten().tolist()[:4] == [0, 255, 255, 255] and got[1][4] == 0


def test_quantise_past_32_bit_offsets(ops):
    rows, K = 140_000, 16384                                                      # 2.3e9 elements, 4.6 GB
    x = torch.empty(rows, K, dtype=BF16, device="cuda")
    x[-3:] = torch.randn(3, K, device="cuda", generator=gen(2)).to(BF16)
    x[:-3].zero_()
    got, want = ops.quantize_mxfp4(x), mx_ref.quantise(x[-3:])
    same(got[0][-3:], want[0])
    same(got[1][-3:], want[1])
    back = ops.dequantize_mxfp4(got)
    same(back[-3:], mx_ref.values(want).to(BF16))


# -------------------------------------------------------------------------------------------------------------------- products
def product_bound(a, b, y):
    """K terms, every product exact in fp32, summed in any order: (K + 1) roundings of partial sums no larger than sum |a b|; then bf16."""
    return (a.shape[1] + 1) * U32 * (a.abs() @ b.abs().t()) + HALF_STEP * y.abs()


def check_product(got, a, b, bias=None, residual=None, act=False, f32=False):
    y = a @ b.t()
    tol = product_bound(a, b, torch.zeros_like(y))
    if bias is not None:
        y = y + bias.double()
        tol = tol + U32 * y.abs()
    if act:
        # |d/dx x sigmoid(1.702 x)| <= 1.1; exp2 and rcp are good to 1 ulp, their argument to |1.702 log2(e) y| half-steps: 4 + 2.5 |y| in all
        tol = 1.1 * tol + (4 + 2.5 * y.abs()) * U32 * y.abs()
        y = mx_ref.gelu(y)
    if residual is not None:
        y = y + residual.double()
        tol = tol + U32 * y.abs()
    if not f32:
        tol = tol + HALF_STEP * (y.abs() + tol)
    err = (got.double() - y).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol + 1e-300).all(), f"worst {(err / (tol + 1e-300)).max().item():.3f} of the bound"


GEMM_SHAPES = [(1, 1, 32), (5, 7, 64), (128, 128, 128), (129, 127, 96), (33, 1000, 160), (256, 256, 512), (867, 515, 4096), (300, 260, 1056), (257, 4096, 1024), (64, 33, 13824),
               (1030, 777, 2048 + 32)]


@pytest.mark.parametrize("M,N,K", GEMM_SHAPES)
def test_gemm_shapes(ops, M, N, K):
    g = gen(M * 31 + N * 7 + K)
    a, b = mx_ref.random_pair(M, K, g, "cuda"), mx_ref.random_pair(N, K, g, "cuda")
    va, vb = mx_ref.values(a), mx_ref.values(b)
    check_product(ops.gemm_mxfp4_nt(a, b), va, vb)
    check_product(ops.gemm_mxfp4_nt(a, b, out_dtype=torch.float32), va, vb, f32=True)
    bias = torch.randn(N, device="cuda", generator=g).to(BF16)
    res = torch.randn(M, N, device="cuda", generator=g).to(BF16)
    check_product(ops.gemm_mxfp4_nt(a, b, bias=bias, act=ops.ACT_QUICK_GELU), va, vb, bias=bias, act=True)
    check_product(ops.gemm_mxfp4_nt(a, b, bias=bias, residual=res), va, vb, bias=bias, residual=res)
    io = res.clone()                                                              # residual in place
    same(ops.gemm_mxfp4_nt(a, b, residual=io, out=io), ops.gemm_mxfp4_nt(a, b, residual=res))


def strided(pair, cpad, coff, spad, soff):
    """The same MXFP4 matrix inside wider buffers full of NaN scales."""
    c, s = pair
    bc = torch.full((c.shape[0], c.shape[1] + cpad), 0x77, dtype=torch.uint8, device=c.device)
    bs = torch.full((s.shape[0], s.shape[1] + spad), 255, dtype=torch.uint8, device=c.device)
    bc[:, coff:coff + c.shape[1]] = c
    bs[:, soff:soff + s.shape[1]] = s
    return bc[:, coff:coff + c.shape[1]], bs[:, soff:soff + s.shape[1]]


@pytest.mark.parametrize("M,N,K", [(130, 140, 96), (40, 300, 1056), (300, 129, 512), (600, 600, 4096)])
def test_gemm_strides(ops, M, N, K):
    """Operand rows inside wider buffers (what lies between them is NaN), outputs and residuals with odd leading dimensions."""
    g = gen(M + N + K)
    a, b = mx_ref.random_pair(M, K, g, "cuda"), mx_ref.random_pair(N, K, g, "cuda")
    want = ops.gemm_mxfp4_nt(a, b)
    check_product(want, mx_ref.values(a), mx_ref.values(b))
    sa, sb = strided(a, 48, 16, 5, 2), strided(b, 16, 0, 3, 1)
    same(ops.gemm_mxfp4_nt(sa, sb), want)
    for pad, off in ((3, 1), (8, 4)):
        buf = torch.full((M, N + pad), 9.0, dtype=BF16, device="cuda")
        res = torch.randn(M, N + pad, device="cuda", generator=g).to(BF16)[:, off - 1:off - 1 + N]
        out = ops.gemm_mxfp4_nt(a, b, residual=res, out=buf[:, off:off + N])
        same(out.contiguous(), ops.gemm_mxfp4_nt(a, b, residual=res.contiguous()))
        assert (buf[:, :off] == 9).all() and (buf[:, off + N:] == 9).all()


def test_gemm_nan_block_stays_in_its_row(ops):
    g = gen(3)
    a, b = mx_ref.random_pair(200, 256, g, "cuda"), mx_ref.random_pair(150, 256, g, "cuda")
    a[1][77, 3] = 255
    b[1][149, 0] = 255
    y = ops.gemm_mxfp4_nt(a, b)
    nan = torch.zeros(200, 150, dtype=torch.bool, device="cuda")
    nan[77], nan[:, 149] = True, True
    assert torch.equal(torch.isnan(y), nan)


def test_gemm_extreme_scales(ops):
    """Scale codes from both ends: the products stay exact powers of two apart."""
    g = gen(4)
    for lo_a, lo_b in ((1, 250), (250, 1), (60, 60), (2, 130), (190, 60)):
        a, b = mx_ref.random_pair(64, 128, g, "cuda", lo_a, lo_a + 2), mx_ref.random_pair(64, 128, g, "cuda", lo_b, lo_b + 2)
        y = mx_ref.values(a) @ mx_ref.values(b).t()
        got = ops.gemm_mxfp4_nt(a, b, out_dtype=torch.float32)
        tol = product_bound(mx_ref.values(a), mx_ref.values(b), torch.zeros_like(y)) + 2.0 ** -126          # (results below the normal range may flush)
        assert ((got.double() - y).abs() <= tol).all()


def test_gemm_past_32_bit_offsets(ops):
    M, N, K = 70_000, 32_101, 32                                                  # 2.2e9 outputs
    g = gen(5)
    a, b = mx_ref.random_pair(M, K, g, "cuda"), mx_ref.random_pair(N, K, g, "cuda")
    y = ops.gemm_mxfp4_nt(a, b)
    check_product(y[-130:], mx_ref.values(a)[-130:], mx_ref.values(b))
    check_product(y[:130], mx_ref.values(a)[:130], mx_ref.values(b))
    del y
    M, K = 140_000, 32768                                                         # 2.3 GB of codes
    a, b = mx_ref.random_pair(M, K, g, "cuda"), mx_ref.random_pair(40, K, g, "cuda")
    check_product(ops.gemm_mxfp4_nt(a, b)[-50:], mx_ref.values((a[0][-50:], a[1][-50:])), mx_ref.values(b))


SKINNY = list(itertools.product((1, 2, 7, 13, 16, 17, 32), ((1, 32), (130, 96), (515, 1056), (4096, 4096), (1000, 13824)))) + [(1, (22016, 4096)), (1, (48, 14336)), (1, (100, 14368)), (2, (50, 7168)), (3, (50, 4768)), (3, (33, 4128)), (2, (40, 8192)), (4, (40, 4096)), (4, (17, 160)), (32, (5120, 13824))]


@pytest.mark.parametrize("M,NK", SKINNY)
def test_w4a16_shapes(ops, M, NK):
    N, K = NK
    g = gen(M * 31 + N * 7 + K)
    w = mx_ref.random_pair(N, K, g, "cuda")
    x = torch.randn(M, K + 8, device="cuda", generator=g).to(BF16)[:, 8:]
    vx, vw = x.double(), mx_ref.values(w)
    check_product(ops.gemm_w4a16_nt(x, w), vx, vw)
    bias = torch.randn(N, device="cuda", generator=g).to(BF16)
    res = torch.randn(M, N, device="cuda", generator=g).to(BF16)
    check_product(ops.gemm_w4a16_nt(x, w, bias=bias, residual=res, act=ops.ACT_QUICK_GELU), vx, vw, bias=bias, residual=res, act=True)
    sw = strided(w, 32, 16, 5, 3)
    same(ops.gemm_w4a16_nt(x.contiguous(), sw, residual=res), ops.gemm_w4a16_nt(x, w, residual=res))
    buf = torch.full((M, N + 3), 9.0, dtype=BF16, device="cuda")
    same(ops.gemm_w4a16_nt(x, w, out=buf[:, 1:1 + N]).contiguous(), ops.gemm_w4a16_nt(x, w))
    assert (buf[:, 0] == 9).all() and (buf[:, 1 + N:] == 9).all()


def test_w4a16_rows_do_not_mix(ops):
    """A NaN in one row of x, an infinity in another: the other rows keep their bits."""
    g = gen(6)
    w = mx_ref.random_pair(300, 1056, g, "cuda")
    x = torch.randn(19, 1056, device="cuda", generator=g).to(BF16)
    want = ops.gemm_w4a16_nt(x, w)
    x[3, 1055], x[17, 0] = float("nan"), float("inf")
    got = ops.gemm_w4a16_nt(x, w)
    keep = [m for m in range(19) if m not in (3, 17)]
    same(got[keep], want[keep])
    assert torch.isnan(got[3]).all() and not torch.isfinite(got[17]).any()


# -------------------------------------------------------------------------------------------------------------------- the cache
def make_cache(ops, B, Hkv, n, dh, g):
    c = ops.KV4Cache.empty(B, n, Hkv, dh, "cuda")
    for code, sc in ((c.k, c.k_scale), (c.v, c.v_scale)):
        q = mx_ref.quantise(torch.randn(B * Hkv * n, dh, device="cuda", generator=g).to(BF16))
        code.copy_(q[0].view(code.shape))
        sc.copy_(q[1].view(sc.shape))
    return c


def attn_ref(q, cache, lens, H, scale):
    """Per sample and head in float64; returns (out, tolerance)."""
    B, Hkv, n, half = cache.k.shape
    dh = 2 * half
    out = torch.zeros(B, H * dh, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(B):
        m = max(0, min(int(lens[b]), n))
        if m == 0:
            continue
        for h in range(H):
            k = mx_ref.values((cache.k[b, h * Hkv // H, :m], cache.k_scale[b, h * Hkv // H, :m]))
            v = mx_ref.values((cache.v[b, h * Hkv // H, :m], cache.v_scale[b, h * Hkv // H, :m]))
            x = q[b, h * dh:(h + 1) * dh].double()
            s = (k @ x) * scale
            p = torch.softmax(s, 0)
            o = p @ v
            # a score is off by its fp32 sum ((dh + 4) terms) and by the rounding of its exponent's argument; both ends of the quotient see it.
            # P is rounded to bf16 once, its sums over the keys in fp32 once per key at worst.
            ds = ((dh + 4) * U32 * (k.abs() @ x.abs() * abs(scale)) + 4 * U32 * (1 + s.abs())).max()
            mean = p @ v.abs()
            sl = slice(h * dh, (h + 1) * dh)
            out[b, sl] = o
            tol[b, sl] = HALF_STEP * o.abs() + (HALF_STEP + 4 * ds + 2 * (m + 8) * U32) * mean
    return out, tol


def check_attn(ops, q, cache, lens, H, scale):
    got = ops.attn_decode_kv4(q, cache, lens, H, scale)
    want, tol = attn_ref(q, cache, lens.tolist(), H, scale)
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (err <= tol + 1e-300).all(), f"worst {(err / (tol + 1e-300)).max().item():.3f} of the bound"
    return got


ATTN = [  # B, H, Hkv, dh, max_len, lens
    (1, 1, 1, 128, 1, [1]), (1, 2, 2, 64, 40, [33]), (3, 4, 4, 128, 130, [0, 1, 130]), (2, 8, 2, 128, 300, [300, 17]), (2, 8, 1, 64, 129, [128, 129]),
    (1, 32, 32, 128, 967, [967]), (5, 6, 2, 128, 257, [31, 32, 33, 64, 255]), (2, 16, 1, 128, 700, [513, 699]), (4, 40, 40, 128, 64, [64, 63, 1, 2]),
    (1, 5, 1, 64, 5000, [4999]), (1, 8, 1, 128, 20000, [19999]), (2, 32, 8, 128, 2048, [2048, 1111]), (1, 3, 3, 64, 1000, [2000])]


@pytest.mark.parametrize("B,H,Hkv,dh,n,lens", ATTN)
def test_attention_shapes(ops, B, H, Hkv, dh, n, lens):
    g = gen(B * 101 + H * 11 + n)
    cache = make_cache(ops, B, Hkv, n, dh, g)
    qkv = torch.randn(B, (H + 2 * Hkv) * dh, device="cuda", generator=g).to(BF16)
    check_attn(ops, qkv, cache, torch.tensor(lens, dtype=torch.int32, device="cuda"), H, dh ** -0.5)


def test_attention_ignores_what_lies_past_the_length(ops):
    """Rows past a sample's length hold NaN scales and the largest codes; a length outside 0 .. max_len is clamped."""
    g = gen(7)
    B, H, n, dh = 4, 4, 200, 128
    cache = make_cache(ops, B, H, n, dh, g)
    lens = torch.tensor([0, 1, 77, -5], dtype=torch.int32, device="cuda")
    q = torch.randn(B, H * dh, device="cuda", generator=g).to(BF16)
    want = check_attn(ops, q, cache, lens, H, 0.09)
    for b, m in enumerate([0, 1, 77, 0]):
        cache.k[b, :, m:], cache.v[b, :, m:] = 0x77, 0x77
        cache.k_scale[b, :, m:], cache.v_scale[b, :, m:] = 255, 255
    same(ops.attn_decode_kv4(q, cache, lens, H, 0.09), want)
    assert (want[0] == 0).all() and (want[3] == 0).all()


def test_attention_sharp_and_flat_scores(ops):
    """One key far above the rest, in every tile position; all keys equal; scores of either sign that no exponential holds unshifted."""
    g = gen(8)
    H, dh, n = 2, 128, 180
    q = torch.randn(1, H * dh, device="cuda", generator=g).to(BF16)
    for at in (0, 31, 32, 95, 127, 128, 179):
        cache = make_cache(ops, 1, H, n, dh, g)
        cache.k_scale[0, :, at] += 6
        for scale in (4.0, -4.0, 0.0):
            check_attn(ops, q, cache, torch.tensor([n], dtype=torch.int32, device="cuda"), H, scale)


def test_attention_nan_in_a_used_row(ops):
    g = gen(9)
    cache = make_cache(ops, 2, 2, 100, 64, g)
    cache.v_scale[1, 1, 50, 1] = 255
    q = torch.randn(2, 128, device="cuda", generator=g).to(BF16)
    out = ops.attn_decode_kv4(q, cache, torch.tensor([100, 100], dtype=torch.int32, device="cuda"), 2, 0.125)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[1, 64 + 32:] = True
    assert torch.equal(torch.isnan(out), bad)


@pytest.mark.parametrize("B,S,H,Hkv,dh,n", [(1, 1, 1, 1, 64, 4), (3, 5, 4, 4, 128, 11), (2, 70, 8, 2, 128, 100), (2, 3, 5, 1, 64, 9)])
def test_append(ops, B, S, H, Hkv, dh, n):
    g = gen(B + S + H)
    qkv = torch.randn(B * S, (H + 2 * Hkv) * dh + 16, device="cuda", generator=g).to(BF16)[:, 8:-8]
    start = torch.tensor([n - 2, -1, 3][:B], dtype=torch.int32, device="cuda")   # rows run over either end: dropped there
    count = torch.tensor([S, max(S - 1, 0), 2][:B], dtype=torch.int32, device="cuda")
    for st, ct in ((None, None), (start, None), (start, count)):
        cache = make_cache(ops, B, Hkv, n, dh, g)
        want = [t.clone() for t in cache]
        ops.kv4_append(qkv, cache, st, H, count=ct)
        for b in range(B):
            for s in range(S if ct is None else int(ct[b])):
                pos = s + (0 if st is None else int(st[b]))
                if not 0 <= pos < n:
                    continue
                for j in range(2):
                    lo = (H + j * Hkv) * dh
                    c, z = mx_ref.quantise(qkv[b * S + s, lo:lo + Hkv * dh].reshape(Hkv, dh))
                    want[2 * j][b, :, pos], want[2 * j + 1][b, :, pos] = c, z
        for a, w in zip(cache, want):
            same(a, w)


def test_cache_past_32_bit_offsets(ops):
    """Two samples of 8 heads with 2^23 rows each: the second one's codes start past 4 GB."""
    B, H, n, dh = 2, 8, 1 << 23, 128
    cache = ops.KV4Cache.empty(B, n, H, dh, "cuda")
    g = gen(10)
    qkv = torch.randn(B * 40, 3 * H * dh, device="cuda", generator=g).to(BF16)
    ops.kv4_append(qkv, cache, None, H)
    lens = torch.tensor([40, 39], dtype=torch.int32, device="cuda")
    q = qkv[:2]
    small = ops.KV4Cache(*(t[:, :, :40].contiguous() for t in cache))
    want, tol = attn_ref(q, small, [40, 39], H, 0.09)
    got = ops.attn_decode_kv4(q, cache, lens, H, 0.09)
    assert ((got.double() - want).abs() <= tol).all()
    ops.kv4_append(qkv[:2], cache, torch.tensor([n - 1, n - 1], dtype=torch.int32, device="cuda"), H)
    c, z = mx_ref.quantise(qkv[1, 2 * H * dh:].reshape(H, dh))
    same(cache.v[1, :, n - 1], c)
    same(cache.v_scale[1, :, n - 1], z)


# ------------------------------------------------------------------------------------------------- together, streams and graphs
def step(ops, x, w, cache, lens, lens1, H, dh, res):
    """A decode step's attention block and a prefill-style product, as the engine issues them."""
    qkv = ops.gemm_w4a16_nt(x, w["qkv"])
    ops.kv4_append(qkv, cache, lens, H)
    ao = ops.attn_decode_kv4(qkv, cache, lens1, H, dh ** -0.5)
    h = ops.gemm_w4a16_nt(ao, w["o"], residual=res)
    return h, ops.gemm_mxfp4_nt(ops.quantize_mxfp4(h), w["up"], act=ops.ACT_QUICK_GELU)


def test_step_against_definition_streams_and_graph(ops):
    g = gen(11)
    B, H, dh, n = 5, 4, 128, 300
    D = H * dh
    w = {k: mx_ref.random_pair(N, D, g, "cuda", 116, 120) for k, N in (("qkv", 3 * D), ("o", D), ("up", 1001))}
    cache = make_cache(ops, B, H, n, dh, g)
    x, res = (torch.randn(B, D, device="cuda", generator=g).to(BF16) for _ in range(2))
    lens = torch.tensor([0, 5, 299, 128, 31], dtype=torch.int32, device="cuda")
    lens1 = lens + 1
    h, y = step(ops, x, w, cache, lens, lens1, H, dh, res)
    # every stage against its definition on the stage's own input
    qkv = ops.gemm_w4a16_nt(x, w["qkv"])
    check_product(qkv, x.double(), mx_ref.values(w["qkv"]))
    c, z = mx_ref.quantise(qkv[:, D:2 * D].reshape(B * H, dh))
    rows = torch.arange(B, device="cuda")
    same(cache.k[rows, :, lens.long()].reshape(B * H, -1), c)
    same(cache.k_scale[rows, :, lens.long()].reshape(B * H, -1), z)
    ao = check_attn(ops, qkv, cache, lens1, H, dh ** -0.5)
    check_product(h, ao.double(), mx_ref.values(w["o"]), residual=res)
    check_product(y, mx_ref.values(mx_ref.quantise(h)), mx_ref.values(w["up"]), act=True)
    # another stream: same bits
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        h2, y2 = step(ops, x, w, cache, lens, lens1, H, dh, res)
    torch.cuda.current_stream().wait_stream(s)
    same(h2, h)
    same(y2, y)
    # two captured steps, replayed in turn with eager work between, against the eager results
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = step(ops, x, w, cache, lens, lens1, H, dh, res)
    x3 = x.roll(1, 0).contiguous()
    cache3 = make_cache(ops, B, H, n, dh, g)
    with torch.cuda.graph(g2):
        o2 = step(ops, x3, w, cache3, lens, lens1, H, dh, res)
    for i in range(3):
        x.copy_(torch.randn(B, D, device="cuda", generator=g).to(BF16))
        x3.copy_(x.roll(1, 0))
        lens.copy_(torch.tensor([i, 7 * i, 299, 128 + i, 31 + i], dtype=torch.int32))
        lens1.copy_(lens + 1)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        r1 = [t.clone() for t in o1]
        r2 = [t.clone() for t in o2]
        for a, b in zip(r1, step(ops, x, w, cache, lens, lens1, H, dh, res)):
            same(a, b)
        for a, b in zip(r2, step(ops, x3, w, cache3, lens, lens1, H, dh, res)):
            same(a, b)


@pytest.mark.parametrize("M,N,K", [(3, 515, 4096), (30, 130, 1056), (130, 333, 96), (600, 900, 512)])
def test_the_result_may_take_the_residual_s_place(ops, M, N, K):
    g = gen(13)
    a, b = mx_ref.random_pair(M, K, g, "cuda"), mx_ref.random_pair(N, K, g, "cuda")
    res = torch.randn(M, N, device="cuda", generator=g).to(BF16)
    calls = [lambda r, out: ops.gemm_mxfp4_nt(a, b, residual=r, out=out)]
    if M <= 32:
        x = torch.randn(M, K, device="cuda", generator=g).to(BF16)
        calls.append(lambda r, out: ops.gemm_w4a16_nt(x, b, residual=r, out=out))
    for call in calls:
        place = res.clone()
        same(call(place, place), call(res, None))


def test_results_do_not_depend_on_what_ran_before(ops):
    """The same call twice with other shapes between: the same bits (no state is kept, no atomics)."""
    g = gen(12)
    B, H, n, dh = 3, 8, 1500, 128
    cache = make_cache(ops, B, H, n, dh, g)
    q = torch.randn(B, H * dh, device="cuda", generator=g).to(BF16)
    lens = torch.tensor([1500, 700, 3], dtype=torch.int32, device="cuda")
    w = mx_ref.random_pair(515, 4096, g, "cuda")
    x = torch.randn(9, 4096, device="cuda", generator=g).to(BF16)
    first = ops.attn_decode_kv4(q, cache, lens, H, 0.09), ops.gemm_w4a16_nt(x, w)
    for _ in range(3):
        ops.attn_decode_kv4(q[:1], ops.KV4Cache(*(t[:1, :, :640].contiguous() for t in cache)), lens[:1], H, 0.09)
        ops.gemm_w4a16_nt(x[:2], mx_ref.random_pair(96, 4096, g, "cuda"))
        again = ops.attn_decode_kv4(q, cache, lens, H, 0.09), ops.gemm_w4a16_nt(x, w)
        same(again[0], first[0])
        same(again[1], first[1])
