"""The products of the 4-bit formats in every launch shape that they choose between, with every epilogue, against the definition in 64 bits: both tiles of the
4-bit product over one and several groups of K and several tiles a workgroup, every K-slice of the weight-streaming one."""
import pytest
import torch

import mx_ref
from test_gpu_mxfp4 import check_product, gen, ops, same, strided  # noqa: F401

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def up(a, b):
    return -(-a // b)


def scales_of(tile, M, N, K):
    """Bytes of the tiled scales: rows in whole tiles, K in groups of four steps of 128 (tiles of 256) or 256."""
    group = 512 if tile == 256 else 1024
    return (up(M, tile) + up(N, tile)) * tile * up(K, group) * group // 32


# tile, groups of K, tiles a workgroup takes at most; odd and even numbers of groups; rests in M, N and K
TILES = [
    (256, 1, 2, (6000, 4300, 32)), (256, 1, 2, (5000, 5000, 512)), (256, 3, 2, (5000, 5003, 1056)), (256, 3, 2, (4500, 4100, 1536)),
    (256, 8, 1, (3500, 2600, 4096)), (256, 8, 2, (2100, 9000, 4096)), (256, 2, 5, (9000, 8201, 1024)), (256, 2, 2, (2049, 12289, 544)),
    (256, 5, 2, (5000, 4000, 2080)), (128, 1, 5, (4400, 4400, 512)), (128, 3, 2, (2500, 3001, 2080)), (128, 2, 2, (2600, 2903, 1056)), (128, 4, 1, (1000, 1899, 4096)),
]


@pytest.mark.parametrize("tile,groups,rounds,shape", TILES)
def test_product_tiles(ops, tile, groups, rounds, shape):  # noqa: F811
    from hvlm import _lib
    M, N, K = shape
    assert scales_of(128, *shape) != scales_of(256, *shape)
    assert _lib.load().hvlm_gemm_mxfp4_ws_bytes(M, N, K) == scales_of(tile, M, N, K)
    assert up(K, 512 if tile == 256 else 1024) == groups and up(up(up(M, tile) * up(N, tile), 8), 32) == rounds
    g = gen(M + 3 * N + 7 * K)
    a, b = mx_ref.random_pair(M, K, g, "cuda"), mx_ref.random_pair(N, K, g, "cuda")
    va, vb = mx_ref.values(a), mx_ref.values(b)
    bias = torch.randn(N, device="cuda", generator=g).to(BF16)
    res = torch.randn(M, N + 5, device="cuda", generator=g).to(BF16)[:, 2:2 + N]             # odd leading dimension
    gelu = ops.ACT_QUICK_GELU
    plain = ops.gemm_mxfp4_nt(a, b)
    check_product(plain, va, vb)
    for f32 in (False, True):
        kw = dict(out_dtype=F32 if f32 else BF16)
        if f32:
            check_product(ops.gemm_mxfp4_nt(a, b, **kw), va, vb, f32=True)
        check_product(ops.gemm_mxfp4_nt(a, b, bias=bias, **kw), va, vb, bias=bias, f32=f32)
        check_product(ops.gemm_mxfp4_nt(a, b, residual=res, **kw), va, vb, residual=res, f32=f32)
        check_product(ops.gemm_mxfp4_nt(a, b, bias=bias, act=gelu, **kw), va, vb, bias=bias, act=True, f32=f32)
        check_product(ops.gemm_mxfp4_nt(a, b, bias=bias, residual=res, **kw), va, vb, bias=bias, residual=res, f32=f32)
        check_product(ops.gemm_mxfp4_nt(a, b, bias=bias, residual=res, act=gelu, **kw), va, vb, bias=bias, residual=res, act=True, f32=f32)
    check_product(ops.gemm_mxfp4_nt(a, b, act=gelu), va, vb, act=True)
    # operands and results inside wider buffers, the result in the residual's place: the same bits, and nothing beside them is touched
    same(ops.gemm_mxfp4_nt(strided(a, 48, 16, 5, 2), strided(b, 16, 0, 3, 1)), plain)
    want = ops.gemm_mxfp4_nt(a, b, residual=res)
    for pad, off in ((3, 1), (8, 4)):
        buf = torch.full((M, N + pad), 9.0, dtype=BF16, device="cuda")
        same(ops.gemm_mxfp4_nt(a, b, residual=res, out=buf[:, off:off + N]).contiguous(), want)
        assert (buf[:, :off] == 9).all() and (buf[:, off + N:] == 9).all()
        buf[:, off:off + N] = res
        place = buf[:, off:off + N]
        same(ops.gemm_mxfp4_nt(a, b, residual=place, out=place).contiguous(), want)
        assert (buf[:, :off] == 9).all() and (buf[:, off + N:] == 9).all()
    for _ in range(3):
        same(ops.gemm_mxfp4_nt(a, b), plain)


# M, (N, K), steps of 128 k in a slice
SLICES = [(5, (4096, 11008), 6), (16, (5003, 13824), 6), (13, (22016, 4096), 8), (8, (5120, 5120), 8), (16, (32101, 4096), 8), (17, (32101, 4096), 8),
          (32, (22016, 4096), 8), (25, (15360, 5120), 8), (32, (10001, 4128), 6), (20, (8000, 4128), 6), (24, (27648, 5120), 6), (31, (4091, 4096), 4), (6, (12288, 4096), 4)]


@pytest.mark.parametrize("M,NK,steps", SLICES)
def test_weight_streaming_slices(ops, M, NK, steps):  # noqa: F811
    from hvlm import _lib
    N, K = NK
    assert _lib.load().hvlm_gemm_w4a16_ws_bytes(M, N, K) == up(up(K, 128), steps) * M * up(N, 4) * 16
    assert len({up(up(K, 128), s) for s in (4, 6, 8)}) == 3
    g = gen(M + 3 * N + 7 * K)
    w = mx_ref.random_pair(N, K, g, "cuda")
    x = torch.randn(M, K + 16, device="cuda", generator=g).to(BF16)[:, 8:8 + K]
    vx, vw = x.double(), mx_ref.values(w)
    bias = torch.randn(N, device="cuda", generator=g).to(BF16)
    res = torch.randn(M, N + 5, device="cuda", generator=g).to(BF16)[:, 2:2 + N]
    gelu = ops.ACT_QUICK_GELU
    plain = ops.gemm_w4a16_nt(x, w)
    check_product(plain, vx, vw)
    check_product(ops.gemm_w4a16_nt(x, w, bias=bias), vx, vw, bias=bias)
    check_product(ops.gemm_w4a16_nt(x, w, residual=res), vx, vw, residual=res)
    check_product(ops.gemm_w4a16_nt(x, w, bias=bias, residual=res, act=gelu), vx, vw, bias=bias, residual=res, act=True)
    same(ops.gemm_w4a16_nt(x.contiguous(), strided(w, 32, 16, 5, 3)), plain)
    buf = torch.full((M, N + 3), 9.0, dtype=BF16, device="cuda")
    buf[:, 1:1 + N] = res
    place = buf[:, 1:1 + N]
    same(ops.gemm_w4a16_nt(x, w, residual=place, out=place).contiguous(), ops.gemm_w4a16_nt(x, w, residual=res))
    assert (buf[:, 0] == 9).all() and (buf[:, 1 + N:] == 9).all()
    for _ in range(3):
        same(ops.gemm_w4a16_nt(x, w), plain)
