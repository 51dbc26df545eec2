"""The ends of the format's range: what bf16 holds of it is exact everywhere, what it does not hold counts as an infinity."""
import pytest
import torch

import mx_ref
from test_gpu_mxfp4 import check_attn, check_product, gen, make_cache, ops, product_bound, same  # noqa: F401

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("M,N,K", [(1, 96, 256), (4, 50, 4096), (13, 130, 544), (32, 600, 1056)])
@pytest.mark.parametrize("lo", [0, 1, 125, 249, 250])
def test_weight_streaming_at_either_end(ops, M, N, K, lo):  # noqa: F811
    """Scale codes 0 .. 252; x takes the products back to the middle of the range (its powers of two are exact)."""
    g = gen(M + N + K + lo)
    w = mx_ref.random_pair(N, K, g, "cuda", lo, lo + 2)
    x = (torch.randn(M, K, device="cuda", generator=g) * 2.0 ** max(min(120 - lo, 100), -100)).to(BF16)
    vx, vw = x.double(), mx_ref.values(w)
    y = vx @ vw.t()
    got = ops.gemm_w4a16_nt(x, w)
    tol = product_bound(vx, vw, torch.zeros_like(y))
    tol = tol + 2.0 ** -8 * (y.abs() + tol) + 2.0 ** -126                          # (below the normal range results may flush)
    assert torch.isfinite(got).all() and ((got.double() - y).abs() <= tol).all()


@pytest.mark.parametrize("scale,code,over", [(252, 7, False), (253, 5, False), (253, 6, True), (253, 7, True), (254, 3, False), (254, 4, True), (254, 15, True)])
def test_values_past_the_range_are_infinities(ops, scale, code, over):  # noqa: F811
    """One element of one weight row; the row's results are infinities of its sign, or what 2^-40 times the value is."""
    g = gen(scale + code)
    sign = -1.0 if code & 8 else 1.0
    for M, N, K in ((3, 40, 64), (20, 300, 1056)):
        w = mx_ref.random_pair(N, K, g, "cuda")
        x = torch.randn(M, K, device="cuda", generator=g).to(BF16)
        x[:, 7] = 2.0 ** -40
        base = ops.gemm_w4a16_nt(x, w)
        w[0][7, 0:16], w[1][7, 0] = 0, scale
        w[0][7, 3] = code << 4                                                     # element 7
        keep = torch.arange(N, device="cuda") != 7
        got = ops.gemm_w4a16_nt(x, w)
        value = ops.dequantize_mxfp4((w[0][7:8], w[1][7:8]))[0, 7].item()
        if over:
            assert value == sign * float("inf") and (got[:, 7] == value).all()
        else:
            assert value == sign * mx_ref.GRID[code & 7].item() * 2.0 ** (scale - 127)
            check_product(got[:, 7:8], x.double(), mx_ref.values((w[0][7:8], w[1][7:8])))
        same(got[:, keep], base[:, keep])


def test_quantised_blocks_stay_inside(ops):  # noqa: F811
    """The largest finite values of either type: no scale code above 252, and every value comes back finite."""
    for dtype in (BF16, torch.float16):
        x = torch.full((4, 64), torch.finfo(dtype).max, dtype=dtype, device="cuda")
        x[1] = -x[1]
        x[2, 1:] = 0
        codes, scales = ops.quantize_mxfp4(x)
        assert int(scales.max()) <= 252 and torch.isfinite(ops.dequantize_mxfp4((codes, scales))).all()


@pytest.mark.parametrize("lo", [40, 200])
def test_attention_on_values_far_from_one(ops, lo):  # noqa: F811
    g = gen(lo)
    cache = make_cache(ops, 2, 4, 300, 128, g)
    cache.v_scale.random_(lo, lo + 3, generator=g)
    q = torch.randn(2, 4 * 128, device="cuda", generator=g).to(BF16)
    check_attn(ops, q, cache, torch.tensor([300, 77], dtype=torch.int32, device="cuda"), 4, 0.09)
