"""MXFP4 from its definition, in 64 bits: what the 4-bit tests compare the kernels with.  Written for any device; no product code."""
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def two_to(e):
    """2.0 ** e for whole e, from its bits (the device's pow is off by an ulp for some whole e, which would move ties)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantise(x):
    """x [R, K] -> (codes uint8 [R, K / 2], scales uint8 [R, K / 32])."""
    R, K = x.shape
    b = x.double().reshape(R, K // 32, 32)
    top = b.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(b).all(-1, keepdim=True)
    m, e = torch.frexp(torch.where(bad, torch.ones_like(top), top))               # top = m 2^e, m in [0.5, 1)
    e = torch.where(top == 0, torch.full_like(e, -127), (e - 3).clamp(min=-127))  # floor(log2 top) - 2
    y = torch.where(bad, torch.zeros_like(b), b) * two_to(-e)
    a = y.abs()
    code = torch.zeros_like(a, dtype=torch.int64)
    g = GRID.tolist()
    for i in range(7):                                                            # code i + 1 from the middle of (i, i + 1); a tie goes to the even code
        mid = (g[i] + g[i + 1]) / 2
        code += (a >= mid) if i % 2 else (a > mid)
    code += 8 * torch.signbit(y).long()
    code = torch.where(bad, torch.zeros_like(code), code).reshape(R, K // 2, 2)
    scale = torch.where(bad, torch.full_like(e, 255), e + 127).reshape(R, K // 32)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), scale.to(torch.uint8)


def values(q):
    """(codes [..., K / 2], scales [..., K / 32]) -> float64 [..., K]."""
    codes, scales = q
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = GRID.to(codes.device)[c & 7] * (1.0 - 2.0 * (c >> 3))
    s = two_to(scales.int() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return v * s.repeat_interleave(32, -1)


def random_pair(rows, K, gen, device, lo=118, hi=126):
    """A random MXFP4 matrix with moderate scales."""
    c = torch.randint(0, 256, (rows, K // 2), dtype=torch.uint8, device=device, generator=gen)
    s = torch.randint(lo, hi + 1, (rows, K // 32), dtype=torch.uint8, device=device, generator=gen)
    return c, s


def gelu(y):
    return y * torch.sigmoid(1.702 * y)
