"""Measured cases of the 4-bit operators: microscaled FP4 quantisation, the matrix products on it and attention over a KV cache held in it.

The format is the public OCP Microscaling "MXFP4": blocks of 32 consecutive elements share one power-of-two scale (E8M0, biased by
127; 255 = NaN), the elements are E2M1 (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte with the
even element in the low nibble.  A matrix [R, K] is (codes uint8 [R, K / 2], scales uint8 [R, K / 32]); the scale exponent of a block is
floor(log2(max |x|)) - 2 and an element is rounded to the nearest representable value, ties to even, saturating at 6.

`own` = False computes every operator from elementary torch operations in 32 bits; `own` = True calls the package.
"""
import math
import random
import sys

import torch

own = False

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = 32


# ------------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # ---- quantisation: the activations in front of a product, and back to values
        # one prompt of the batch-1 evaluation (867 rows of the 7B decoder)
        dict(name="quant-prompt", op="quant", rows=867, k=4096, dtype="bf16"),
        # the SwiGLU output of a 16-sample batch: the largest activation that a prefill quantises
        dict(name="quant-batch", op="quant", rows=13872, k=11008, dtype="bf16"),
        # ---- product of 4-bit activations and 4-bit weights (prefill): quantise the rows, multiply
        # q|k|v projection of one prompt: few tiles
        dict(name="linear-prompt-qkv", op="linear", m=867, n=12288, k=4096, epilogue="none"),
        # down projection of one prompt: long K, residual added
        dict(name="linear-prompt-down", op="linear", m=867, n=4096, k=11008, epilogue="residual"),
        # fc1 of the vision tower over one sample's 100 frames of 257 tokens: bias + QuickGELU, short K
        dict(name="linear-vision-fc1", op="linear", m=25700, n=4096, k=1024, epilogue="gelu"),
        # gate|up projection of a 16-sample batch: the largest product of the prefill
        dict(name="linear-batch-gateup", op="linear", m=13872, n=22016, k=4096, epilogue="none"),
        # ---- product of bf16 activations and 4-bit weights (decode steps): one read of the weights
        # one generated token, gate|up
        dict(name="decode-1-gateup", op="decode", m=1, n=22016, k=4096, epilogue="none"),
        # an odd batch in lock step through the 13B down projection
        dict(name="decode-13-down13b", op="decode", m=13, n=5120, k=13824, epilogue="residual"),
        # 32 samples in lock step, the vocabulary projection (odd number of rows)
        dict(name="decode-32-vocab", op="decode", m=32, n=32101, k=4096, epilogue="none"),
        # ---- append the new token's k / v rows to the 4-bit cache and attend over it
        # one sample of the evaluation
        dict(name="attn-1", op="attn", batch=1, heads=32, kv_heads=32, dh=128, max_len=967),
        # 32 samples in lock step with ragged prompts
        dict(name="attn-32", op="attn", batch=32, heads=32, kv_heads=32, dh=128, max_len=1131),
        # long contexts with shared heads
        dict(name="attn-long", op="attn", batch=8, heads=32, kv_heads=8, dh=128, max_len=32768),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("quant", "linear", "decode", "attn"))
    if op == "quant":
        return dict(op=op, rows=_log(rng, 1, 13872), k=BLOCK * _log(rng, 1, 344), dtype=rng.choice(("bf16", "bf16", "f16")))
    epilogue = rng.choice(("none", "residual", "gelu"))
    if op == "linear":
        while True:
            m, n, k = _log(rng, 33, 25700), _log(rng, 64, 32101), BLOCK * _log(rng, 2, 432)
            if m * n * k <= 13872 * 22016 * 4096:
                return dict(op=op, m=m, n=n, k=k, epilogue=epilogue)
    if op == "decode":
        return dict(op=op, m=rng.randint(1, 32), n=_log(rng, 64, 32101), k=BLOCK * _log(rng, 2, 432), epilogue=epilogue)
    while True:
        group = rng.choice((1, 1, 2, 4, 8))
        kv = rng.choice((4, 5, 8, 16, 32, 40))
        dh = rng.choice((64, 128, 128))
        batch, max_len = _log(rng, 1, 64), _log(rng, 1, 32768)
        if group * kv <= 64 and batch * kv * dh * max_len <= 8 * 8 * 128 * 32768 and batch * kv * group * max_len <= 8 * 32 * 32768:
            return dict(op=op, batch=batch, heads=group * kv, kv_heads=kv, dh=dh, max_len=max_len)


def work(case):
    """Each input read once, each output written once: 17 / 32 bytes for an element held in 4 bits."""
    q = 0.5 + 1.0 / BLOCK
    if case["op"] == "quant":
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 + q + 2), "flops": 4 * n}
    if case["op"] in ("linear", "decode"):
        m, n, k = case["m"], case["n"], case["k"]
        extra = {"none": 0, "residual": 2 * m * n, "gelu": 2 * n}[case["epilogue"]]
        return {"bytes": 2 * m * k + q * n * k + 2 * m * n + extra, "flops": 2 * m * n * k}
    B, H, kv, dh = case["batch"], case["heads"], case["kv_heads"], case["dh"]
    keys = sum(_lens(case, 0)) + B                       # (lengths differ a little from seed to seed)
    return {"bytes": 2 * keys * kv * dh * q + B * (2 * H + 2 * kv) * dh * 2, "flops": 4 * keys * H * dh}


def _lens(case, seed):
    """Tokens in the cache before this one: between a third of the capacity and all but the row to be written."""
    r = random.Random(seed * 7919 + case["max_len"])
    top = case["max_len"] - 1
    return [top if case["batch"] == 1 else r.randint(top // 3, top) for _ in range(case["batch"])]


# ------------------------------------------------------------------------------------------------------------- the plain form
def _pow2(e):
    """2 ** e for whole e in [-127, 127], built from its bits."""
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def quantise_plain(x):
    """Float matrix [R, K] -> (codes, scales), 32-bit arithmetic (every step but the rounding to E2M1 is exact)."""
    R, K = x.shape
    xb = x.float().view(R, K // BLOCK, BLOCK)
    amax = xb.abs().amax(-1, keepdim=True)
    e = (torch.frexp(amax)[1] - 3).clamp(-127, 127)                    # floor(log2 amax) - 2
    e = torch.where(amax > 0, e, torch.full_like(e, -127))
    y = xb * _pow2(-e)
    a = y.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    r = torch.round(a / step) * step                                    # half to even on every binade's grid
    code = torch.where(r < 2, 2 * r, torch.where(r < 4, r + 2, r / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(y).to(torch.uint8) << 3)
    bad = ~torch.isfinite(amax)
    code = torch.where(bad, torch.zeros_like(code), code).view(R, K // 2, 2)
    scale = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return code[..., 0] | (code[..., 1] << 4), scale.view(R, K // BLOCK)


_PAIRS = {}


def dequantise_plain(codes, scales):
    """(codes [..., K / 2], scales [..., K / 32]) -> float32 [..., K]."""
    dev = codes.device
    if dev not in _PAIRS:
        g = torch.tensor(GRID + tuple(-v for v in GRID))
        _PAIRS[dev] = torch.stack((g.repeat(16), g.repeat_interleave(16)), 1).to(dev)       # byte -> (low, high) value
    v = _PAIRS[dev].index_select(0, codes.reshape(-1).int()).view(*scales.shape, BLOCK)
    s = torch.where(scales == 255, math.nan, _pow2(scales.int().clamp(max=254) - 127))
    return v.mul_(s.unsqueeze(-1)).view(*codes.shape[:-1], codes.shape[-1] * 2)


def _epilogue(y, st):
    if st["bias"] is not None:
        y = y + st["bias"].to(y.dtype)
        y = y * torch.sigmoid(1.702 * y)
    if st["residual"] is not None:
        y = y + st["residual"].to(y.dtype)
    return y


def _run_plain(st):
    op = st["op"]
    if op == "quant":
        return dequantise_plain(*quantise_plain(st["x"])).to(st["x"].dtype)
    if op in ("linear", "decode"):
        x = dequantise_plain(*quantise_plain(st["x"])) if op == "linear" else st["x"].float()
        return _epilogue(x @ dequantise_plain(st["w"], st["ws"]).t(), st).to(torch.bfloat16)
    B, H, kv, dh, lens = st["batch"], st["heads"], st["kv_heads"], st["dh"], st["lens"]
    rows = torch.arange(B, device=lens.device)
    new = st["qkv"][:, H * dh:].reshape(B, 2, kv, dh)
    for j, (c, s) in enumerate((("k", "ks"), ("v", "vs"))):
        nc, ns = quantise_plain(new[:, j].reshape(B * kv, dh))
        st[c][rows, :, lens.long()] = nc.view(B, kv, dh // 2)
        st[s][rows, :, lens.long()] = ns.view(B, kv, dh // BLOCK)
    q = st["qkv"][:, : H * dh].float().reshape(B, kv, H // kv, dh)
    score = q @ dequantise_plain(st["k"], st["ks"]).transpose(2, 3) * dh ** -0.5
    dead = torch.arange(score.shape[-1], device=lens.device) >= st["lens1"].view(B, 1, 1, 1)
    score = score.masked_fill(dead, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = dequantise_plain(st["v"], st["vs"])
    return dict(out=(p @ v).reshape(B, H * dh).to(torch.bfloat16), k=st["k"], ks=st["ks"], v=st["v"], vs=st["vs"])


# ---------------------------------------------------------------------------------------------------------------- the package
def _ops():
    if "handsonvlm-release_amd" not in sys.path:
        sys.path.insert(0, "handsonvlm-release_amd")
    from hvlm import ops
    return ops


def _run_own(st):
    ops, op = _ops(), st["op"]
    if op == "quant":
        return ops.dequantize_mxfp4(ops.quantize_mxfp4(st["x"]), out_dtype=st["x"].dtype)
    if op in ("linear", "decode"):
        w = (st["w"], st["ws"])
        act = ops.ACT_NONE if st["bias"] is None else ops.ACT_QUICK_GELU
        if op == "linear":
            return ops.gemm_mxfp4_nt(ops.quantize_mxfp4(st["x"]), w, bias=st["bias"], residual=st["residual"], act=act)
        return ops.gemm_w4a16_nt(st["x"], w, bias=st["bias"], residual=st["residual"], act=act)
    cache = ops.KV4Cache(st["k"], st["ks"], st["v"], st["vs"])
    ops.kv4_append(st["qkv"], cache, st["lens"], st["heads"])
    out = ops.attn_decode_kv4(st["qkv"], cache, st["lens1"], st["heads"], st["dh"] ** -0.5)
    return dict(out=out, k=st["k"], ks=st["ks"], v=st["v"], vs=st["vs"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------------------------------------------------- inputs
def _activations(gen, m, k, dtype):
    """Normal values with a few channels far larger than the rest, as a decoder's hidden states have."""
    x = torch.randn((m, k), device="cuda", generator=gen)
    loud = torch.rand(k, device="cuda", generator=gen) < 0.01
    return (x * torch.where(loud, 12.0, 1.0)).to(dtype)


def _cache(gen, B, kv, n, dh):
    """Keys / values of an earlier prompt, quantised head by head: [B, kv, n, dh / 2] codes and [B, kv, n, dh / 32] scales."""
    c = torch.empty((B, kv, n, dh // 2), dtype=torch.uint8, device="cuda")
    s = torch.empty((B, kv, n, dh // BLOCK), dtype=torch.uint8, device="cuda")
    for b in range(B):
        a, z = quantise_plain(_activations(gen, kv * n, dh, torch.bfloat16))
        c[b], s[b] = a.view(kv, n, -1), z.view(kv, n, -1)
    return c, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "quant":
        return dict(op=op, x=_activations(gen, case["rows"], case["k"], torch.float16 if case["dtype"] == "f16" else torch.bfloat16))
    if op in ("linear", "decode"):
        m, n, k = case["m"], case["n"], case["k"]
        st = dict(op=op, x=_activations(gen, m, k, torch.bfloat16), bias=None, residual=None)
        st["w"], st["ws"] = quantise_plain((torch.randn((n, k), device="cuda", generator=gen) * 0.02).to(torch.bfloat16))
        if case["epilogue"] == "residual":
            st["residual"] = torch.randn((m, n), device="cuda", generator=gen).to(torch.bfloat16)
        if case["epilogue"] == "gelu":
            st["bias"] = (torch.randn(n, device="cuda", generator=gen) * 0.1).to(torch.bfloat16)
        return st
    B, H, kv, dh, n = (case[x] for x in ("batch", "heads", "kv_heads", "dh", "max_len"))
    lens = torch.tensor(_lens(case, seed), dtype=torch.int32, device="cuda")
    st = dict(op=op, batch=B, heads=H, kv_heads=kv, dh=dh, lens=lens, lens1=lens + 1)
    st["qkv"] = torch.randn((B, (H + 2 * kv) * dh), device="cuda", generator=gen).to(torch.bfloat16)
    st["k"], st["ks"] = _cache(gen, B, kv, n, dh)
    st["v"], st["vs"] = _cache(gen, B, kv, n, dh)
    return st


# ------------------------------------------------------------------------------------------------- the definition in 64 bits
def _two_to(e):
    """2.0 ** e in float64 from its bits (the device's pow is off by an ulp for some whole e, which would move ties)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_exact(x):
    """Values that MXFP4 holds for x [R, K], straight from the definition: the nearest member of the scaled grid, the even code of two
    that are equally near."""
    R, K = x.shape
    out = torch.empty((R, K), dtype=torch.float64, device=x.device)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    mids = (grid[1:] + grid[:-1]) / 2                                   # between codes i and i + 1
    for r in range(0, R, 4096):
        b = x[r:r + 4096].double().reshape(-1, BLOCK)
        top = b.abs().max(dim=1, keepdim=True).values
        unit = _two_to((torch.frexp(top)[1] - 3).clamp(min=-127))           # floor(log2 top) - 2
        a = (b / unit).abs()
        code = torch.zeros_like(a, dtype=torch.int64)
        for i, mid in enumerate(mids.tolist()):
            code += (a > mid) | ((a == mid) & (i % 2 == 1))             # a tie goes up only from an odd code
        out[r:r + 4096] = (torch.copysign(grid[code], b) * unit).view(-1, K)
    return out


def _values_exact(codes, scales):
    lo, hi = (codes & 15).long(), (codes >> 4).long()
    c = torch.stack((lo, hi), -1).flatten(-2)
    grid = torch.tensor(GRID, dtype=torch.float64, device=codes.device)
    v = grid[c & 7] * (1.0 - 2.0 * (c >> 3).double())
    return v * _two_to(scales.int() - 127).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        return _round_exact(st["x"])
    if op in ("linear", "decode"):
        x = _round_exact(st["x"]) if op == "linear" else st["x"].double()
        y = x @ _values_exact(st["w"], st["ws"]).t()
        if case["epilogue"] == "gelu":
            y = y + st["bias"].double()
            y = y / (1 + torch.exp(-1.702 * y))
        return y + st["residual"].double() if case["epilogue"] == "residual" else y
    H, kv, dh = case["heads"], case["kv_heads"], case["dh"]
    out = torch.empty((case["batch"], H * dh), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case, seed)):
        row = st["qkv"][b].double().view(H + 2 * kv, dh)
        fresh = _round_exact(st["qkv"][b, H * dh:].view(2 * kv, dh))
        for h in range(kv):
            k = torch.cat((_values_exact(st["k"][b, h, :n], st["ks"][b, h, :n]), fresh[None, h]))
            v = torch.cat((_values_exact(st["v"][b, h, :n], st["vs"][b, h, :n]), fresh[None, kv + h]))
            for i in range(h * H // kv, (h + 1) * H // kv):
                p = torch.softmax(k @ row[i] / math.sqrt(dh), 0)
                out[b, i * dh:(i + 1) * dh] = p @ v
    return dict(out=out, k=None, ks=None, v=None, vs=None)
