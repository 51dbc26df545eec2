"""4-bit operators without a GPU: the definition the GPU tests compare with, and every refusal (all are raised before a launch)."""
import ctypes

import pytest
import torch

import mx_ref

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from hvlm import _lib, ops
    _lib.load()
    return ops


def pair(R, K):
    return torch.zeros(R, K // 2, dtype=torch.uint8), torch.full((R, K // 32), 127, dtype=torch.uint8)


def test_definition_by_hand():
    x = torch.zeros(1, 32)
    x[0, :12] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.2, -0.3, 7.9, -1.0])
    codes, scales = mx_ref.quantise(x)
    assert scales.item() == 127                                              # floor(log2 7.9) - 2 = 0
    c = torch.stack((codes & 15, codes >> 4), -1).flatten().tolist()
    assert c[:12] == [7, 0, 2, 2, 4, 4, 6, 6, 8, 9, 7, 10]                    # ties to the even code, 7.9 saturates, -0.2 keeps its sign
    v = mx_ref.values((codes, scales))[0, :12].tolist()
    assert v == [6, 0, 1, 1, 2, 2, 4, 4, 0, -0.5, 6, -1]
    x[0, 3] = float("inf")
    codes, scales = mx_ref.quantise(x)
    assert scales.item() == 255 and int(codes.sum()) == 0 and torch.isnan(mx_ref.values((codes, scales))).all()


@pytest.mark.parametrize("K", [32, 256])
def test_definition_error_bound(K):
    """Half a step of the block's own grid for every element that does not saturate; a quarter of its size for those that do."""
    x = torch.randn(64, K, generator=torch.Generator().manual_seed(K), dtype=torch.float64)
    c, s = mx_ref.quantise(x)
    unit = mx_ref.two_to(s.int() - 127).repeat_interleave(32, -1)
    err, a = (mx_ref.values((c, s)) - x).abs(), x.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)) * unit
    assert (err <= torch.where(a <= 6, step / 2, x.abs() / 4)).all()


def refused(fn, *words):
    from hvlm import _lib
    with pytest.raises(_lib.HvlmError) as e:
        fn()
    assert all(w in str(e.value) for w in words), str(e.value)


def test_wrapper_refusals(ops):
    x = torch.zeros(4, 64, dtype=BF16)
    refused(lambda: ops.quantize_mxfp4(x.float()), "bf16 or fp16")
    refused(lambda: ops.quantize_mxfp4(x[:, :48]), "multiple of 32")
    refused(lambda: ops.quantize_mxfp4(x.t()), "contiguous rows")
    refused(lambda: ops.quantize_mxfp4(x[:0]), "positive")
    refused(lambda: ops.quantize_mxfp4(x, out=pair(4, 32)), "out is for")
    refused(lambda: ops.quantize_mxfp4(x), "current device")
    refused(lambda: ops.dequantize_mxfp4(pair(4, 64), out_dtype=torch.float32), "bf16 or fp16")
    refused(lambda: ops.dequantize_mxfp4((torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 3, dtype=torch.uint8))), "MXFP4 matrix")
    refused(lambda: ops.dequantize_mxfp4(pair(4, 64)), "current device")
    refused(lambda: ops.gemm_mxfp4_nt(pair(4, 64), pair(4, 96)), "K=64", "K=96")
    refused(lambda: ops.gemm_mxfp4_nt(pair(4, 64), pair(5, 64), bias=torch.zeros(4, dtype=BF16)), "bias")
    refused(lambda: ops.gemm_mxfp4_nt(pair(4, 64), pair(5, 64), residual=torch.zeros(5, 4, dtype=BF16)), "residual")
    refused(lambda: ops.gemm_mxfp4_nt(pair(4, 64), pair(5, 64), out=torch.zeros(4, 5, dtype=torch.float16)), "out must be")
    refused(lambda: ops.gemm_mxfp4_nt(pair(4, 64), pair(5, 64)), "current device")
    refused(lambda: ops.gemm_w4a16_nt(x.float(), pair(5, 64)), "a")
    refused(lambda: ops.gemm_w4a16_nt(x, pair(5, 64)), "current device")


def test_cache_refusals(ops):
    c = ops.KV4Cache.empty(2, 8, 2, 64, "cpu")
    assert c.checked("t") == (2, 2, 8, 64) and c.k.shape == (2, 2, 8, 32) and c.v_scale.shape == (2, 2, 8, 2)
    refused(lambda: c._replace(v=c.v[:, :, :4]).checked("t"), "dense")
    refused(lambda: c._replace(v=c.v[:, :, :4].contiguous()).checked("t"), "shapes")
    refused(lambda: c._replace(k_scale=c.k_scale.float()).checked("t"), "uint8")
    refused(lambda: ops.kv4_append(torch.zeros(2, 6 * 64, dtype=BF16), c, None, 2), "current device")
    refused(lambda: ops.attn_decode_kv4(torch.zeros(2, 128, dtype=BF16), c, torch.zeros(2, dtype=torch.int32), 2, 0.1), "current device")


def test_c_refusals(ops):
    """The C entry points check what they are given before they touch the device (the pointers here are never dereferenced)."""
    from hvlm import _lib
    lib = _lib.load()
    p, odd, N = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 2), None

    def bad(rc, *words):
        assert rc == -1 and all(w in _lib.last_error() for w in words), (rc, _lib.last_error())

    bad(lib.hvlm_quantize_mxfp4(N, p, p, 1, 32, 32, 16, 1, 0, N), "null")
    bad(lib.hvlm_quantize_mxfp4(p, p, p, 0, 32, 32, 16, 1, 0, N), "positive")
    bad(lib.hvlm_quantize_mxfp4(p, p, p, 1, 48, 48, 24, 2, 0, N), "multiple of 32")
    bad(lib.hvlm_quantize_mxfp4(odd, p, p, 1, 32, 32, 16, 1, 0, N), "16-byte")
    bad(lib.hvlm_quantize_mxfp4(p, p, p, 1, 32, 36, 16, 1, 0, N), "16-byte")
    bad(lib.hvlm_quantize_mxfp4(p, odd, p, 1, 32, 32, 16, 1, 0, N), "4-byte")
    bad(lib.hvlm_quantize_mxfp4(p, p, p, 1, 64, 64, 32, 1, 0, N), "scales")
    bad(lib.hvlm_quantize_mxfp4(p, p, p, 1 << 30, 32, 32, 16, 1, 0, N), "too many")
    bad(lib.hvlm_quantize_mxfp4(p, p, p, 1, 32, 32, 16, 1, 2, N), "f16")
    bad(lib.hvlm_dequantize_mxfp4(p, p, p, 1, 32, 8, 1, 32, 0, N), "codes")
    gm = lambda A=p, M=1, N_=1, K=32, lda=16, ldas=1, ldc=1, res=N, ldr=0, act=0, C=p, ws=p: lib.hvlm_gemm_mxfp4_nt(  # noqa: E731
        A, p, p, p, C, M, N_, K, lda, ldas, 16 * (K // 32), K // 32, ldc, N, res, ldr, act, 0, ws, N)
    bad(gm(A=N), "null")
    bad(gm(M=0), "positive")
    bad(gm(K=16), "multiple of 32")
    bad(gm(lda=24), "16-byte")
    bad(gm(A=odd), "16-byte")
    bad(gm(lda=1 << 22), "4 MiB")
    bad(gm(ldas=0), "scales")
    bad(gm(N_=3), "leading dimensions of C")
    bad(gm(res=p), "leading dimensions of C")
    bad(gm(act=7), "act")
    bad(gm(ws=N), "null")
    bad(gm(ws=odd), "workspace")
    assert lib.hvlm_gemm_mxfp4_ws_bytes(0, 4, 32) == 0 and lib.hvlm_gemm_mxfp4_ws_bytes(867, 4096, 4096) == (7 + 32) * 2 * 32 * 256
    sk = lambda M=1, K=32, ldx=32, ws=p, x=p: lib.hvlm_gemm_w4a16_nt(x, p, p, p, M, 4, K, ldx, 16 * (K // 32), K // 32, 4, N, N, 0, 0, ws, N)  # noqa: E731
    bad(sk(x=N), "null")
    bad(sk(M=5, ws=N), "workspace")
    bad(sk(K=14368, ldx=14368, ws=N), "workspace")
    bad(sk(M=33), "1 .. 32")
    bad(sk(M=0), "1 .. 32")
    bad(sk(K=40, ldx=40), "multiple of 32")
    bad(sk(x=odd), "16-byte")
    bad(sk(M=5, ws=odd), "workspace")
    ap = lambda ld=192, B=1, S=1, n=4, H=1, dh=64, q=p, kc=p: lib.hvlm_kv4_append(q, ld, kc, p, p, p, N, N, B, S, n, H, 1, dh, N)  # noqa: E731
    bad(ap(q=N), "null")
    bad(ap(kc=N), "null")
    bad(ap(kc=odd), "16-byte")
    bad(ap(ld=191), "16-byte")
    bad(ap(ld=128), "rows")
    bad(ap(dh=96), "head dimension")
    bad(ap(S=0), "S=0")
    bad(ap(B=0), "positive")
    at = lambda H=1, Hkv=1, ldq=64, lens=p, ws=p, n=4, ldo=64, dh=64: lib.hvlm_attn_decode_kv4(p, ldq, p, p, p, p, lens, p, ldo, 1, n, H, Hkv, dh, 0.1, ws, N)  # noqa: E731
    bad(at(lens=N), "null")
    bad(at(H=3, Hkv=2), "times")
    bad(at(H=17), "times")
    bad(at(ldq=32), "16-byte")
    bad(at(ldo=32), "out")
    bad(at(n=0), "positive")
    bad(at(n=100000, ws=N), "workspace")
    for dh, off in ((128, 1), (128, 2), (64, 1)):                               # scales that a row's bytes straddle
        s = ctypes.c_void_p((1 << 20) + off)
        bad(lib.hvlm_kv4_append(p, 3 * dh, p, s, p, p, N, N, 1, 1, 4, 1, 1, dh, N), "scales must be aligned")
        bad(lib.hvlm_attn_decode_kv4(p, dh, p, p, p, s, p, p, dh, 1, 4, 1, 1, dh, 0.1, p, N), "scales must be aligned")
    assert lib.hvlm_attn_decode_kv4_ws_bytes(64, 32, 32, 128, 1000) == 0 and lib.hvlm_attn_decode_kv4_ws_bytes(1, 32, 32, 128, 1000) == 0
    assert lib.hvlm_attn_decode_kv4_ws_bytes(1, 32, 32, 128, 1025) == 32 * 9 * 130 * 4
    assert lib.hvlm_attn_decode_kv4_ws_bytes(0, 32, 32, 128, 1000) == 0 and lib.hvlm_gemm_w4a16_ws_bytes(0, 4, 32) == 0
    assert lib.hvlm_gemm_w4a16_ws_bytes(4, 5, 4096) == 0 and lib.hvlm_gemm_w4a16_ws_bytes(1, 5, 14336) == 0 and lib.hvlm_gemm_w4a16_ws_bytes(5, 5, 32) == 5 * 8 * 4
