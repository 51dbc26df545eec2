// MXFP4 quantisation and de-quantisation of row-major matrices (format: mxfp4.h).
//
// Both are streams: 2 bytes in and 17/32 bytes out per element, or the reverse.  A lane owns 16 bytes of 16-bit elements, so a wave reads
// (or writes) 1 KB in one instruction; the four lanes of a block find its maximum with two DPP steps, no LDS.
#include "mxfp4.h"

namespace hvlm {
namespace {

constexpr int MXQ_THREADS = 256;

template <bool F16>
__global__ __launch_bounds__(MXQ_THREADS) void quantize_mxfp4_kernel(const bf16_t* __restrict__ x, unsigned char* __restrict__ codes,
                                                                     unsigned char* __restrict__ scales, unsigned chunks, unsigned cpr,
                                                                     long ldx, long ldc, long lds) {
  for (unsigned i = blockIdx.x * MXQ_THREADS + threadIdx.x; i < chunks; i += gridDim.x * MXQ_THREADS) {
    const unsigned row = i / cpr, c = i - row * cpr;                      // chunk = 8 elements; cpr is a multiple of 4: a quad is one block
    const u32x4 v = *reinterpret_cast<const u32x4*>(x + row * ldx + c * 8L);
    const unsigned s = mx_scale_code<F16>(mx_quad_max(mx_amax8(v)));
    *reinterpret_cast<unsigned*>(codes + row * ldc + c * 4L) = mx_quant8<F16>(v, s);
    if ((c & 3) == 0) scales[row * lds + (c >> 2)] = (unsigned char)s;
  }
}

template <bool F16>
__global__ __launch_bounds__(MXQ_THREADS) void dequantize_mxfp4_kernel(const unsigned char* __restrict__ codes,
                                                                       const unsigned char* __restrict__ scales, bf16_t* __restrict__ out,
                                                                       unsigned chunks, unsigned cpr, long ldc, long lds, long ldo) {
  for (unsigned i = blockIdx.x * MXQ_THREADS + threadIdx.x; i < chunks; i += gridDim.x * MXQ_THREADS) {
    const unsigned row = i / cpr, c = i - row * cpr;
    const unsigned w = *reinterpret_cast<const unsigned*>(codes + row * ldc + c * 4L);
    const float sc = mx_scale(scales[row * lds + (c >> 2)]);
    u32x4 r;
    if constexpr (F16) {
      r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 0));
      r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 1));
      r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 2));
      r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 3));
    } else {
      r = __builtin_bit_cast(u32x4, mx_bf16x8(w, sc));
    }
    *reinterpret_cast<u32x4*>(out + row * ldo + c * 8L) = r;
  }
}

}  // namespace
}  // namespace hvlm

using namespace hvlm;

static int mx_grid(long chunks) {
  const long g = (chunks + MXQ_THREADS - 1) / MXQ_THREADS;
  return (int)(g < 8192 ? g : 8192);
}

static int mx_check(const char* what, const void* x, const void* codes, const void* scales, int rows, int K, long ldx, long ldc, long lds, int f16) {
  HVLM_REQUIRE(x && codes && scales, "%s: null pointer", what);
  HVLM_REQUIRE(rows > 0 && K > 0 && K % MX_BLOCK == 0, "%s: rows=%d must be positive, K=%d a positive multiple of 32", what, rows, K);
  HVLM_REQUIRE((long)rows * (K / 8) < (1L << 31), "%s: %d x %d elements are too many for one call", what, rows, K);
  HVLM_REQUIRE(ldx >= K && ldx % 8 == 0 && ((uintptr_t)x & 15) == 0, "%s: rows of the 16-bit matrix must be 16-byte aligned", what);
  HVLM_REQUIRE(ldc >= K / 2 && ldc % 4 == 0 && ((uintptr_t)codes & 3) == 0, "%s: rows of codes must be 4-byte aligned", what);
  HVLM_REQUIRE(lds >= K / MX_BLOCK, "%s: leading dimension of the scales", what);
  HVLM_REQUIRE(f16 == 0 || f16 == 1, "%s: f16 must be 0 or 1", what);
  return HVLM_OK;
}

extern "C" int hvlm_quantize_mxfp4(const void* x, void* codes, void* scales, int rows, int K, long ldx, long ld_codes, long ld_scales, int f16,
                                   void* stream) {
  const int rc = mx_check("quantize_mxfp4", x, codes, scales, rows, K, ldx, ld_codes, ld_scales, f16);
  if (rc) return rc;
  const long chunks = (long)rows * (K / 8);
  const auto k = f16 ? quantize_mxfp4_kernel<true> : quantize_mxfp4_kernel<false>;
  hipLaunchKernelGGL(k, dim3(mx_grid(chunks)), dim3(MXQ_THREADS), 0, as_stream(stream), (const bf16_t*)x, (unsigned char*)codes,
                     (unsigned char*)scales, (unsigned)chunks, (unsigned)(K / 8), ldx, ld_codes, ld_scales);
  return check_launch("quantize_mxfp4");
}

extern "C" int hvlm_dequantize_mxfp4(const void* codes, const void* scales, void* out, int rows, int K, long ld_codes, long ld_scales, long ldo,
                                     int f16, void* stream) {
  const int rc = mx_check("dequantize_mxfp4", out, codes, scales, rows, K, ldo, ld_codes, ld_scales, f16);
  if (rc) return rc;
  const long chunks = (long)rows * (K / 8);
  const auto k = f16 ? dequantize_mxfp4_kernel<true> : dequantize_mxfp4_kernel<false>;
  hipLaunchKernelGGL(k, dim3(mx_grid(chunks)), dim3(MXQ_THREADS), 0, as_stream(stream), (const unsigned char*)codes,
                     (const unsigned char*)scales, (bf16_t*)out, (unsigned)chunks, (unsigned)(K / 8), ld_codes, ld_scales, ldo);
  return check_launch("dequantize_mxfp4");
}
