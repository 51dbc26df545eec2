// out[M, N] = act(x[M, K] @ W[N, K]^T + bias) + residual for M <= 32, x in bf16 and W in MXFP4 (format: mxfp4.h): the projections of a
// decode step, whose cost is one read of W (17/32 bytes per element).
//
// W goes from global memory to registers and from there, de-quantised to bf16 (exact), straight into v_mfma_f32_16x16x32_bf16 as its first
// operand: lane (r = l & 15, q = l >> 4) holds one whole block of row r, 16 bytes of codes, consumed by four MFMAs of 8 k per lane
// against the same k of x.  A wave owns 16 rows of W and one K-slice of at most 1024 k: all of its 8 code loads and its one scale load
// are in flight before anything is consumed (8.5 KB per wave; there is no ring to keep filled).  A code load is issued in the coalesced
// order (lane = row l >> 2, 16-byte chunk l & 3) and turned into fragment order by ds_bpermute_b32 when it is consumed.  x is staged once
// per workgroup and slice in LDS.  K-slices are summed, in order, from fp32 slabs by a second small kernel with the epilogue.
#include "mxfp4.h"

namespace hvlm {
namespace {

constexpr int W4_WAVES = 8;               // 128 rows of W per workgroup
constexpr int W4_STEPS = 8;               // steps of 128 k per K-slice at most
constexpr int W4_XSTRIDE = W4_STEPS * 128 + 8;   // elements per x row in LDS: 16 bytes of padding put eight rows into eight bank groups

template <int HALVES>
__global__ __launch_bounds__(W4_WAVES * 64) void gemm_w4a16_kernel(const bf16_t* __restrict__ x, const unsigned char* __restrict__ W,
                                                                   const unsigned char* __restrict__ wsc, float* __restrict__ ws, int M, int N,
                                                                   int K, long ldx, long ldw, long ldws, int steps, int np) {
  extern __shared__ __attribute__((aligned(16))) bf16_t xs[];
  const int t = threadIdx.x, w = t >> 6, l = t & 63, r16 = l & 15, q = l >> 4;
  const int nblk = K / MX_BLOCK, b0 = blockIdx.y * steps * 4;               // first block of this slice
  const int nb = min(steps * 4, nblk - b0);                                  // its blocks
  const int n0 = blockIdx.x * (W4_WAVES * 16) + w * 16;

  const unsigned char* wp = W + (long)min(n0 + (l >> 2), N - 1) * ldw + (long)b0 * 16;
  u32x4 ring[W4_STEPS];
#pragma unroll
  for (int i = 0; i < W4_STEPS; ++i) ring[i] = *reinterpret_cast<const u32x4*>(wp + min(i * 4 + (l & 3), nb - 1) * 16);
  // scales: lane (r, q) takes bytes 8 q .. 8 q + 7 of row r's slice, the blocks of steps 2 q and 2 q + 1
  unsigned sc[2] = {0x7f7f7f7fu, 0x7f7f7f7fu};
  {
    const unsigned char* sp = wsc + (long)min(n0 + r16, N - 1) * ldws + b0;
    if (nb == W4_STEPS * 4) {
      __builtin_memcpy(sc, sp + 8 * q, 8);                                   // any alignment
    } else {
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const unsigned v = sp[min(8 * q + b, nb - 1)];
        sc[b >> 2] = (sc[b >> 2] & ~(255u << (8 * (b & 3)))) | (8 * q + b < nb ? v : 127u) << (8 * (b & 3));
      }
    }
  }

  // x slice -> LDS: rows 0 .. M - 1, zero past K (a block past K meets finite codes at scale 2^0)
  for (int m = w; m < M; m += W4_WAVES) {
    const bf16_t* xp = x + (long)m * ldx + (long)b0 * MX_BLOCK;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int c = l + 64 * u;
      u32x4 v = {0u, 0u, 0u, 0u};
      if (c < nb * 4) v = *reinterpret_cast<const u32x4*>(xp + c * 8);
      *reinterpret_cast<u32x4*>(xs + m * W4_XSTRIDE + c * 8) = v;
    }
  }
  __syncthreads();

  f32x4 acc[HALVES];
#pragma unroll
  for (int h = 0; h < HALVES; ++h) acc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int perm = (4 * r16 + q) << 2;                                       // fragment lane (r, q) <- load lane 4 r + q
  const bf16_t* xr[HALVES];                                                  // columns past M repeat the last row, their results are dropped
#pragma unroll
  for (int h = 0; h < HALVES; ++h) xr[h] = xs + min(h * 16 + r16, M - 1) * W4_XSTRIDE + q * 32;
#pragma unroll
  for (int i = 0; i < W4_STEPS; ++i) {
    if (i * 4 >= nb) break;
    const unsigned s4 = (unsigned)__builtin_amdgcn_ds_bpermute((r16 + 16 * (i >> 1)) << 2, (int)sc[i & 1]);
    const float s = mx_scale((s4 >> (8 * q)) & 255u);
    u32x4 c;
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = (unsigned)__builtin_amdgcn_ds_bpermute(perm, (int)ring[i][j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16x8 wf = mx_bf16x8(c[j], s);
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
        acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, *reinterpret_cast<const bf16x8*>(xr[h] + i * 128 + j * 8), acc[h], 0, 0, 0);
    }
  }

  // D: lane holds column m = r16 (+ 16), rows n0 + 4 q .. + 3 of W
  const int n = n0 + 4 * q;
  if (n < np) {
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      const int m = h * 16 + r16;
      if (m < M) *reinterpret_cast<f32x4*>(ws + ((long)blockIdx.y * M + m) * np + n) = acc[h];
    }
  }
}

__global__ __launch_bounds__(256) void w4a16_finalize_kernel(const float* __restrict__ ws, int splits, const bf16_t* __restrict__ bias,
                                                             const bf16_t* __restrict__ res, long ldr, int act, bf16_t* __restrict__ C,
                                                             long ldc, int M, int N, int np) {
  const int per_row = np / 4;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < M * per_row; i += gridDim.x * 256) {
    const int m = i / per_row, n = (i - m * per_row) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const f32x4*>(ws + ((long)s * M + m) * np + n);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (n + e >= N) break;
      float y = v[e] + (bias ? bf2f(bias[n + e]) : 0.f);
      if (act == HVLM_ACT_QUICK_GELU) y *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.702f * 1.4426950408889634f * y));
      C[(long)m * ldc + n + e] = f2bf(y + (res ? bf2f(res[(long)m * ldr + n + e]) : 0.f));
    }
  }
}

// steps per K-slice: long slices unless the launch would not put two workgroups on every CU
int w4_steps(int N, int K) {
  const int steps = (K / MX_BLOCK + 3) / 4, cols = cdiv(N, W4_WAVES * 16);
  int per = W4_STEPS;
  while (per > 2 && (long)cols * cdiv(steps, per) < 512) per -= 2;
  return per;
}
int w4_splits(int N, int K) { return cdiv((K / MX_BLOCK + 3) / 4, w4_steps(N, K)); }

}  // namespace
}  // namespace hvlm

using namespace hvlm;

extern "C" size_t hvlm_gemm_w4a16_ws_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K < MX_BLOCK) return 0;
  return (size_t)w4_splits(N, K) * M * ((size_t)(N + 3) / 4 * 4) * 4;
}

extern "C" int hvlm_gemm_w4a16_nt(const void* x, const void* W, const void* w_scale, void* C, int M, int N, int K, long ldx, long ldw, long ldws,
                                  long ldc, const void* bias, const void* residual, long ldr, int act, void* ws, void* stream) {
  HVLM_REQUIRE(x && W && w_scale && C && ws, "gemm_w4a16_nt: null pointer");
  HVLM_REQUIRE(M > 0 && M <= 32, "gemm_w4a16_nt: M must be 1 .. 32 (got %d)", M);
  HVLM_REQUIRE(N > 0 && N <= (1 << 24) && K > 0 && K % MX_BLOCK == 0, "gemm_w4a16_nt: N=%d must be positive, K=%d a positive multiple of 32", N, K);
  HVLM_REQUIRE(ldx >= K && ldx % 8 == 0 && ((uintptr_t)x & 15) == 0, "gemm_w4a16_nt: rows of x must be 16-byte aligned");
  HVLM_REQUIRE(ldw >= K / 2 && ldw % 16 == 0 && ((uintptr_t)W & 15) == 0, "gemm_w4a16_nt: rows of codes must be 16-byte aligned");
  HVLM_REQUIRE(ldws >= K / MX_BLOCK && ldc >= N && (!residual || ldr >= N), "gemm_w4a16_nt: leading dimensions");
  HVLM_REQUIRE(((uintptr_t)ws & 15) == 0, "gemm_w4a16_nt: the workspace must be 16-byte aligned");
  HVLM_REQUIRE(act == HVLM_ACT_NONE || act == HVLM_ACT_QUICK_GELU, "gemm_w4a16_nt: unknown act %d", act);
  const int steps = w4_steps(N, K), splits = w4_splits(N, K), np = (N + 3) / 4 * 4;
  HVLM_REQUIRE(splits < 65536, "gemm_w4a16_nt: K=%d is too long", K);
  const dim3 grid(cdiv(N, W4_WAVES * 16), splits), block(W4_WAVES * 64);
  constexpr int lds_max = 32 * W4_XSTRIDE * 2;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_w4a16_kernel<2>), hipFuncAttributeMaxDynamicSharedMemorySize, lds_max);
  if (attr != hipSuccess) { set_error("gemm_w4a16_nt: hipFuncSetAttribute: %s", hipGetErrorString(attr)); return HVLM_ERR_LAUNCH; }
  const auto k = M <= 16 ? gemm_w4a16_kernel<1> : gemm_w4a16_kernel<2>;
  hipLaunchKernelGGL(k, grid, block, (size_t)M * W4_XSTRIDE * 2, as_stream(stream), (const bf16_t*)x, (const unsigned char*)W,
                     (const unsigned char*)w_scale, (float*)ws, M, N, K, ldx, ldw, ldws, steps, np);
  const int rc = check_launch("gemm_w4a16_nt");
  if (rc) return rc;
  const long items = (long)M * (np / 4);
  hipLaunchKernelGGL(w4a16_finalize_kernel, dim3((unsigned)min(cdiv(items, 256), 2048)), dim3(256), 0, as_stream(stream), (const float*)ws, splits,
                     (const bf16_t*)bias, (const bf16_t*)residual, ldr, act, (bf16_t*)C, ldc, M, N, np);
  return check_launch("gemm_w4a16_nt");
}
