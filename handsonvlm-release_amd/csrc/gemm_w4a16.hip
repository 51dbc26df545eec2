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

// the blocks b0 .. b0 + nb - 1 (nb <= 32) of sixteen rows of W, as a wave holds them: codes in the coalesced order, scales eight bytes a lane
struct W4Slice {
  u32x4 ring[W4_STEPS];
  unsigned sc[2];
};
__device__ __forceinline__ void w4_load(W4Slice& f, const unsigned char* __restrict__ W, const unsigned char* __restrict__ wsc, long ldw, long ldws, int n0, int N,
                                        int b0, int nb, int l) {
  const int r16 = l & 15, q = l >> 4;
  const unsigned char* wp = W + (long)min(n0 + (l >> 2), N - 1) * ldw + (long)b0 * 16;
#pragma unroll
  for (int i = 0; i < W4_STEPS; ++i) {
    if (i * 4 >= nb) break;
    f.ring[i] = *reinterpret_cast<const u32x4*>(wp + min(i * 4 + (l & 3), nb - 1) * 16);
  }
  // scales: lane (r, q) takes bytes 8 q .. 8 q + 7 of row r's slice, the blocks of steps 2 q and 2 q + 1; past the end 2^0 (x is zero there)
  const unsigned char* sp = wsc + (long)min(n0 + r16, N - 1) * ldws + b0 + 8 * q;
  const int mine = nb - 8 * q;
  f.sc[0] = f.sc[1] = 0x7f7f7f7fu;
  if (mine >= 8) __builtin_memcpy(f.sc, sp, 8);                                // any alignment
  else if (mine >= 4) __builtin_memcpy(f.sc, sp, 4);
#pragma unroll
  for (int b = 0; b < 7; ++b)
    if (mine < 8 && b >= (mine & ~3) && b < mine) f.sc[b >> 2] = (f.sc[b >> 2] & ~(255u << (8 * (b & 3)))) | (unsigned)sp[b] << (8 * (b & 3));
}
// acc[h] += the slice times x: xr[h] points at this lane's 32 k of step 0 of its row of x
template <int HALVES>
__device__ __forceinline__ void w4_product(const W4Slice& f, const bf16_t* const (&xr)[HALVES], f32x4 (&acc)[HALVES], int nb, int l) {
  const int r16 = l & 15, q = l >> 4, perm = (4 * r16 + q) << 2;               // fragment lane (r, q) <- load lane 4 r + q
#pragma unroll
  for (int i = 0; i < W4_STEPS; ++i) {
    if (i * 4 >= nb) break;
    const unsigned s4 = (unsigned)__builtin_amdgcn_ds_bpermute((r16 + 16 * (i >> 1)) << 2, (int)f.sc[i & 1]);
    const float s = mx_scale((s4 >> (8 * q)) & 255u);
    u32x4 c;
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = (unsigned)__builtin_amdgcn_ds_bpermute(perm, (int)f.ring[i][j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16x8 wf = mx_bf16x8(c[j], s);
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
        acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, *reinterpret_cast<const bf16x8*>(xr[h] + i * 128 + j * 8), acc[h], 0, 0, 0);
    }
  }
}

// TILES: 16-row tiles of W per wave that share what the workgroup stages of x
template <int HALVES, int TILES>
__global__ __launch_bounds__(W4_WAVES * 64) void gemm_w4a16_kernel(const bf16_t* __restrict__ x, const unsigned char* __restrict__ W,
                                                                   const unsigned char* __restrict__ wsc, float* __restrict__ ws, int M, int N,
                                                                   int K, long ldx, long ldw, long ldws, int steps, int np) {
  extern __shared__ __attribute__((aligned(16))) bf16_t xs[];
  const int t = threadIdx.x, w = t >> 6, l = t & 63, r16 = l & 15, q = l >> 4;
  const int nblk = K / MX_BLOCK, b0 = blockIdx.y * steps * 4;               // first block of this slice
  const int nb = min(steps * 4, nblk - b0);                                  // its blocks
  const int n0 = (blockIdx.x * W4_WAVES + w) * 16 * TILES;

  W4Slice f[TILES];
#pragma unroll
  for (int i = 0; i < TILES; ++i) w4_load(f[i], W, wsc, ldw, ldws, n0 + 16 * i, N, b0, nb, l);

  // x slice -> LDS: rows 0 .. M - 1, zero past K
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

  const bf16_t* xr[HALVES];                                                  // columns past M repeat the last row, their results are dropped
#pragma unroll
  for (int h = 0; h < HALVES; ++h) xr[h] = xs + min(h * 16 + r16, M - 1) * W4_XSTRIDE + q * 32;
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    f32x4 acc[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) acc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
    w4_product<HALVES>(f[i], xr, acc, nb, l);
    // D: lane holds column m = r16 (+ 16), rows 4 q .. + 3 of the tile
    const int n = n0 + 16 * i + 4 * q;
    if (n < np) {
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        const int m = h * 16 + r16;
        if (m < M) *reinterpret_cast<f32x4*>(ws + ((long)blockIdx.y * M + m) * np + n) = acc[h];
      }
    }
  }
}

__device__ __forceinline__ bf16_t w4_finish(float y, const bf16_t* bias, const bf16_t* res, long ldr, int act, int m, int n) {
  if (bias) y += bf2f(bias[n]);
  if (act == HVLM_ACT_QUICK_GELU) y *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.702f * 1.4426950408889634f * y));
  if (res) y += bf2f(res[(long)m * ldr + n]);
  return f2bf(y);
}

__global__ __launch_bounds__(256) void w4a16_finalize_kernel(const float* __restrict__ ws, int splits, const bf16_t* __restrict__ bias,
                                                             const bf16_t* __restrict__ res, long ldr, int act, bf16_t* __restrict__ C,
                                                             long ldc, int M, int N, int np) {
  const int per_row = np / 4;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < M * per_row; i += gridDim.x * 256) {
    const int m = i / per_row, n = (i - m * per_row) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < splits; s0 += 8) {                                   // eight slabs' loads at a time
      f32x4 a[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) a[s] = *reinterpret_cast<const f32x4*>(ws + ((long)min(s0 + s, splits - 1) * M + m) * np + n);
#pragma unroll
      for (int s = 0; s < 8; ++s) if (s0 + s < splits) v += a[s];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < N) C[(long)m * ldc + n + e] = w4_finish(v[e], bias, res, ldr, act, m, n + e);
  }
}

// How many tiles a wave, how long a K-slice
struct W4Plan {
  int tiles, steps, splits;
};
W4Plan w4_plan(int N, int K) {
  const int total = (K / MX_BLOCK + 3) / 4;
  W4Plan r{1, W4_STEPS, 0};
  // two tiles a wave halve what is staged of x per byte of W, as long as two workgroups are left for every CU; then long slices, likewise
  if ((long)cdiv(N, W4_WAVES * 32) * cdiv(total, W4_STEPS) >= 512) r.tiles = 2;
  while (r.steps > 2 && (long)cdiv(N, W4_WAVES * 16 * r.tiles) * cdiv(total, r.steps) < 512) r.steps -= 2;
  r.splits = cdiv(total, r.steps);
  return r;
}

}  // namespace
}  // namespace hvlm

using namespace hvlm;

extern "C" size_t hvlm_gemm_w4a16_ws_bytes(int M, int N, int K) {
  if (M <= 0 || M > 32 || N <= 0 || K < MX_BLOCK) return 0;
  return (size_t)w4_plan(N, K).splits * M * ((size_t)(N + 3) / 4 * 4) * 4;
}

extern "C" int hvlm_gemm_w4a16_nt(const void* x, const void* W, const void* w_scale, void* C, int M, int N, int K, long ldx, long ldw, long ldws,
                                  long ldc, const void* bias, const void* residual, long ldr, int act, void* ws, void* stream) {
  HVLM_REQUIRE(x && W && w_scale && C && ws, "gemm_w4a16_nt: null pointer");
  HVLM_REQUIRE(M > 0 && M <= 32, "gemm_w4a16_nt: M must be 1 .. 32 (got %d)", M);
  HVLM_REQUIRE(N > 0 && N <= (1 << 24) && K > 0 && K % MX_BLOCK == 0, "gemm_w4a16_nt: N=%d must be positive, K=%d a positive multiple of 32", N, K);
  HVLM_REQUIRE(ldx >= K && ldx % 8 == 0 && ((uintptr_t)x & 15) == 0, "gemm_w4a16_nt: rows of x must be 16-byte aligned");
  HVLM_REQUIRE(ldw >= K / 2 && ldw % 16 == 0 && ((uintptr_t)W & 15) == 0, "gemm_w4a16_nt: rows of codes must be 16-byte aligned");
  HVLM_REQUIRE(ldws >= K / MX_BLOCK && ldc >= N && (!residual || ldr >= N), "gemm_w4a16_nt: leading dimensions");
  HVLM_REQUIRE(act == HVLM_ACT_NONE || act == HVLM_ACT_QUICK_GELU, "gemm_w4a16_nt: unknown act %d", act);
  const W4Plan plan = w4_plan(N, K);
  const dim3 block(W4_WAVES * 64);
  HVLM_REQUIRE(((uintptr_t)ws & 15) == 0, "gemm_w4a16_nt: a 16-byte aligned workspace of hvlm_gemm_w4a16_ws_bytes() is needed");
  HVLM_REQUIRE(plan.splits < 65536, "gemm_w4a16_nt: K=%d is too long", K);
  const int np = (N + 3) / 4 * 4;
  const dim3 grid(cdiv(N, W4_WAVES * 16 * plan.tiles), plan.splits);
  constexpr int lds_max = 32 * W4_XSTRIDE * 2;
  const auto set = [](const void* k) { return hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, lds_max); };
  static const hipError_t a1 = set(reinterpret_cast<const void*>(gemm_w4a16_kernel<2, 1>)), a2 = set(reinterpret_cast<const void*>(gemm_w4a16_kernel<2, 2>));
  if (a1 != hipSuccess || a2 != hipSuccess) { set_error("gemm_w4a16_nt: hipFuncSetAttribute: %s", hipGetErrorString(a1 != hipSuccess ? a1 : a2)); return HVLM_ERR_LAUNCH; }
  const auto k = M <= 16 ? (plan.tiles == 1 ? gemm_w4a16_kernel<1, 1> : gemm_w4a16_kernel<1, 2>) : (plan.tiles == 1 ? gemm_w4a16_kernel<2, 1> : gemm_w4a16_kernel<2, 2>);
  hipLaunchKernelGGL(k, grid, block, (size_t)M * W4_XSTRIDE * 2, as_stream(stream), (const bf16_t*)x, (const unsigned char*)W,
                     (const unsigned char*)w_scale, (float*)ws, M, N, K, ldx, ldw, ldws, plan.steps, np);
  const int rc = check_launch("gemm_w4a16_nt");
  if (rc) return rc;
  const long items = (long)M * (np / 4);
  hipLaunchKernelGGL(w4a16_finalize_kernel, dim3((unsigned)min(cdiv(items, 256), 2048)), dim3(256), 0, as_stream(stream), (const float*)ws, plan.splits,
                     (const bf16_t*)bias, (const bf16_t*)residual, ldr, act, (bf16_t*)C, ldc, M, N, np);
  return check_launch("gemm_w4a16_nt");
}
