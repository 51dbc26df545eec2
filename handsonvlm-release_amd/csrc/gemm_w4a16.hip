// out[M, N] = act(x[M, K] @ W[N, K]^T + bias) + residual for M <= 32, x in bf16 and W in MXFP4 (format: mxfp4.h): the projections of a
// decode step, whose cost is one read of W (17/32 bytes per element).
//
// W goes from global memory to registers and from there, de-quantised to bf16 (exact), straight into v_mfma_f32_16x16x32_bf16 as its first
// operand: lane (r = l & 15, q = l >> 4) holds one whole block of row r, 16 bytes of codes, consumed by four MFMAs of 8 k per lane
// against the same k of x.  A wave owns 16 rows of W (or 32) and one K-slice of at most 1024 k: all of its code loads and scale loads are in
// flight before anything is consumed (8.5 KB per 16 rows; there is no ring to keep filled).  A code load is issued in the coalesced order
// (lane = row l >> 2, 16-byte chunk l & 3) and turned into fragment order by ds_bpermute_b32 when it is consumed.  x is staged once per
// workgroup and slice in LDS.  K-slices are summed, in order, from fp32 slabs by a second small kernel with the epilogue; with one to four rows
// of x the slices are the waves of one workgroup and no second kernel runs.
//
// Bound by the read of W where W is large: 22016 x 4096 at one row 12.3 us (3.9 TB/s; a copy's rate would take 10.0 us),
// 32101 x 4096 at 32 rows 26.3 us + 4.8 us for the slabs (15.1 us; there the staging of x, half as many bytes again from L2, and the slabs, 16 MB, come on top).
#include "mxfp4.h"

namespace hvlm {
namespace {

constexpr int W4_WAVES = 8;               // 128 or 256 rows of W per workgroup
constexpr int W4_STEPS = 8;               // steps of 128 k per K-slice at most
constexpr int W4_XSTRIDE = W4_STEPS * 128 + 8;   // elements per x row in LDS: 16 bytes of padding put eight rows into eight bank groups

// the blocks b0 .. b0 + nb - 1 (nb <= 32) of sixteen rows of W, as a wave holds them: codes in the coalesced order, scales eight bytes a lane
template <int STEPS>
struct W4Slice {
  u32x4 ring[STEPS];
  unsigned sc[2];
};
template <int STEPS>
__device__ __forceinline__ void w4_load(W4Slice<STEPS>& f, const unsigned char* __restrict__ W, const unsigned char* __restrict__ wsc, long ldw, long ldws, int n0, int N,
                                        int b0, int nb, int l) {
  const int r16 = l & 15, q = l >> 4;
  const unsigned char* wp = W + (long)min(n0 + (l >> 2), N - 1) * ldw + (long)b0 * 16;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
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
// acc[t][h] += the slices times x: xr[h] points at this lane's 32 k of step 0 of its row of x, whose fragments the tiles share
template <int STEPS, int HALVES, int TILES>
__device__ __forceinline__ void w4_product(const W4Slice<STEPS> (&f)[TILES], const bf16_t* const (&xr)[HALVES], f32x4 (&acc)[TILES][HALVES], int nb, int l) {
  const int r16 = l & 15, q = l >> 4, perm = (4 * r16 + q) << 2;               // fragment lane (r, q) <- load lane 4 r + q
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    if (i * 4 >= nb) break;
    float s[TILES];
    u32x4 c[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const unsigned s4 = (unsigned)__builtin_amdgcn_ds_bpermute((r16 + 16 * (i >> 1)) << 2, (int)f[t].sc[i & 1]);
      s[t] = mx_scale((s4 >> (8 * q)) & 255u);
#pragma unroll
      for (int j = 0; j < 4; ++j) c[t][j] = (unsigned)__builtin_amdgcn_ds_bpermute(perm, (int)f[t].ring[i][j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bf16x8 xf[HALVES];
#pragma unroll
      for (int h = 0; h < HALVES; ++h) xf[h] = *reinterpret_cast<const bf16x8*>(xr[h] + i * 128 + j * 8);
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        const bf16x8 wf = mx_bf16x8(c[t][j], s[t]);
#pragma unroll
        for (int h = 0; h < HALVES; ++h) acc[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[h], acc[t][h], 0, 0, 0);
      }
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

  W4Slice<W4_STEPS> f[TILES];
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
  f32x4 acc[TILES][HALVES];
#pragma unroll
  for (int i = 0; i < TILES; ++i)
#pragma unroll
    for (int h = 0; h < HALVES; ++h) acc[i][h] = f32x4{0.f, 0.f, 0.f, 0.f};
  w4_product<W4_STEPS, HALVES, TILES>(f, xr, acc, nb, l);
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    // D: lane holds column m = r16 (+ 16), rows 4 q .. + 3 of the tile
    const int n = n0 + 16 * i + 4 * q;
    if (n < np) {
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        const int m = h * 16 + r16;
        if (m < M) *reinterpret_cast<f32x4*>(ws + ((long)blockIdx.y * M + m) * np + n) = acc[i][h];
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

// A few rows of x, all of them in LDS: the waves of a workgroup share sixteen rows of W, at most STEPS steps of K each, and add up in LDS, in order; no
// slabs, no second kernel.  At most 64 registers, so that a CU holds 32 waves.  The body is a __device__ template under plain kernels.
constexpr int W4_ROWS = 4;
template <int WAVES, int STEPS>
__device__ __forceinline__ void gemm_w4a16_rows_body(const bf16_t* __restrict__ x, const unsigned char* __restrict__ W, const unsigned char* __restrict__ wsc,
                                                     const bf16_t* __restrict__ bias, const bf16_t* __restrict__ res, bf16_t* __restrict__ C, int M, int N,
                                                     int K, long ldx, long ldw, long ldws, long ldc, long ldr, int act, int per, int xstride) {
  extern __shared__ __attribute__((aligned(16))) bf16_t xs[];
  const int t = threadIdx.x, w = t >> 6, l = t & 63, r16 = l & 15, q = l >> 4;
  const int nblk = K / MX_BLOCK, b0 = min(w * per * 4, nblk), nb = min(per * 4, nblk - b0);      // this wave's blocks, perhaps none
  const int n0 = blockIdx.x * 16;
  W4Slice<STEPS> f[1];
  if (nb > 0) w4_load(f[0], W, wsc, ldw, ldws, n0, N, b0, nb, l);
  // x -> LDS: rows 0 .. M - 1, zero from K to the end of its last step
  const int ends = (nblk + 3) / 4 * 16;                                      // chunks of eight
  for (int m = 0; m < M; ++m)
    for (int c = t; c < ends; c += WAVES * 64) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (c < K / 8) v = *reinterpret_cast<const u32x4*>(x + (long)m * ldx + c * 8);
      *reinterpret_cast<u32x4*>(xs + m * xstride + c * 8) = v;
    }
  __syncthreads();
  f32x4 acc[1][1] = {{f32x4{0.f, 0.f, 0.f, 0.f}}};
  if (nb > 0) {
    const bf16_t* const xr[1] = {xs + min(r16, M - 1) * xstride + b0 * MX_BLOCK + q * 32};
    w4_product<STEPS, 1, 1>(f, xr, acc, nb, l);
  }
  __syncthreads();                                                           // x is read; its room takes the partial sums [wave][m][16]
  float* red = reinterpret_cast<float*>(xs);
  if (r16 < M) *reinterpret_cast<f32x4*>(red + (w * M + r16) * 16 + 4 * q) = acc[0][0];
  __syncthreads();
  if (t < 16 * M) {
    const int m = t >> 4, n = n0 + (t & 15);
    float y = 0.f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) y += red[(v * M + m) * 16 + (t & 15)];
    if (n < N) C[(long)m * ldc + n] = w4_finish(y, bias, res, ldr, act, m, n);
  }
}

__global__ __launch_bounds__(512, 8) void gemm_w4a16_rows_8_kernel(const bf16_t* __restrict__ x, const unsigned char* __restrict__ W,
                                                                   const unsigned char* __restrict__ wsc, const bf16_t* __restrict__ bias,
                                                                   const bf16_t* __restrict__ res, bf16_t* __restrict__ C, int M, int N, int K, long ldx,
                                                                   long ldw, long ldws, long ldc, long ldr, int act, int per, int xstride) {
  gemm_w4a16_rows_body<8, 4>(x, W, wsc, bias, res, C, M, N, K, ldx, ldw, ldws, ldc, ldr, act, per, xstride);
}
__global__ __launch_bounds__(1024, 8) void gemm_w4a16_rows_16_kernel(const bf16_t* __restrict__ x, const unsigned char* __restrict__ W,
                                                                     const unsigned char* __restrict__ wsc, const bf16_t* __restrict__ bias,
                                                                     const bf16_t* __restrict__ res, bf16_t* __restrict__ C, int M, int N, int K, long ldx,
                                                                     long ldw, long ldws, long ldc, long ldr, int act, int per, int xstride) {
  gemm_w4a16_rows_body<16, 8>(x, W, wsc, bias, res, C, M, N, K, ldx, ldw, ldws, ldc, ldr, act, per, xstride);
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

// One kernel while x is small enough to be staged whole by every sixteen rows of W: up to 32 KB.  Measured against the two kernels (us, back to back, M N K):
// 1 4096 4096 4.8 / 8.2, 1 22016 4096 13.9 / 18.0, 4 22016 4096 17.1 / 16.9 (and a launch of the host less), 1 4096 11008 9.2 / 12.4,
// 1 5120 13824 16.1 / 16.2, 1 15360 5120 14.8 / 16.2; beyond the rule 4 5120 13824 20.7 / 16.7, 4 27648 5120 27.8 / 25.5.
constexpr int W4_ROWS_MK = 16384;
bool w4_rows(int M, int K) { return M <= W4_ROWS && (long)M * K <= W4_ROWS_MK; }

// How many tiles a wave, how long a K-slice
constexpr long W4_FILL = 480;
struct W4Plan {
  int tiles, steps, splits;
};
W4Plan w4_plan(int N, int K) {
  const int total = (K / MX_BLOCK + 3) / 4;
  W4Plan r{1, W4_STEPS, 0};
  // two tiles a wave halve what is staged and read of x per byte of W, as long as about two workgroups are left for every CU (32 rows, 32104 x 4096:
  // 504 workgroups 32.3 us, 1004 with one tile 36.4 us); then long slices, likewise
  if ((long)cdiv(N, W4_WAVES * 32) * cdiv(total, W4_STEPS) >= W4_FILL) r.tiles = 2;
  while (r.steps > 2 && (long)cdiv(N, W4_WAVES * 16 * r.tiles) * cdiv(total, r.steps) < W4_FILL) r.steps -= 2;
  r.splits = cdiv(total, r.steps);
  return r;
}

}  // namespace
}  // namespace hvlm

using namespace hvlm;

extern "C" size_t hvlm_gemm_w4a16_ws_bytes(int M, int N, int K) {
  if (M <= 0 || M > 32 || N <= 0 || K < MX_BLOCK || w4_rows(M, K)) return 0;
  return (size_t)w4_plan(N, K).splits * M * ((size_t)(N + 3) / 4 * 4) * 4;
}

extern "C" int hvlm_gemm_w4a16_nt(const void* x, const void* W, const void* w_scale, void* C, int M, int N, int K, long ldx, long ldw, long ldws,
                                  long ldc, const void* bias, const void* residual, long ldr, int act, void* ws, void* stream) {
  HVLM_REQUIRE(x && W && w_scale && C, "gemm_w4a16_nt: null pointer");
  HVLM_REQUIRE(M > 0 && M <= 32, "gemm_w4a16_nt: M must be 1 .. 32 (got %d)", M);
  HVLM_REQUIRE(N > 0 && N <= (1 << 24) && K > 0 && K % MX_BLOCK == 0, "gemm_w4a16_nt: N=%d must be positive, K=%d a positive multiple of 32", N, K);
  HVLM_REQUIRE(ldx >= K && ldx % 8 == 0 && ((uintptr_t)x & 15) == 0, "gemm_w4a16_nt: rows of x must be 16-byte aligned");
  HVLM_REQUIRE(ldw >= K / 2 && ldw % 16 == 0 && ((uintptr_t)W & 15) == 0, "gemm_w4a16_nt: rows of codes must be 16-byte aligned");
  HVLM_REQUIRE(ldws >= K / MX_BLOCK && ldc >= N && (!residual || ldr >= N), "gemm_w4a16_nt: leading dimensions");
  HVLM_REQUIRE(act == HVLM_ACT_NONE || act == HVLM_ACT_QUICK_GELU, "gemm_w4a16_nt: unknown act %d", act);
  if (w4_rows(M, K)) {
    const int total = cdiv(K, 128), waves = total <= 8 * 4 ? 8 : 16, per = cdiv(total, waves), xstride = total * 128 + 8;
    const size_t need = (size_t)M * xstride * 2, red = (size_t)waves * M * 64;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_w4a16_rows_16_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                       (W4_ROWS_MK + W4_ROWS * (128 + 8)) * 2);
    if (attr != hipSuccess) { set_error("gemm_w4a16_nt: hipFuncSetAttribute: %s", hipGetErrorString(attr)); return HVLM_ERR_LAUNCH; }
    const auto k = waves == 8 ? gemm_w4a16_rows_8_kernel : gemm_w4a16_rows_16_kernel;
    hipLaunchKernelGGL(k, dim3((unsigned)cdiv(N, 16)), dim3((unsigned)waves * 64), need > red ? need : red, as_stream(stream), (const bf16_t*)x,
                       (const unsigned char*)W, (const unsigned char*)w_scale, (const bf16_t*)bias, (const bf16_t*)residual, (bf16_t*)C, M, N, K, ldx,
                       ldw, ldws, ldc, ldr, act, per, xstride);
    return check_launch("gemm_w4a16_nt");
  }
  const W4Plan plan = w4_plan(N, K);
  HVLM_REQUIRE(ws && ((uintptr_t)ws & 15) == 0, "gemm_w4a16_nt: a 16-byte aligned workspace of hvlm_gemm_w4a16_ws_bytes() is needed");
  HVLM_REQUIRE(plan.splits < 65536, "gemm_w4a16_nt: K=%d is too long", K);
  const int np = (N + 3) / 4 * 4;
  const dim3 grid(cdiv(N, W4_WAVES * 16 * plan.tiles), plan.splits), block(W4_WAVES * 64);
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
