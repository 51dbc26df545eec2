// out[M, N] = act(x[M, K] @ W[N, K]^T + bias) + residual for M <= 32, x in bf16 and W in MXFP4 (format: mxfp4.h): the projections of a
// decode step, whose cost is one read of W (17/32 bytes per element).
//
// W goes from global memory to registers and from there, de-quantised to bf16 (exact), straight into v_mfma_f32_16x16x32_bf16 as its first
// operand: lane (r = l & 15, q = l >> 4) holds one whole block of row r, 16 bytes of codes, consumed by four MFMAs of 8 k per lane
// against the same k of x.  A wave owns 16 rows of W and one K-slice of at most 1024 k: all of its code loads and its scale load are in flight
// before anything is consumed (8.5 KB; there is no ring to keep filled).  A code load is issued in the coalesced order
// (lane = row l >> 2, 16-byte chunk l & 3) and turned into fragment order by ds_bpermute_b32 when it is consumed.  x is staged once per
// workgroup and slice in LDS.  K-slices are summed, in order, from fp32 slabs by a second small kernel with the epilogue; with one to four rows
// of x the slices are the waves of one workgroup and no second kernel runs.
//
// Bound by the read of W where W is large: 22016 x 4096 at one row 10.8 us (4.4 TB/s; a copy's rate would take 10.0 us),
// 32101 x 4096 at 32 rows 21.2 us + 4.6 us to sum the slabs (15.1 us; there the staging of x, as many bytes from L2 as W has, and the slabs, 16 MB, come on top).
#include "mxfp4.h"

namespace hvlm {
namespace {

constexpr int W4_WAVES = 8;               // 128 rows of W per workgroup
__host__ __device__ constexpr int w4_xstride(int steps) { return steps * 128 + 8; }   // elements per x row in LDS: the 16 bytes of padding put sixteen rows into different banks

// A barrier for LDS alone: the wave's own LDS accesses are done, its loads from memory may still be out.
__device__ __forceinline__ void w4_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The blocks b0 .. b0 + nb - 1 (at most 4 STEPS; a multiple of four but at the end of a row of nblk) of sixteen rows of W, as a wave holds them: codes
// in the coalesced order, scales eight bytes a lane.
template <int STEPS>
struct W4Slice {
  u32x4 ring[STEPS];
  unsigned long sc;
  int past;                                // bytes of sc that lie before its first
};
// No branch on what is there: loads of whole steps past the end repeat the last block, so that every product knows how many loads are behind its own.
template <int STEPS>
__device__ __forceinline__ void w4_load(W4Slice<STEPS>& f, const unsigned char* __restrict__ W, const unsigned char* __restrict__ wsc, long ldw, long ldws, int n0, int N,
                                        int b0, int nb, int nblk, int l) {
  const int r16 = l & 15, q = l >> 4;
  // scales: lane (r, q) takes bytes 8 q .. 8 q + 7 of row r's slice, the blocks of steps 2 q and 2 q + 1; near the row's end its last eight bytes
  const unsigned char* sp = wsc + (long)min(n0 + r16, N - 1) * ldws;
  const int at = min(b0 + 8 * q, max(nblk - 8, 0));
  f.past = b0 + 8 * q - at;
  if (nblk >= 8) {
    __builtin_memcpy(&f.sc, sp + at, 8);                                       // any alignment
  } else {
    f.sc = 0;
#pragma unroll
    for (int b = 0; b < 7; ++b) f.sc |= (unsigned long)(b < nblk ? sp[min(b, nblk - 1)] : 127) << (8 * b);
  }
  const unsigned char* wp = W + (long)min(n0 + (l >> 2), N - 1) * ldw + (long)b0 * 16;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) f.ring[i] = *reinterpret_cast<const u32x4*>(wp + min(i * 4 + (l & 3), nb - 1) * 16);
}
// acc[h] += the slice times x: xr[h] points at this lane's 32 k of step 0 of its row of x
template <int STEPS, int HALVES>
__device__ __forceinline__ void w4_product(const W4Slice<STEPS>& f, const bf16_t* const (&xr)[HALVES], f32x4 (&acc)[HALVES], int nb, int l) {
  const int r16 = l & 15, q = l >> 4, perm = (4 * r16 + q) << 2;               // fragment lane (r, q) <- load lane 4 r + q
  const unsigned long ones = 0x7f7f7f7f7f7f7f7ful;                             // past the row's end 2^0 (x is zero there)
  const int sh = 8 * f.past;
  const unsigned long v = sh == 0 ? f.sc : sh < 64 ? f.sc >> sh | ones << (64 - sh) : ones;
  const unsigned sc[2] = {(unsigned)v, (unsigned)(v >> 32)};
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    if (i * 4 >= nb) break;
    const unsigned s4 = (unsigned)__builtin_amdgcn_ds_bpermute((r16 + 16 * (i >> 1)) << 2, (int)sc[i & 1]);
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

struct W4Args {
  const bf16_t *x, *bias, *res;
  const unsigned char *W, *wsc;
  float* ws;
  bf16_t* C;
  int M, N, K, np, act, per;
  long ldx, ldw, ldws, ldc, ldr;
};
// STEPS: steps of 128 k of the K-slice
template <int HALVES, int STEPS>
__device__ __forceinline__ void gemm_w4a16_body(const W4Args& p) {
  extern __shared__ __attribute__((aligned(16))) bf16_t xs[];
  constexpr int XS = w4_xstride(STEPS), XU = (STEPS * 16 + 63) / 64;
  const int t = threadIdx.x, w = t >> 6, l = t & 63, r16 = l & 15, q = l >> 4, M = p.M, nblk = p.K / MX_BLOCK;
  const int b0 = blockIdx.y * STEPS * 4, nb = min(STEPS * 4, nblk - b0);      // this slice's blocks
  const int n0 = (blockIdx.x * W4_WAVES + w) * 16;

  // x slice -> LDS: rows 0 .. M - 1, zero past K.  Its loads go first (loads come back in order), and nothing waits for W before the products do.
  u32x4 xv[2 * HALVES][XU];
#pragma unroll
  for (int i = 0; i < 2 * HALVES; ++i)
#pragma unroll
    for (int u = 0; u < XU; ++u)
      xv[i][u] = *reinterpret_cast<const u32x4*>(p.x + (long)min(w + i * W4_WAVES, M - 1) * p.ldx + (long)b0 * MX_BLOCK + min(l + 64 * u, nb * 4 - 1) * 8);
  W4Slice<STEPS> f;
  w4_load(f, p.W, p.wsc, p.ldw, p.ldws, n0, p.N, b0, nb, nblk, l);
#pragma unroll
  for (int i = 0; i < 2 * HALVES; ++i)
#pragma unroll
    for (int u = 0; u < XU; ++u) {
      const int m = w + i * W4_WAVES, c = l + 64 * u;
      if (m < M && c < STEPS * 16) *reinterpret_cast<u32x4*>(xs + m * XS + c * 8) = c < nb * 4 ? xv[i][u] : u32x4{0u, 0u, 0u, 0u};
    }
  w4_barrier();

  const bf16_t* xr[HALVES];                                                  // columns past M repeat the last row, their results are dropped
#pragma unroll
  for (int h = 0; h < HALVES; ++h) xr[h] = xs + min(h * 16 + r16, M - 1) * XS + q * 32;
  f32x4 acc[HALVES];
#pragma unroll
  for (int h = 0; h < HALVES; ++h) acc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
  w4_product<STEPS, HALVES>(f, xr, acc, nb, l);
  // D: lane holds column m = r16 (+ 16), rows 4 q .. + 3 of the tile
  const int n = n0 + 4 * q;
  if (n < p.np) {
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      const int m = h * 16 + r16;
      if (m < M) *reinterpret_cast<f32x4*>(p.ws + ((long)blockIdx.y * M + m) * p.np + n) = acc[h];
    }
  }
}
#define W4_KERNEL(H, S) \
  __global__ __launch_bounds__(W4_WAVES * 64, 4) void gemm_w4a16_##H##_##S##_kernel(W4Args p) { gemm_w4a16_body<H, S>(p); }
W4_KERNEL(1, 4) W4_KERNEL(1, 6) W4_KERNEL(1, 8) W4_KERNEL(2, 4) W4_KERNEL(2, 6) W4_KERNEL(2, 8)
#undef W4_KERNEL

__device__ __forceinline__ bf16_t w4_finish(float y, float bias, float res, int act) {
  y += bias;
  if (act == HVLM_ACT_QUICK_GELU) y *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.702f * 1.4426950408889634f * y));
  return f2bf(y + res);
}

// A few rows of x, all of them in LDS: the waves of a workgroup share sixteen rows of W, at most STEPS steps of K each, and add up in LDS, in order; no
// slabs, no second kernel.  At most 64 registers, so that a CU holds 32 waves.
constexpr int W4_ROWS = 4;
template <int WAVES, int STEPS>
__device__ __forceinline__ void gemm_w4a16_rows_body(const W4Args& p) {
  extern __shared__ __attribute__((aligned(16))) bf16_t xs[];
  const int t = threadIdx.x, w = t >> 6, l = t & 63, r16 = l & 15, q = l >> 4, M = p.M, nblk = p.K / MX_BLOCK;
  constexpr int XU = WAVES == 8 ? 4 : 2;
  const int ends = (nblk + 3) / 4 * 16, all = M * ends, xstride = ends * 8 + 8;                  // chunks of eight of a row of x, of all
  const int b0 = min(w * p.per * 4, nblk - 1), nb = min(p.per * 4, nblk - w * p.per * 4);        // this wave's blocks, perhaps none
  const int n0 = blockIdx.x * 16;
  // x -> LDS: rows 0 .. M - 1, zero from K to the end of its last step; at most XU chunks a thread (w4_rows).  Its loads go first.
  u32x4 xv[XU];
#pragma unroll
  for (int u = 0; u < XU; ++u) {
    const int i = min(t + u * WAVES * 64, all - 1), m = i / ends, c = i - m * ends;
    if (u * WAVES * 64 < all) xv[u] = *reinterpret_cast<const u32x4*>(p.x + (long)m * p.ldx + min(c * 8, p.K - 8));
  }
  W4Slice<STEPS> f;
  w4_load(f, p.W, p.wsc, p.ldw, p.ldws, n0, p.N, b0, max(nb, 1), nblk, l);
#pragma unroll
  for (int u = 0; u < XU; ++u) {
    const int i = t + u * WAVES * 64, m = i / ends, c = i - m * ends;
    if (i < all) *reinterpret_cast<u32x4*>(xs + m * xstride + c * 8) = c < p.K / 8 ? xv[u] : u32x4{0u, 0u, 0u, 0u};
  }
  w4_barrier();
  f32x4 acc[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
  const bf16_t* const xr[1] = {xs + min(r16, M - 1) * xstride + b0 * MX_BLOCK + q * 32};
  w4_product<STEPS, 1>(f, xr, acc, nb, l);
  __syncthreads();                                                           // x is read; its room takes the partial sums [wave][m][16]
  float* red = reinterpret_cast<float*>(xs);
  if (r16 < M) *reinterpret_cast<f32x4*>(red + (w * M + r16) * 16 + 4 * q) = acc[0];
  __syncthreads();
  if (t < 16 * M) {
    const int m = t >> 4, n = n0 + (t & 15);
    float y = 0.f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) y += red[(v * M + m) * 16 + (t & 15)];
    if (n < p.N) p.C[(long)m * p.ldc + n] = w4_finish(y, p.bias ? bf2f(p.bias[n]) : 0.f, p.res ? bf2f(p.res[(long)m * p.ldr + n]) : 0.f, p.act);
  }
}
__global__ __launch_bounds__(512, 8) void gemm_w4a16_rows_8_kernel(W4Args p) { gemm_w4a16_rows_body<8, 4>(p); }
__global__ __launch_bounds__(1024, 8) void gemm_w4a16_rows_16_kernel(W4Args p) { gemm_w4a16_rows_body<16, 7>(p); }

// C = the slabs' sum, in order, with the epilogue: four columns a thread
__global__ __launch_bounds__(256) void w4a16_finalize_kernel(W4Args p, int splits) {
  const int per_row = p.np / 4;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < p.M * per_row; i += gridDim.x * 256) {
    const int m = i / per_row, n = (i - m * per_row) * 4;
    float b[4] = {0.f, 0.f, 0.f, 0.f}, r[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.bias)
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = bf2f(p.bias[min(n + e, p.N - 1)]);
    if (p.res)
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = bf2f(p.res[(long)m * p.ldr + min(n + e, p.N - 1)]);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < splits; s0 += 8) {                                   // eight slabs' loads at a time
      f32x4 a[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) a[s] = *reinterpret_cast<const f32x4*>(p.ws + ((long)min(s0 + s, splits - 1) * p.M + m) * p.np + n);
#pragma unroll
      for (int s = 0; s < 8; ++s) if (s0 + s < splits) v += a[s];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) p.C[(long)m * p.ldc + n + e] = w4_finish(v[e], b[e], r[e], p.act);
  }
}


// One kernel while x is small enough to be staged whole by every sixteen rows of W: up to 32 KB.  Measured against the two kernels (us, back to back, M N K):
// 1 4096 4096 4.2 / 6.5, 4 4096 4096 5.0 / 6.9, 1 22016 4096 11.7 / 15, 4 22016 4096 15.6 / 15.4 (and a launch of the host less), 1 4096 11008 9.4 / 11,
// 1 27648 5120 23.2 / 23.9; beyond the rule, before the loads of x went first, 4 5120 13824 20.7 / 16.7, 4 27648 5120 27.8 / 25.5.
bool w4_rows(int M, int K) { return M <= W4_ROWS && (K <= 8 * 4 * 128 || (long)M * K <= 16 * 7 * 128); }

// How long a K-slice: 8, 6 or 4 steps, whichever gives the CU with the most workgroups the least to do, a workgroup's start and end counted as two steps.
// Measured at 32 rows (us for 8 / 6 / 4; the rule's choice first): 12288 x 4096 15.6 (4) / 16.6 (8) / 16.4 (6), 22016 x 4096 21.6 (8) / 22.9 (6) / 24.1 (4),
// 5120 x 13824 19.7 (6) / 20.1 (8) / 22.0 (4), 5120 x 5120 11.4 (8) / 12.9 (6) / 13.1 (4).
struct W4Plan {
  int steps, splits;
};
W4Plan w4_plan(int N, int K) {
  W4Plan r{0, 0};
  long least = 0;
  for (int steps = 8; steps >= 4; steps -= 2) {
    const int splits = cdiv(cdiv(K, 128), steps);
    const long cost = (long)cdiv((long)cdiv(N, W4_WAVES * 16) * splits, 256) * (steps + 2);
    if (r.steps == 0 || cost < least) { r = W4Plan{steps, splits}; least = cost; }
  }
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
  const int total = cdiv(K, 128);
  W4Args p{};
  p.x = (const bf16_t*)x; p.bias = (const bf16_t*)bias; p.res = (const bf16_t*)residual; p.W = (const unsigned char*)W; p.wsc = (const unsigned char*)w_scale;
  p.ws = (float*)ws; p.C = (bf16_t*)C; p.M = M; p.N = N; p.K = K; p.act = act; p.ldx = ldx; p.ldw = ldw; p.ldws = ldws; p.ldc = ldc; p.ldr = ldr;
  p.np = (N + 3) / 4 * 4;
  typedef void (*kernel)(W4Args);
  if (w4_rows(M, K)) {
    const int waves = total <= 8 * 4 ? 8 : 16;
    p.per = cdiv(total, waves);
    const size_t need = (size_t)M * (total * 128 + 8) * 2, red = (size_t)waves * M * 64;
    hipLaunchKernelGGL(waves == 8 ? gemm_w4a16_rows_8_kernel : gemm_w4a16_rows_16_kernel, dim3((unsigned)cdiv(N, 16)), dim3((unsigned)waves * 64),
                       need > red ? need : red, as_stream(stream), p);
    return check_launch("gemm_w4a16_nt");
  }
  const W4Plan plan = w4_plan(N, K);
  HVLM_REQUIRE(ws && ((uintptr_t)ws & 15) == 0, "gemm_w4a16_nt: a 16-byte aligned workspace of hvlm_gemm_w4a16_ws_bytes() is needed");
  HVLM_REQUIRE(plan.splits < 65536, "gemm_w4a16_nt: K=%d is too long", K);
  static const kernel kernels[2][3] = {{gemm_w4a16_1_4_kernel, gemm_w4a16_1_6_kernel, gemm_w4a16_1_8_kernel},
                                       {gemm_w4a16_2_4_kernel, gemm_w4a16_2_6_kernel, gemm_w4a16_2_8_kernel}};
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_w4a16_2_8_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 32 * w4_xstride(8) * 2);
  if (attr != hipSuccess) { set_error("gemm_w4a16_nt: hipFuncSetAttribute: %s", hipGetErrorString(attr)); return HVLM_ERR_LAUNCH; }
  hipLaunchKernelGGL(kernels[M > 16][plan.steps / 2 - 2], dim3(cdiv(N, W4_WAVES * 16), plan.splits), dim3(W4_WAVES * 64),
                     (size_t)M * w4_xstride(plan.steps) * 2, as_stream(stream), p);
  const int rc = check_launch("gemm_w4a16_nt");
  if (rc) return rc;
  const long items = (long)M * (p.np / 4);
  hipLaunchKernelGGL(w4a16_finalize_kernel, dim3((unsigned)min(cdiv(items, 256), 2048)), dim3(256), 0, as_stream(stream), p, plan.splits);
  return check_launch("gemm_w4a16_nt");
}
