// C[M, N] = act(A[M, K] @ B[N, K]^T + bias[N]) + residual[M, N] on MXFP4 operands (format: mxfp4.h), fp32 accumulation.
//
//   C[m, n] = sum over blocks g of 2^(sa[m, g] + sb[n, g] - 254) * sum_{k in g} a[m, k] b[n, k]
//
// is what v_mfma_scale_f32_16x16x128_f8f6f4 computes on fp4 operands: lane (r = l & 15, q = l >> 4) holds block q (32 codes, 16 bytes) of
// row r and that block's E8M0 byte, so a K-step of 128 takes one 16-byte LDS read and one byte of scale per fragment.  The weights are the
// first MFMA operand: a lane's four results are four consecutive columns of one output row.
//
// A workgroup of four waves computes a BM x BN tile, each wave a quarter.  Operand codes go from global memory to LDS without passing
// registers (16 rows x 64 B per wave instruction, 16-byte chunks permuted by c ^ ((row >> 1) & 3) so that eight adjacent rows of a
// fragment read fall into eight bank groups), two stages of 128 k ahead of their use; the scale bytes (4 per row and stage)
// take the way through a register, because their rows may start at any byte.  Rows past M / N and blocks
// past K read as zero codes.
#include "mxfp4.h"

namespace hvlm {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((address_space(3))) void* lds_ptr_t;

struct Mx4Args {
  const unsigned char *A, *B, *as, *bs;
  void* C;
  const bf16_t *bias, *res;
  int M, N, K;
  long lda, ldb, ldas, ldbs, ldc, ldr;
  int act, out_f32, tiles_m, tiles_n, vec;
};

constexpr int MX_GROUP_M = 8;             // row panels per group of the tile order
constexpr int MX_STAGES = 3;              // LDS ring: one stage being read, two in flight

template <int BM, int BN>
__global__ __launch_bounds__(256) void gemm_mxfp4_kernel(Mx4Args p) {
  constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16;
  constexpr unsigned CODES = (BM + BN) * 64, STAGE = CODES + (BM + BN) * 4;
  constexpr int PIECES = (BM + BN) / 64;  // LDS-DMA instructions per wave and stage
  extern __shared__ __attribute__((aligned(128))) char smem[];
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), l = t & 63, r16 = l & 15, q = l >> 4;

  // tile order: each XCD (blockIdx & 7) works through its own contiguous piece of the grouped order
  const int tiles = p.tiles_m * p.tiles_n, per = (tiles + 7) / 8;
  const int id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if (id >= tiles) return;
  const int gsz = MX_GROUP_M * p.tiles_n, grp = id / gsz, first = grp * MX_GROUP_M;
  const int gm = min(MX_GROUP_M, p.tiles_m - first), in = id - grp * gsz;
  const int m0 = (first + in % gm) * BM, n0 = (in / gm) * BN;

  const int nblk = p.K / MX_BLOCK, nst = (nblk + 3) / 4;
  // descriptors end with the last valid row; offsets within a tile stay below 2^31 (checked by the host), 2^31 and more reads as zero
  const long ba = (long)(p.M - m0 - 1) * p.lda + p.K / 2, bb = (long)(p.N - n0 - 1) * p.ldb + p.K / 2;
  const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.A) + (long)m0 * p.lda, 0, (unsigned)min(ba, 0x7fffffffL), 0x00020000);
  const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.B) + (long)n0 * p.ldb, 0, (unsigned)min(bb, 0x7fffffffL), 0x00020000);
  // piece i of wave w: rows 16 (w + 4 i) .. + 15 of the stacked (A rows, B rows) image
  unsigned off[PIECES];
  int chunk[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int row = 16 * (w + 4 * i) + (l >> 2);
    chunk[i] = (l & 3) ^ ((row >> 1) & 3);
    off[i] = (unsigned)(row < BM ? row * p.lda : (row - BM) * p.ldb) + (unsigned)chunk[i] * 16u;
  }
  auto stage_codes = [&](int s) {
    const unsigned base = (unsigned)(s % MX_STAGES) * STAGE;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const bool is_a = 16 * (w + 4 * i) < BM;
      const unsigned o = s * 4 + chunk[i] < nblk ? off[i] : 0x80000000u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(is_a ? ra : rb, (lds_ptr_t)(smem + base + (unsigned)(w + 4 * i) * 1024u), 16, o, (unsigned)s * 64u, 0, 0);
    }
  };
  // scale bytes of stage s: thread t takes rows t, t + 256 of the stacked image.  Rows past M / N repeat the last one (their results are
  // not stored); blocks past K get 2^0 against their zero codes (a NaN scale there would not stay invisible).
  constexpr int SR = (BM + BN) / 256;
  const unsigned char* srow[SR];
#pragma unroll
  for (int i = 0; i < SR; ++i) {
    const int row = t + 256 * i;
    srow[i] = row < BM ? p.as + (long)min(m0 + row, p.M - 1) * p.ldas : p.bs + (long)min(n0 + row - BM, p.N - 1) * p.ldbs;
  }
  auto load_scales = [&](int s, unsigned (&v)[SR]) {
    if (s * 4 + 4 <= nblk) {
#pragma unroll
      for (int i = 0; i < SR; ++i) __builtin_memcpy(&v[i], srow[i] + s * 4, 4);        // any alignment
    } else {
#pragma unroll
      for (int i = 0; i < SR; ++i) {
        v[i] = 0x7f7f7f7fu;
        for (int b = s * 4; b < nblk; ++b) v[i] = (v[i] & ~(255u << (8 * (b & 3)))) | (unsigned)srow[i][b] << (8 * (b & 3));
      }
    }
  };
  auto put_scales = [&](int s, const unsigned (&v)[SR]) {
    unsigned* d = reinterpret_cast<unsigned*>(smem + (unsigned)(s % MX_STAGES) * STAGE + CODES);
#pragma unroll
    for (int i = 0; i < SR; ++i) d[t + 256 * i] = v[i];
  };

  const int wm = (w & 1) * WM, wn = (w >> 1) * WN;
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  unsigned sv[SR];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    load_scales(s, sv);                     // (a stage past the end stages zeros)
    stage_codes(s);
    put_scales(s, sv);
  }
  const unsigned swz = (unsigned)(q ^ ((r16 >> 1) & 3)) * 16u;
  for (int s = 0; s < nst; ++s) {
    // this wave's pieces of stages <= s have landed (only stage s + 1's are still out), its scale writes are done; behind the barrier
    // everyone's have, and nobody reads stage s - 1 any more
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PIECES) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    load_scales(s + 2, sv);
    stage_codes(s + 2);
    const char* base = smem + (unsigned)(s % MX_STAGES) * STAGE;
    const unsigned char* sc = reinterpret_cast<const unsigned char*>(base) + CODES;
    i32x8 fb[TN];
    int sb[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(base + (unsigned)(BM + wn + 16 * j + r16) * 64u + swz);
      fb[j] = i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
      sb[j] = sc[(BM + wn + 16 * j + r16) * 4 + q];
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(base + (unsigned)(wm + 16 * i + r16) * 64u + swz);
      const i32x8 fa = i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
      const int sa = sc[(wm + 16 * i + r16) * 4 + q];
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, acc[i][j], 4, 4, 0, sb[j], 0, sa);
    }
    put_scales(s + 2, sv);
  }

  // D: lane holds row m = .. + r16 and the four columns n = .. + 4 q
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm + 16 * i + r16;
    if (m >= p.M) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + wn + 16 * j + 4 * q;
      if (n >= p.N) continue;
      f32x4 v = acc[i][j];
      const bool whole = p.vec && n + 4 <= p.N;
      float b[4] = {0.f, 0.f, 0.f, 0.f}, rs[4] = {0.f, 0.f, 0.f, 0.f};
      if (p.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = n + e < p.N ? bf2f(p.bias[n + e]) : 0.f;
      }
      if (p.res) {
        if (whole) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(p.res + (long)m * p.ldr + n);
          rs[0] = bf_lo(x[0]); rs[1] = bf_hi(x[0]); rs[2] = bf_lo(x[1]); rs[3] = bf_hi(x[1]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) rs[e] = n + e < p.N ? bf2f(p.res[(long)m * p.ldr + n + e]) : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] += b[e];
        if (p.act == HVLM_ACT_QUICK_GELU) v[e] *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.702f * 1.4426950408889634f * v[e]));
        v[e] += rs[e];
      }
      if (p.out_f32) {
        float* o = reinterpret_cast<float*>(p.C) + (long)m * p.ldc + n;
        if (whole) *reinterpret_cast<f32x4*>(o) = v;
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) if (n + e < p.N) o[e] = v[e];
      } else {
        bf16_t* o = reinterpret_cast<bf16_t*>(p.C) + (long)m * p.ldc + n;
        if (whole) *reinterpret_cast<u32x2*>(o) = u32x2{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3])};
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) if (n + e < p.N) o[e] = f2bf(v[e]);
      }
    }
  }
}

template <int BM, int BN>
int mx4_launch(Mx4Args p, hipStream_t stream) {
  constexpr int lds = MX_STAGES * (BM + BN) * 68;
  const auto k = gemm_mxfp4_kernel<BM, BN>;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (attr != hipSuccess) { set_error("gemm_mxfp4: hipFuncSetAttribute: %s", hipGetErrorString(attr)); return HVLM_ERR_LAUNCH; }
  p.tiles_m = cdiv(p.M, BM);
  p.tiles_n = cdiv(p.N, BN);
  const int tiles = p.tiles_m * p.tiles_n;
  hipLaunchKernelGGL(k, dim3((unsigned)cdiv(tiles, 8) * 8), dim3(256), lds, stream, p);
  return check_launch("gemm_mxfp4_nt");
}

}  // namespace
}  // namespace hvlm

using namespace hvlm;

extern "C" int hvlm_gemm_mxfp4_nt(const void* A, const void* a_scale, const void* B, const void* b_scale, void* C, int M, int N, int K, long lda,
                                  long ldas, long ldb, long ldbs, long ldc, const void* bias, const void* residual, long ldr, int act, int out_f32,
                                  void* stream) {
  HVLM_REQUIRE(A && a_scale && B && b_scale && C, "gemm_mxfp4_nt: null pointer");
  HVLM_REQUIRE(M > 0 && N > 0 && K > 0 && K % MX_BLOCK == 0, "gemm_mxfp4_nt: M=%d, N=%d must be positive, K=%d a positive multiple of 32", M, N, K);
  HVLM_REQUIRE(lda >= K / 2 && ldb >= K / 2 && lda % 16 == 0 && ldb % 16 == 0 && ((uintptr_t)A & 15) == 0 && ((uintptr_t)B & 15) == 0,
               "gemm_mxfp4_nt: rows of codes must be 16-byte aligned");
  HVLM_REQUIRE(lda < (1L << 22) && ldb < (1L << 22), "gemm_mxfp4_nt: leading dimensions of the codes must be below 4 MiB");
  HVLM_REQUIRE(ldas >= K / MX_BLOCK && ldbs >= K / MX_BLOCK, "gemm_mxfp4_nt: leading dimensions of the scales");
  HVLM_REQUIRE(ldc >= N && (!residual || ldr >= N), "gemm_mxfp4_nt: leading dimensions of C / residual");
  HVLM_REQUIRE(act == HVLM_ACT_NONE || act == HVLM_ACT_QUICK_GELU, "gemm_mxfp4_nt: unknown act %d", act);
  HVLM_REQUIRE((long)cdiv(M, 128) * cdiv(N, 128) < (1L << 30), "gemm_mxfp4_nt: too many tiles");
  Mx4Args p{};
  p.A = (const unsigned char*)A; p.B = (const unsigned char*)B; p.as = (const unsigned char*)a_scale; p.bs = (const unsigned char*)b_scale;
  p.C = C; p.bias = (const bf16_t*)bias; p.res = (const bf16_t*)residual;
  p.M = M; p.N = N; p.K = K; p.lda = lda; p.ldb = ldb; p.ldas = ldas; p.ldbs = ldbs; p.ldc = ldc; p.ldr = ldr; p.act = act; p.out_f32 = out_f32;
  const int es = out_f32 ? 4 : 2;
  p.vec = ldc % 4 == 0 && ((uintptr_t)C & (4 * es - 1)) == 0 && (!residual || (ldr % 4 == 0 && ((uintptr_t)residual & 7) == 0));
  return mx4_launch<128, 128>(p, as_stream(stream));
}
