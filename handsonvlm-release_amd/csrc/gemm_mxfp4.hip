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
#include <algorithm>
#include <type_traits>

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
  int act, out_f32, tiles_m, tiles_n;
};

constexpr int MX_GROUP_M = 8;             // row panels per group of the tile order
constexpr int MX_NS = 4;                  // LDS ring: one stage being read, three landing or landed
constexpr int MX_CUS = 256;               // persistent workgroups, one per CU

// s_waitcnt lgkmcnt(0) vmcnt(V)
template <int V>
__device__ __forceinline__ void mx_wait() {
  __builtin_amdgcn_s_waitcnt((V & 15) | ((V >> 4) << 14) | 0x70);
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void mx_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
// lane quarters l >> 4 = 0 .. 3 hold four units a, b, c, d each: quarter j gets unit j of every quarter (its own inverse when read backwards)
__device__ __forceinline__ void mx_swap32(unsigned& a, unsigned& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0]; b = r[1];
}
__device__ __forceinline__ void mx_swap16(unsigned& a, unsigned& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0]; b = r[1];
}

// Results of a wave: rows m + 16 i, 16 TN columns from n0 on.  A lane holds four consecutive columns of each 16-column fragment; quarters
// of the wave exchange them (packed to bf16) so that it stores 4 TN consecutive columns.  Stores may be unaligned (odd leading dimensions).
// PRE: 0 = nothing, 1 = bias, 2 = bias (if any) and QuickGELU.  One straight-line body per combination: with the choices inside, the
// accumulators meet in the branches and are spilled.
template <int TM, int TN, int PRE, bool RES, bool F32>
__device__ __forceinline__ void mx_epilogue(const Mx4Args& p, const f32x4 (&acc)[TM][TN], int m, int n0, int q) {
  typedef u32x4 __attribute__((aligned(2))) u32x4_u;
  typedef f32x4 __attribute__((aligned(4))) f32x4_u;
  const int n = n0 + (TN == 4 ? 16 * q : 16 * (q >> 1) + 8 * (q & 1));           // the lane's columns after the exchange
  const bool whole = n + 4 * TN <= p.N;
  float b[TN][4];
  if constexpr (PRE > 0) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) b[j][e] = p.bias ? bf2f(p.bias[min(n0 + 16 * j + 4 * q + e, p.N - 1)]) : 0.f;
  }
  unsigned r[RES ? TM : 1][TN][2];                                               // residual rows: all loads first, C may be the residual itself
  if constexpr (RES) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const bf16_t* s = p.res + (long)min(m + 16 * i, p.M - 1) * p.ldr + n;
      if (whole) {
        const u32x4 x = *reinterpret_cast<const u32x4_u*>(s);
        r[i][0][0] = x[0]; r[i][0][1] = x[1]; r[i][1][0] = x[2]; r[i][1][1] = x[3];
        if constexpr (TN == 4) {
          const u32x4 y = *reinterpret_cast<const u32x4_u*>(s + 8);
          r[i][2][0] = y[0]; r[i][2][1] = y[1]; r[i][3][0] = y[2]; r[i][3][1] = y[3];
        }
      } else {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = 4 * j + 2 * e;
            const unsigned lo = n + c < p.N ? s[c] : 0u, hi = n + c + 1 < p.N ? s[c + 1] : 0u;
            r[i][j][e] = lo | hi << 16;
          }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int row = m + 16 * i;
    f32x4 v[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      v[j] = acc[i][j];
      if constexpr (PRE > 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[j][e] += b[j][e];
          if constexpr (PRE == 2) v[j][e] *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.702f * 1.4426950408889634f * v[j][e]));
        }
      }
    }
    if constexpr (RES) {                                                         // back into the layout of the accumulators
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if constexpr (TN == 4) {
          mx_swap16(r[i][0][e], r[i][1][e]); mx_swap16(r[i][2][e], r[i][3][e]);
          mx_swap32(r[i][0][e], r[i][2][e]); mx_swap32(r[i][1][e], r[i][3][e]);
        } else {
          mx_swap16(r[i][0][e], r[i][1][e]); mx_swap32(r[i][0][e], r[i][1][e]);
        }
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        v[j][0] += bf_lo(r[i][j][0]); v[j][1] += bf_hi(r[i][j][0]);
        v[j][2] += bf_lo(r[i][j][1]); v[j][3] += bf_hi(r[i][j][1]);
      }
    }
    if constexpr (F32) {
      if (row < p.M) {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int c = n0 + 16 * j + 4 * q;
          float* o = reinterpret_cast<float*>(p.C) + (long)row * p.ldc + c;
          if (c + 4 <= p.N) *reinterpret_cast<f32x4_u*>(o) = v[j];
          else
#pragma unroll
            for (int e = 0; e < 4; ++e) if (c + e < p.N) o[e] = v[j][e];
        }
      }
    } else {
      unsigned d[TN][2];
#pragma unroll
      for (int j = 0; j < TN; ++j) { d[j][0] = pack_bf2(v[j][0], v[j][1]); d[j][1] = pack_bf2(v[j][2], v[j][3]); }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if constexpr (TN == 4) {
          mx_swap32(d[0][e], d[2][e]); mx_swap32(d[1][e], d[3][e]);
          mx_swap16(d[0][e], d[1][e]); mx_swap16(d[2][e], d[3][e]);
        } else {
          mx_swap32(d[0][e], d[1][e]); mx_swap16(d[0][e], d[1][e]);
        }
      }
      if (row < p.M) {
        bf16_t* o = reinterpret_cast<bf16_t*>(p.C) + (long)row * p.ldc + n;
        if (whole) {
          *reinterpret_cast<u32x4_u*>(o) = u32x4{d[0][0], d[0][1], d[1][0], d[1][1]};
          if constexpr (TN == 4) *reinterpret_cast<u32x4_u*>(o + 8) = u32x4{d[2][0], d[2][1], d[3][0], d[3][1]};
        } else {
#pragma unroll
          for (int e = 0; e < 4 * TN; ++e) if (n + e < p.N) o[e] = (bf16_t)(d[e >> 2][(e >> 1) & 1] >> (16 * (e & 1)));
        }
      }
    }
  }
}

template <int TM, int TN, int PRE>
__device__ __forceinline__ void mx_epilogue_pre(const Mx4Args& p, const f32x4 (&acc)[TM][TN], int m, int n0, int q) {
  if (p.out_f32) {
    if (p.res) mx_epilogue<TM, TN, PRE, true, true>(p, acc, m, n0, q);
    else mx_epilogue<TM, TN, PRE, false, true>(p, acc, m, n0, q);
  } else {
    if (p.res) mx_epilogue<TM, TN, PRE, true, false>(p, acc, m, n0, q);
    else mx_epilogue<TM, TN, PRE, false, false>(p, acc, m, n0, q);
  }
}

// The lane's number, computed where it is used: registers of the K loop are full, and what is derived from threadIdx once is spilled.
__device__ __forceinline__ int mx_lane() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}

template <int BM, int BN, int KS>
struct Mx4Geo {
  static constexpr int WM = BM / 2, WN = BN / 4, TM = WM / 16, TN = WN / 16;
  static constexpr unsigned SUB = (BM + BN) * 64, STAGE = KS * SUB;             // 128 k of both operands; a stage
  static constexpr unsigned SROW = (BM + BN) * 4, SIMG = 4 * KS * SROW;          // scale bytes of 128 k; a group of four stages
  static constexpr int LDS = MX_NS * (int)STAGE + 2 * (int)SIMG;
  static constexpr int PIECES = (BM + BN) / 128 * KS;                            // LDS-DMA instructions per wave and stage
};

// (a __device__ template under plain __global__ wrappers, as in gemm_pp.hip)
template <int BM, int BN, int KS>
__device__ __forceinline__ void gemm_mxfp4_body(const Mx4Args& p) {
  using G = Mx4Geo<BM, BN, KS>;
  constexpr int TM = G::TM, TN = G::TN, PIECES = G::PIECES, SQ = (BM + BN) / 64;
  static_assert((TM == 8 && TN == 4) || (TM == 4 && TN == 2), "fragment layouts of the epilogue");
  extern __shared__ __attribute__((aligned(128))) char smem[];
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), l = t & 63, r16 = l & 15, q = l >> 4;
  const int tiles = p.tiles_m * p.tiles_n, per = (tiles + 7) / 8;
  // stages of a tile; at least three, so that the next tile's first two are always issued inside this one's (those past K are zeros)
  const int nblk = p.K / MX_BLOCK, nst = max((nblk + 4 * KS - 1) / (4 * KS), 3), ngr = (nst + 3) / 4;

  // tile order: XCD x (blockIdx & 7) owns tiles x * per .. of the grouped order, its workgroups take every (gridDim / 8)-th of them
  const int lim = min(tiles, ((int)(blockIdx.x & 7) + 1) * per);
  int id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if (id >= lim) return;

  // codes: DMA piece j of wave w = rows 16 (w + 8 j) .. + 15 of the stacked (A rows, B rows) image, lane = (row l >> 2, chunk position l & 3)
  const int chunk = (l & 3) ^ ((l >> 3) & 3);
  const unsigned off_a = (unsigned)(16 * w + (l >> 2)) * (unsigned)p.lda + (unsigned)chunk * 16u;
  const unsigned off_b = (unsigned)(16 * w + (l >> 2)) * (unsigned)p.ldb + (unsigned)chunk * 16u;
  auto coords = [&](int tile, int& m0, int& n0) {
    const int gsz = MX_GROUP_M * p.tiles_n, grp = tile / gsz, first = grp * MX_GROUP_M;
    const int gm = min(MX_GROUP_M, p.tiles_m - first), in = tile - grp * gsz;
    m0 = (first + in % gm) * BM;
    n0 = (in / gm) * BN;
  };
  // descriptors of a tile's operands end with the last valid row; offsets within a tile stay below 2^31 (checked by the host), 2^31 and more
  // reads as zero
  __amdgpu_buffer_rsrc_t ra, rb;
  auto point = [&](int m0, int n0) {
    const long ba = (long)(p.M - m0 - 1) * p.lda + p.K / 2, bb = (long)(p.N - n0 - 1) * p.ldb + p.K / 2;
    ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.A) + (long)m0 * p.lda, 0, (unsigned)min(ba, 0x7fffffffL), 0x00020000);
    rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.B) + (long)n0 * p.ldb, 0, (unsigned)min(bb, 0x7fffffffL), 0x00020000);
  };
  // one DMA piece of a stage into ring slot `slot`; blocks past K come as zeros
  auto dma = [&](int s, int slot, int i) {
    const int u = i / (PIECES / KS), j = i % (PIECES / KS);
    const unsigned base = (unsigned)(slot & (MX_NS - 1)) * G::STAGE + u * G::SUB + (unsigned)(w + 8 * j) * 1024u;
    const int b0 = (s * KS + u) * 4;
    constexpr int JA = BM / 128;                                                  // pieces 0 .. JA - 1 are rows of A
    unsigned o = j < JA ? off_a : off_b;
    asm volatile("" : "+v"(o));                                                   // (one address register for all pieces of an operand)
    o += j < JA ? (unsigned)j * 128u * (unsigned)p.lda : (unsigned)(j - JA) * 128u * (unsigned)p.ldb;
    if (b0 + 4 > nblk) o = b0 + chunk < nblk ? o : 0x80000000u;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(j < JA ? ra : rb, (lds_ptr_t)(smem + base), 16, o, (unsigned)b0 * 16u, 0, 0);
  };
  // scales of a group = 512 KS k: KS loads of 16 bytes a lane, at any alignment, or more and narrower ones where the row ends.  The descriptor
  // ends with the last valid row, past which 2^-127 comes back.
  // Wave w stages rows 64 w .. + 63 of the stacked image, lane = (row l >> 2 of a 16-row tile, tile l & 3): the four lanes of a quad hold the
  // four tiles whose bytes share a dword of the image.
  __amdgpu_buffer_rsrc_t rs;
  const bool s_of_a = w < BM / 64;
  const int s_row0 = s_of_a ? 64 * w : 64 * min(w, SQ - 1) - BM;
  const unsigned char* const s_ptr = s_of_a ? p.as : p.bs;
  const long s_ld = s_of_a ? p.ldas : p.ldbs;
  const int s_rows = s_of_a ? p.M : p.N;
  auto point_scales = [&](int first) {                                          // first row of the tile in this wave's operand
    rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(s_ptr) + first * s_ld, 0,
                                           (unsigned)min((s_rows - first - 1) * s_ld + nblk, 0x7fffffffL), 0x00020000);
  };
  auto load_scales = [&](int g, u32x4 (&v)[KS]) {
    const int sl = mx_lane();
    const unsigned s_off = (unsigned)(s_row0 + 16 * (sl & 3) + (sl >> 2)) * (unsigned)s_ld;
#pragma unroll
    for (int u = 0; u < KS; ++u) {
      const int b0 = (g * KS + u) * 16;
      if (b0 + 16 <= nblk) {
        v[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, s_off, b0, 0));
      } else if (nblk >= 4) {                                                    // the row's end: whole dwords, none of them past it
#pragma unroll
        for (int j = 0; j < 4; ++j) v[u][j] = __builtin_amdgcn_raw_buffer_load_b32(rs, s_off, min(b0 + 4 * j, nblk - 4), 0);
      } else {
        v[u] = u32x4{0u, 0u, 0u, 0u};
        for (int j = 0; j < nblk; ++j) v[u][0] |= (unsigned)__builtin_amdgcn_raw_buffer_load_b8(rs, s_off, j, 0) << (8 * (4 - nblk + j));
      }
    }
  };
  // image of a group: [128-k step][quad of row tiles][q][r16] dwords, byte = row tile of the quad: a 4 x 4 byte transpose within lane quads
  auto put_scales = [&](int img, int g, const u32x4 (&v)[KS]) {
    const int pl = mx_lane();
    const unsigned psel = 0x0c0c0400u + (pl & 3) * 0x0101u;
    char* d = smem + MX_NS * G::STAGE + (unsigned)(img & 1) * G::SIMG + w * 256u + (pl & 3) * 64u + (pl >> 2) * 4u;
#pragma unroll
    for (int u = 0; u < KS; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int live = nblk - ((g * KS + u) * 4 + j) * 4;                      // blocks of this dword inside K; the rest: 2^0 against zero codes
        // (a dword that reaches past K was loaded from the last four bytes of the row)
        const unsigned cut = live >= 4 ? 0u : live <= 0 ? 31u : 8u * (4 - live), keep = live >= 4 ? ~0u : live <= 0 ? 0u : ~0u >> cut;
        const int x = (int)(((v[u][j] >> cut) & keep) | (0x7f7f7f7fu & ~keep));
        const unsigned x0 = (unsigned)__builtin_amdgcn_update_dpp(0, x, 0x00, 0xF, 0xF, true), x1 = (unsigned)__builtin_amdgcn_update_dpp(0, x, 0x55, 0xF, 0xF, true);
        const unsigned x2 = (unsigned)__builtin_amdgcn_update_dpp(0, x, 0xAA, 0xF, 0xF, true), x3 = (unsigned)__builtin_amdgcn_update_dpp(0, x, 0xFF, 0xF, 0xF, true);
        const unsigned y = __builtin_amdgcn_perm(x1, x0, psel) | __builtin_amdgcn_perm(x3, x2, psel) << 16;
        if (w < SQ) *reinterpret_cast<unsigned*>(d + (u * 4 + j) * G::SROW) = y;
      }
  };

  const int wm = (w & 1) * G::WM, wn = (w >> 1) * G::WN;
  const unsigned swz = (unsigned)(q ^ ((r16 >> 1) & 3)) * 16u;
  const unsigned f_addr = (unsigned)r16 * 64u + swz, l4 = l * 4u;                 // a lane's place in a fragment, in a quad of scale bytes
  const unsigned a_base = wm * 64u, b_base = (BM + wn) * 64u, as_base = MX_NS * G::STAGE + (wm >> 6) * 256u, bs_base = MX_NS * G::STAGE + ((BM + wn) >> 6) * 256u;

  int m0, n0;
  coords(id, m0, n0);
  point(m0, n0);
  point_scales(s_of_a ? m0 : n0);
  u32x4 sc[KS];
  int slot = 0, img = 0;                                                         // ring slot of the tile's stage 0, image of its group 0
  load_scales(0, sc);
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < PIECES; ++i) dma(s, s, i);
  mx_wait<0>();
  put_scales(0, 0, sc);

  for (;;) {
    const int nid = id + (int)(gridDim.x >> 3);
    const bool more = nid < lim;
    int nm0 = m0, nn0 = n0;
    if (more) coords(nid, nm0, nn0);
    const int nsf = __builtin_amdgcn_readfirstlane(s_of_a ? nm0 : nn0);
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // both wave groups meet: stages 0, 1 and the first scale image are there
    __builtin_amdgcn_s_waitcnt(0xC07F);                                          // lgkmcnt(0)
    mx_barrier();
#pragma unroll
    for (int i = 0; i < PIECES; ++i) dma(2, slot + 2, i);
    if (w >= 4) mx_barrier();                                                    // the second group runs one barrier behind the first

    u32x4 fa[KS][TM], fb[KS][TN];
    unsigned sa[KS][(TM + 3) / 4], sb[KS];
    auto stage = [&](auto j4_t, int s) {
      constexpr int J4 = decltype(j4_t)::value;                                  // s & 3
      // -- reads: fragments and scales of stage s
      const char* base = smem + (unsigned)((slot + s) & (MX_NS - 1)) * G::STAGE;
      const char* sbase = smem + (unsigned)((img + (s >> 2)) & 1) * G::SIMG + J4 * KS * G::SROW;
#pragma unroll
      for (int u = 0; u < KS; ++u) {
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[u][j] = *reinterpret_cast<const u32x4*>(base + u * G::SUB + b_base + f_addr + j * 1024);
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[u][i] = *reinterpret_cast<const u32x4*>(base + u * G::SUB + a_base + f_addr + i * 1024);
#pragma unroll
        for (int i = 0; i < (TM + 3) / 4; ++i) sa[u][i] = *reinterpret_cast<const unsigned*>(sbase + u * G::SROW + as_base + l4 + 256 * i);
        sb[u] = *reinterpret_cast<const unsigned*>(sbase + u * G::SROW + bs_base + l4);
        if constexpr (TN == 2) sb[u] >>= (wn & 32) / 2;
      }
      __builtin_amdgcn_sched_barrier(0);
      // this wave's pieces of stage s + 1 have landed: still out may be those of s + 2 and, issued behind them, the KS scale loads of J4 = 0
      // (stage 1 landed before the tile began: the first wait leaves the last tile's stores alone)
      if constexpr (J4 == 0) { if (s == 0) __builtin_amdgcn_s_waitcnt(0xC07F); else mx_wait<PIECES>(); }
      else if constexpr (J4 == 1) mx_wait<PIECES + KS>();
      else mx_wait<PIECES>();
      // (at the end of the tile: the next one's stages 0 and 1, then nothing: a stage far past K, whose pieces are zeros)
      int fs = s + 3;
      if (fs >= nst) {
        if (fs == nst) point(nm0, nn0);
        fs = more && fs < nst + 2 ? fs - nst : 1 << 18;
      }
      const bool last = J4 == 0 && s / 4 + 1 == ngr;
      if (last) point_scales(nsf);
      mx_barrier();
      // -- products, and the DMA of stage s + 3 into the slot that every wave has finished with
      __builtin_amdgcn_s_setprio(1);
#define MX_MM(u, i, j)                                                                                                                      \
  {                                                                                                                                         \
    const i32x8 x_ = {(int)fa[u][i][0], (int)fa[u][i][1], (int)fa[u][i][2], (int)fa[u][i][3], 0, 0, 0, 0};                                  \
    const i32x8 y_ = {(int)fb[u][j][0], (int)fb[u][j][1], (int)fb[u][j][2], (int)fb[u][j][3], 0, 0, 0, 0};                                  \
    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(y_, x_, acc[i][j], 4, 4, j, (int)sb[u], (i) & 3, (int)sa[u][(i) / 4]);     \
  }
  /* the empty statement keeps the row where it is: the compiler would sink it behind the DMA and the barrier */
#define MX_ROW(u, i)                                                                                                                        \
  {                                                                                                                                         \
    MX_MM(u, i, 0) MX_MM(u, i, 1) if constexpr (TN == 4) { MX_MM(u, i, 2) MX_MM(u, i, 3) }                                                  \
    if constexpr (TN == 4) asm volatile("" : "+v"(acc[i][0]), "+v"(acc[i][1]), "+v"(acc[i][TN - 2]), "+v"(acc[i][TN - 1])::"memory");       \
    else asm volatile("" : "+v"(acc[i][0]), "+v"(acc[i][1])::"memory");                                                                     \
    __builtin_amdgcn_sched_barrier(0);                                                                                                      \
  }
#define MX_DMA(i) { dma(fs, slot + s + 3, i); __builtin_amdgcn_sched_barrier(0); }
      static_assert(PIECES == 4, "one DMA piece behind each of the first four rows of products");
      MX_ROW(0, 0) MX_DMA(0) MX_ROW(0, 1) MX_DMA(1) MX_ROW(0, 2) MX_DMA(2) MX_ROW(0, 3) MX_DMA(3)
      if constexpr (J4 == 0) load_scales(last ? 0 : s / 4 + 1, sc);
      if constexpr (KS == 1) { MX_ROW(0, 4) MX_ROW(0, 5) MX_ROW(0, 6) } else { MX_ROW(1, 0) MX_ROW(1, 1) MX_ROW(1, 2) }
      if constexpr (J4 == 2) { if (s / 4 + 1 < ngr) put_scales(img + s / 4 + 1, s / 4 + 1, sc); }
      // the other group may start its products while this one's last are in the pipe
      mx_barrier();
      if constexpr (KS == 1) { MX_ROW(0, 7) } else { MX_ROW(1, 3) }
      __builtin_amdgcn_s_setprio(0);
    };
    for (int s = 0; s < nst; s += 4) {
      stage(std::integral_constant<int, 0>{}, s);
      if (s + 1 < nst) stage(std::integral_constant<int, 1>{}, s + 1);
      if (s + 2 < nst) stage(std::integral_constant<int, 2>{}, s + 2);
      if (s + 3 < nst) stage(std::integral_constant<int, 3>{}, s + 3);
    }
    if (w < 4) mx_barrier();
    slot += nst;
    img += ngr;
    mx_wait<0>();                                                                // the next tile's stages 0 and 1 (and no DMA outlives the kernel)
    if (more) put_scales(img, 0, sc);
    const int el = mx_lane();
    const int em = m0 + wm + (el & 15), en = n0 + wn, eq = el >> 4;
    if (p.act) mx_epilogue_pre<TM, TN, 2>(p, acc, em, en, eq);
    else if (p.bias) mx_epilogue_pre<TM, TN, 1>(p, acc, em, en, eq);
    else mx_epilogue_pre<TM, TN, 0>(p, acc, em, en, eq);
    if (!more) return;
    id = nid;
    m0 = nm0;
    n0 = nn0;
  }
}

__global__ __launch_bounds__(512, 2) void gemm_mxfp4_256_kernel(Mx4Args p) { gemm_mxfp4_body<256, 256, 1>(p); }
__global__ __launch_bounds__(512, 2) void gemm_mxfp4_128_kernel(Mx4Args p) { gemm_mxfp4_body<128, 128, 2>(p); }

template <int BM, int BN, int KS>
int mx4_launch(void (*k)(Mx4Args), Mx4Args p, hipStream_t stream) {
  constexpr int lds = Mx4Geo<BM, BN, KS>::LDS;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (attr != hipSuccess) { set_error("gemm_mxfp4: hipFuncSetAttribute: %s", hipGetErrorString(attr)); return HVLM_ERR_LAUNCH; }
  p.tiles_m = cdiv(p.M, BM);
  p.tiles_n = cdiv(p.N, BN);
  const int tiles = p.tiles_m * p.tiles_n;
  hipLaunchKernelGGL(k, dim3((unsigned)std::min(cdiv(tiles, 8) * 8, MX_CUS)), dim3(512), lds, stream, p);
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
  HVLM_REQUIRE(ldas >= K / MX_BLOCK && ldbs >= K / MX_BLOCK && ldas < (1L << 22) && ldbs < (1L << 22), "gemm_mxfp4_nt: leading dimensions of the scales");
  HVLM_REQUIRE(ldc >= N && (!residual || ldr >= N), "gemm_mxfp4_nt: leading dimensions of C / residual");
  HVLM_REQUIRE(act == HVLM_ACT_NONE || act == HVLM_ACT_QUICK_GELU, "gemm_mxfp4_nt: unknown act %d", act);
  HVLM_REQUIRE((long)cdiv(M, 128) * cdiv(N, 128) < (1L << 30), "gemm_mxfp4_nt: too many tiles");
  Mx4Args p{};
  p.A = (const unsigned char*)A; p.B = (const unsigned char*)B; p.as = (const unsigned char*)a_scale; p.bs = (const unsigned char*)b_scale;
  p.C = C; p.bias = (const bf16_t*)bias; p.res = (const bf16_t*)residual;
  p.M = M; p.N = N; p.K = K; p.lda = lda; p.ldb = ldb; p.ldas = ldas; p.ldbs = ldbs; p.ldc = ldc; p.ldr = ldr; p.act = act; p.out_f32 = out_f32;
  if ((long)cdiv(M, 256) * cdiv(N, 256) >= 128) return mx4_launch<256, 256, 1>(gemm_mxfp4_256_kernel, p, as_stream(stream));
  return mx4_launch<128, 128, 2>(gemm_mxfp4_128_kernel, p, as_stream(stream));
}
