// C[M, N] = act(A[M, K] @ B[N, K]^T + bias[N]) + residual[M, N] on MXFP4 operands (format: mxfp4.h), fp32 accumulation.
//
//   C[m, n] = sum over blocks g of 2^(sa[m, g] + sb[n, g] - 254) * sum_{k in g} a[m, k] b[n, k]
//
// is what v_mfma_scale_f32_16x16x128_f8f6f4 computes on fp4 operands: lane (r = l & 15, q = l >> 4) holds block q (32 codes, 16 bytes) of
// row r and that block's E8M0 byte, so 128 k of a fragment are one 16-byte LDS read and one byte of scale (a byte of a register that four
// fragments share).  The weights are the first MFMA operand: a lane's four results are four consecutive columns of one output row.
//
// Bound: the instruction issue of the four waves, one per SIMD.  A product lasts 16 cycles and the matrix pipe queues nothing behind it, so a
// wave that issues anything longer than that between two products idles the pipe.  What follows from it:
//   * a wave owns a quarter of the tile (128 x 128 of 256 x 256: all 256 accumulation registers) and keeps the fragments of two steps, so a
//     step is 64 products without a wait, with the next step's 17 LDS reads and 8 LDS-DMA pieces strewn between them one at a time;
//   * codes go from global memory to LDS by DMA in rows of 128 bytes (rows of 64 halve the L2's rate: 16.7 instead of 32 TB/s), addressed by a
//     register that runs along, with 16-byte chunks permuted by c ^ (row & 7): eight rows of a fragment read fall into eight bank groups;
//   * scales are tiled once per call by a kernel of their own (3.6 us for 867 + 12 288 rows of 4096, 5.3 for 13 872 + 22 016) so that a step's fit one dword per four fragments:
//     gathered row by row inside the K loop they cost a quarter of it (0.15 of 0.78 us a step);
//   * workgroups are persistent and the ring runs on into the next tile, whose first 512 k land during the last of this one.
// 13872 x 22016 x 4096: median 646 us = 3.9 PFLOP/s over inputs that change from call to call (the best of such runs 579 - 612; two groups of four
// waves one barrier apart, the shape of gemm_pp.hip, 723 at best).  Without DMA and scales a step would take 0.46 us instead of 0.62, the products alone 0.43; the
// rest is the tiles' ends (vision shapes with K = 1024 are mostly that: 90 us where the result's bytes need 44).
// Registers: the 256 x 256 kernel keeps 132 scalars in lanes of vector registers (the 128 x 128 one 55), tile coordinates and the epilogue's addresses; they are
// saved and fetched between tiles, the body of the K loop touches none of them.
#include "mxfp4.h"
#include <algorithm>
#include <type_traits>

namespace hvlm {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((address_space(3))) void* lds_ptr_t;

struct Mx4Args {
  const unsigned char *A, *B;
  const unsigned char* ts;                 // scales of A's rows, then of B's, tiled (mx4_tile_scales_kernel)
  void* C;
  const bf16_t *bias, *res;
  int M, N, K;
  long lda, ldb, ldc, ldr;
  int act, out_f32, tiles_m, tiles_n;
};

constexpr int MX_GROUP_M = 8;             // row panels per group of the tile order
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
// An accumulator fragment, moved to ordinary registers where it is used: left to the compiler, all of a wave's 256 would move at once.
__device__ __forceinline__ f32x4 mx_take(const f32x4& c) {
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(x) : "a"(c[e]));
    v[e] = x;
  }
  return v;
}

// The lane's number, computed where it is used: registers of the K loop are full, and what is derived from threadIdx once is spilled.
__device__ __forceinline__ int mx_lane() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}

// Results of a wave, rows m .. m + 16 TM - 1, columns n .. n + 16 TN - 1, sixteen rows at a time through 4 KB of the wave's own LDS: a lane
// holds four consecutive columns of one row of each fragment, and stores (or adds a residual to) eight consecutive columns where the
// lanes of an instruction cover whole lines.  16-byte chunks are permuted by c ^ row.  With a residual or float32 results the rows go
// through LDS in fp32, 64 columns at a time; otherwise rounded.  Stores may be unaligned (odd leading dimensions).
// PRE: 0 = nothing, 1 = bias, 2 = bias (if any) and QuickGELU.  One straight-line body per combination: with the choices inside, the
// accumulators meet in the branches and are spilled.
template <int TM, int TN, int PRE, bool RES, bool F32>
__device__ __forceinline__ void mx_epilogue(const Mx4Args& p, const f32x4 (&acc)[TM][TN], int m, int n, char* buf) {
  typedef u32x4 __attribute__((aligned(2))) u32x4_u;
  typedef f32x4 __attribute__((aligned(4))) f32x4_u;
  constexpr bool WIDE = RES || F32;
  constexpr int TP = WIDE ? 4 : TN;                                              // fragments of a pass
  constexpr int LPR = WIDE ? 8 : 2 * TP;                                         // lanes that share a row, eight columns each
  constexpr int RPI = 64 / LPR, NI = 16 / RPI;                                   // rows of one instruction, instructions of sixteen rows
  constexpr int RB = WIDE ? 256 : 32 * TP, CH = RB / 16 - 1, ES = F32 ? 4 : 2;   // bytes of a row in LDS, its chunks - 1, bytes of a result
  const int l = mx_lane(), r16 = l & 15, q = l >> 4;
  const int cl = l & (LPR - 1), rl = l / LPR;                                    // this lane's columns / row behind the exchange
  // where fragment j is written: ^ 64 j (a chunk a quarter) or ^ 32 j (half a chunk)
  const unsigned at = r16 * RB + (WIDE ? (q ^ (r16 & CH)) * 16 : ((q >> 1) ^ (r16 & CH)) * 16 + (q & 1) * 8);
  // where row rl + RPI k of the sixteen is read: the row's permutation differs from k to k in bits that RPI k does not share with rl
  auto from = [&](int k, int c) { return (unsigned)((rl + RPI * k) * RB + (c ^ ((rl + RPI * k) & CH)) * 16); };
  const int rows = p.M - m;                                                      // rows of this wave inside C
#pragma unroll
  for (int h = 0; h < TN / TP; ++h) {
    const int col = n + 16 * TP * h, cols = p.N - col;
    const int mine = 8 * cl + 8 <= cols ? rows : 0;                              // rows whose eight columns of this lane are all inside C
    float b[TP][4];
    if constexpr (PRE > 0) {
#pragma unroll
      for (int j = 0; j < TP; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) b[j][e] = p.bias ? bf2f(p.bias[min(col + 16 * j + 4 * q + e, p.N - 1)]) : 0.f;
    }
    const char* const rbase = reinterpret_cast<const char*>(p.res) + ((long)m * p.ldr + col) * 2;
    char* const cbase = reinterpret_cast<char*>(p.C) + ((long)m * p.ldc + col) * ES;
    const unsigned rv = (unsigned)rl * (unsigned)p.ldr * 2u + cl * 16u, cv = (unsigned)rl * (unsigned)p.ldc * ES + cl * 8u * ES;
    auto residual = [&](int i, int k) {
      u32x4 x = {0u, 0u, 0u, 0u};
      if (16 * i + RPI * k + rl < mine) x = *reinterpret_cast<const u32x4_u*>(rbase + (long)(16 * i + RPI * k) * p.ldr * 2 + rv);
      return x;
    };
    u32x4 rn[NI];                                                                // (a row's residual is read before its results are stored: C may be the residual)
    if constexpr (RES) {
#pragma unroll
      for (int k = 0; k < NI; ++k) rn[k] = residual(0, k);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TP; ++j) {
        f32x4 v = mx_take(acc[i][TP * h + j]);
        if constexpr (PRE > 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] += b[j][e];
            if constexpr (PRE == 2) v[e] *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.702f * 1.4426950408889634f * v[e]));
          }
        }
        if constexpr (WIDE) *reinterpret_cast<f32x4*>(buf + (at ^ (64u * j))) = v;
        else *reinterpret_cast<u32x2*>(buf + (at ^ (32u * j))) = u32x2{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3])};
      }
      u32x4 rc[NI];
      if constexpr (RES) {
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          rc[k] = rn[k];
          if (i + 1 < TM) rn[k] = residual(i + 1, k);
        }
      }
#pragma unroll
      for (int k = 0; k < NI; ++k) {
        char* const o = cbase + (long)(16 * i + RPI * k) * p.ldc * ES;
        const bool in = 16 * i + RPI * k + rl < mine;
        if constexpr (!WIDE) {
          const u32x4 d = *reinterpret_cast<const u32x4*>(buf + from(k, cl));
          if (in) *reinterpret_cast<u32x4_u*>(o + cv) = d;
        } else {
          f32x4 x = *reinterpret_cast<const f32x4*>(buf + from(k, 2 * cl)), y = *reinterpret_cast<const f32x4*>(buf + from(k, 2 * cl + 1));
          if constexpr (RES) {
            x += f32x4{bf_lo(rc[k][0]), bf_hi(rc[k][0]), bf_lo(rc[k][1]), bf_hi(rc[k][1])};
            y += f32x4{bf_lo(rc[k][2]), bf_hi(rc[k][2]), bf_lo(rc[k][3]), bf_hi(rc[k][3])};
          }
          if (in) {
            if constexpr (F32) {
              *reinterpret_cast<f32x4_u*>(o + cv) = x;
              *reinterpret_cast<f32x4_u*>(o + cv + 16) = y;
            } else {
              *reinterpret_cast<u32x4_u*>(o + cv) = u32x4{pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]), pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3])};
            }
          }
        }
      }
      if (cols > 0 && cols < 16 * TP && (cols & 7)) {                            // the last, partial eight columns of C: an element a lane
#pragma unroll 1
        for (int e = l; e < 128; e += 64) {
          const int r = e >> 3, c = (cols & ~7) + (e & 7);
          if (16 * i + r < rows && c < cols) {
            const long row = m + 16 * i + r;
            if constexpr (!WIDE) {
              reinterpret_cast<bf16_t*>(p.C)[row * p.ldc + col + c] = *reinterpret_cast<const bf16_t*>(buf + r * RB + ((c >> 3) ^ (r & CH)) * 16 + (c & 7) * 2);
            } else {
              float x = *reinterpret_cast<const float*>(buf + r * RB + ((c >> 2) ^ (r & CH)) * 16 + (c & 3) * 4);
              if constexpr (RES) x += bf2f(p.res[row * p.ldr + col + c]);
              if constexpr (F32) reinterpret_cast<float*>(p.C)[row * p.ldc + col + c] = x;
              else reinterpret_cast<bf16_t*>(p.C)[row * p.ldc + col + c] = f2bf(x);
            }
          }
        }
      }
    }
  }
}

template <int TM, int TN, int PRE>
__device__ __forceinline__ void mx_epilogue_pre(const Mx4Args& p, const f32x4 (&acc)[TM][TN], int m, int n, char* buf) {
  if (p.out_f32) {
    if (p.res) mx_epilogue<TM, TN, PRE, true, true>(p, acc, m, n, buf);
    else mx_epilogue<TM, TN, PRE, false, true>(p, acc, m, n, buf);
  } else {
    if (p.res) mx_epilogue<TM, TN, PRE, true, false>(p, acc, m, n, buf);
    else mx_epilogue<TM, TN, PRE, false, false>(p, acc, m, n, buf);
  }
}

// c += W X^T for one 16 x 16 fragment over 128 k; the scale bytes are byte J / I of sw / sx.  In assembly because the accumulators of a
// 256 x 256 tile fill all 256 accumulation registers: the builtin's result is a register of its own, and with none free it is copied
// back and forth.  (Operands come from LDS reads, which the compiler waits for; nothing reads a result before mx_settle.)
template <int J, int I>
__device__ __forceinline__ void mx_mfma(f32x4& c, u32x4 wf, u32x4 xf, unsigned sw, unsigned sx) {
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
               : "+a"(c) : "v"(wf), "v"(xf), "v"(sw), "v"(sx), "n"(J & 1), "n"(I & 1), "n"(J >> 1), "n"(I >> 1));
}
// wait states between the accumulators' initialisation and the first product, between the last product and the first use of its result (at
// most 18 are needed), and nothing may move across
__device__ __forceinline__ void mx_settle() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <int BM, int BN, int KS>
struct Mx4Geo {
  static constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16;
  static constexpr unsigned SLOT = (BM + BN) * 128;                              // ring slot: 256 k of both operands
  static constexpr int SLOTS = 2 * KS;
  static constexpr unsigned SIMG = 4 * KS * (BM + BN) * 4;                       // scale bytes of a group (512 KS k)
  static constexpr unsigned RING = SLOTS * SLOT, EPI = RING + 2 * SIMG;
  static constexpr int LDS = (int)EPI + 4 * 4096;
  static constexpr int PIECES = (BM + BN) / 32;                                  // LDS-DMA instructions per wave and slot
  static constexpr int SQW = (BM + BN) / 256;                                    // quads of row tiles whose scales a wave stages
};

// (a __device__ template under plain __global__ wrappers, as in gemm_pp.hip)
template <int BM, int BN, int KS>
__device__ __forceinline__ void gemm_mxfp4_body(const Mx4Args& p) {
  using G = Mx4Geo<BM, BN, KS>;
  constexpr int TM = G::TM, TN = G::TN, PIECES = G::PIECES, SQW = G::SQW, SLOADS = KS * SQW;
  static_assert(TM == TN && KS * TM == 8 && PIECES * KS == 16 && SLOADS == 2, "the schedule of a step");
  extern __shared__ __attribute__((aligned(128))) char smem[];
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), l = t & 63, r16 = l & 15, q = l >> 4;
  const int tiles = p.tiles_m * p.tiles_n, per = (tiles + 7) / 8;
  // a tile's K in whole groups of four steps (a step = 128 KS k): ring slot and registers are known at compile time (what lies past K is zeros)
  const int nblk = p.K / MX_BLOCK, ngr = (nblk + 16 * KS - 1) / (16 * KS);

  // tile order: XCD x (blockIdx & 7) owns tiles x * per .. of the grouped order, its workgroups take every (gridDim / 8)-th of them
  const int lim = min(tiles, ((int)(blockIdx.x & 7) + 1) * per);
  int id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if (id >= lim) return;
  auto coords = [&](int tile, int& m0, int& n0) {
    const int gsz = MX_GROUP_M * p.tiles_n, grp = tile / gsz, first = grp * MX_GROUP_M;
    const int gm = min(MX_GROUP_M, p.tiles_m - first), in = tile - grp * gsz;
    m0 = (first + in % gm) * BM;
    n0 = (in / gm) * BN;
  };

  // codes: DMA piece j of wave w = rows 8 (w + 4 j) .. + 7 of the stacked (A rows, B rows) image, 128 bytes each (half of a line would cost the
  // L2 a whole one), lane = (row l >> 3, chunk position l & 7)
  const int chunk = (l & 7) ^ (l >> 3);
  const unsigned off_a = (unsigned)(8 * w + (l >> 3)) * (unsigned)p.lda + (unsigned)chunk * 16u;
  const unsigned off_b = (unsigned)(8 * w + (l >> 3)) * (unsigned)p.ldb + (unsigned)chunk * 16u;
  // descriptors of a tile's operands end with the last valid row; offsets within a tile stay below 2^31 (checked by the host), 2^31 and more
  // reads as zero
  __amdgpu_buffer_rsrc_t ra, rb;
  auto point = [&](int m0, int n0) {
    const long ba = (long)(p.M - m0 - 1) * p.lda + p.K / 2, bb = (long)(p.N - n0 - 1) * p.ldb + p.K / 2;
    ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.A) + (long)m0 * p.lda, 0, (unsigned)min(ba, 0x7fffffffL), 0x00020000);
    rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.B) + (long)n0 * p.ldb, 0, (unsigned)min(bb, 0x7fffffffL), 0x00020000);
  };
  // DMA piece j of the 256 k number s into ring slot `slot`; pieces of a slot are issued in order (va / vb run along the rows).  Blocks past K
  // come as zeros: those lanes start past the descriptor.
  unsigned va = 0, vb = 0;
  auto dma = [&](int s, int slot, int j) {
    constexpr int JA = BM / 32;                                                   // pieces that are rows of A
    if (j == 0) {
      const bool live = s * 8 + chunk < nblk;
      va = live ? off_a : 0x80000000u;
      vb = live ? off_b : 0x80000000u;
    }
    unsigned wb = (unsigned)w * 1024u;
    asm volatile("" : "+s"(wb));                                                  // (not a register for every piece's place)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(j < JA ? ra : rb, (lds_ptr_t)(smem + wb + ((unsigned)slot * G::SLOT + (unsigned)j * 4096u)), 16, j < JA ? va : vb,
                                             (unsigned)s * 128u, 0, 0);
    if (j < JA) va += 32u * (unsigned)p.lda; else vb += 32u * (unsigned)p.ldb;
  };
  // scales: a quad of row tiles (64 rows) and a group of four steps are KS KB of the tiled copy, one DMA piece each; wave w brings SQW quads
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.ts), 0, 0x7fffffffu, 0x00020000);
  const unsigned quad_bytes = (unsigned)ngr * 1024u * KS;
  auto scale_base = [&](int m0, int n0) {                                       // of this wave's first quad of a tile
    const int first = w < 2 ? m0 / 64 + SQW * w : p.tiles_m * (BM / 64) + n0 / 64 + SQW * (w - 2);
    return (unsigned)first * quad_bytes;
  };
  auto dma_scales = [&](unsigned base, int g, int img) {
#pragma unroll
    for (int x = 0; x < SLOADS; ++x)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(smem + G::RING + (unsigned)(img & 1) * G::SIMG + ((w * SQW + x / KS) * KS + x % KS) * 1024u), 16,
                                               (unsigned)l * 16u, base + (x / KS) * quad_bytes + (unsigned)(g * KS + x % KS) * 1024u, 0, 0);
  };

  const int wm = (w & 1) * G::WM, wn = (w >> 1) * G::WN;
  // a lane's place in a fragment (chunk q of the first 128 k; ^ 64: of the second), in a quad of scale bytes
  const unsigned f_addr = (unsigned)r16 * 128u + (unsigned)(q ^ (r16 & 7)) * 16u, l4 = l * 4u;
  struct Frag {
    u32x4 a[KS][TM], b[KS][TN];
    unsigned sa[KS][TM / 4], sb[KS][TN / 4];
  } f0, f1;
  // item c of what step j4 of a group reads: 0 .. 7 the fragments of B, which the first products need all of, 8 .. 15 those of A, 16 the scales
  auto read = [&](Frag& f, int img, int j4, int c) {
    const char* base = smem + (unsigned)(KS == 1 ? j4 >> 1 : j4) * G::SLOT;
    if (c == 16) {
      const char* sbase = smem + G::RING + (unsigned)(img & 1) * G::SIMG + (unsigned)j4 * KS * 256u + l4;
#pragma unroll
      for (int u = 0; u < KS; ++u)
#pragma unroll
        for (int i = 0; i < TM / 4; ++i) {
          f.sb[u][i] = *reinterpret_cast<const unsigned*>(sbase + u * 256 + ((BM + wn) / 64 + i) * 1024 * KS);
          f.sa[u][i] = *reinterpret_cast<const unsigned*>(sbase + u * 256 + (wm / 64 + i) * 1024 * KS);
        }
      return;
    }
    const int u = (c % 8) / TN, i = c % TN;
    const char* at = base + ((KS == 1 ? j4 & 1 : u) ? f_addr ^ 64u : f_addr);
    if (c < 8) f.b[u][i] = *reinterpret_cast<const u32x4*>(at + (BM + wn + 16 * i) * 128);
    else f.a[u][i] = *reinterpret_cast<const u32x4*>(at + (wm + 16 * i) * 128);
  };

  int m0, n0;
  coords(id, m0, n0);
  point(m0, n0);
  unsigned sbase = scale_base(m0, n0);
  int img = 0;                                                                   // image of the tile's group 0
  dma_scales(sbase, 0, 0);
#pragma unroll
  for (int s = 0; s < G::SLOTS; ++s)
#pragma unroll
    for (int j = 0; j < PIECES; ++j) dma(s, s, j);
  mx_wait<0>();
  mx_barrier();
#pragma unroll
  for (int c = 0; c < 17; ++c) read(f0, 0, 0, c);

  for (;;) {
    const int nid = id + (int)(gridDim.x >> 3);
    const bool more = nid < lim;
    int nm0 = m0, nn0 = n0;
    if (more) coords(nid, nm0, nn0);
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) asm volatile("" : "+a"(acc[i][j]));
    mx_settle();

    for (int g = 0; g < ngr; ++g) {
      const bool last = g + 1 == ngr;                                            // then what is fetched ahead belongs to the next tile
      auto step = [&](auto j4_t, const Frag& cur, Frag& nxt) {
        constexpr int J4 = decltype(j4_t)::value;
        // Beside the products of a step the fragments of the next one are read.
        // KS = 1: a slot is two steps.  The even step's reads are the last of their slot: behind the barrier in the middle of that step the slot
        // is filled again, by the end of the odd step.  The odd step begins when the other slot has landed (still out: the six pieces
        // issued in the even step, and the scales').
        // KS = 2: a slot is one step; it is free and filled again when the step begins, for four steps later.  (Then still out: the pieces of
        // two steps, and the scales' among them.  A tile's steps 1 and 2 landed before it began: their waits leave the last tile's stores
        // alone.)
        if constexpr (KS == 2) {
          if (J4 < 2 && g == 0) __builtin_amdgcn_s_waitcnt(0xC07F);
          else if constexpr (J4 == 1 || J4 == 2) mx_wait<2 * PIECES + SLOADS>();
          else mx_wait<2 * PIECES>();
          mx_barrier();
        } else if constexpr (J4 & 1) {
          if constexpr (J4 == 1) mx_wait<6 + SLOADS>(); else mx_wait<6>();
          mx_barrier();
        }
        // the 256 k that go where this step's were: two slots / four steps on (past the last tile: far past K, whose pieces are zeros)
        if (J4 == 0 && last) point(nm0, nn0);
        constexpr int SL = KS == 1 ? J4 >> 1 : J4;
        const int fs = !last ? G::SLOTS * (g + 1) + SL : more ? SL : 1 << 18;
        if constexpr (J4 == 0) {                                                   // the next group's scales
          if (last) sbase = scale_base(nm0, nn0);
          dma_scales(sbase, last ? 0 : g + 1, img + g + 1);
          __builtin_amdgcn_sched_barrier(0);
        }
        // What is issued beside product k of a step, one small piece at a time: the matrix pipe holds little more than the
        // product it works on, so whatever takes longer to issue than a product to compute leaves it idle.
        auto beside = [&](auto k_t) {
          constexpr int k = decltype(k_t)::value;
          if constexpr (KS == 1) {
            if constexpr (k == 0) read(nxt, J4 == 3 ? img + g + 1 : img + g, (J4 + 1) & 3, 16);
            else if constexpr ((k & 1) && k < 32) read(nxt, img, (J4 + 1) & 3, k >> 1);
            if constexpr (J4 & 1) {
              if constexpr (k % 4 == 2 && k < 40) dma(fs, SL, 6 + k / 4);
            } else {
              if constexpr (k == 40) { __builtin_amdgcn_s_waitcnt(0xC07F); mx_barrier(); }
              else if constexpr (k > 40 && k % 4 == 2) dma(fs, SL, (k - 42) / 4);
            }
          } else {
            if constexpr (k == 0) read(nxt, J4 == 3 ? img + g + 1 : img + g, (J4 + 1) & 3, 16);
            if constexpr (k < 16) read(nxt, img, (J4 + 1) & 3, k);
            else if constexpr (k % 2 == 0) dma(fs, SL, (k - 16) / 2);
          }
          __builtin_amdgcn_sched_barrier(0);
        };
#define MX_ONE(r, j) { mx_mfma<(j) & 3, ((r) % TM) & 3>(acc[(r) % TM][j], cur.b[(r) / TM][j], cur.a[(r) / TM][(r) % TM], cur.sb[(r) / TM][(j) / 4], \
                                                          cur.sa[(r) / TM][((r) % TM) / 4]); __builtin_amdgcn_sched_barrier(0);                        \
                        beside(std::integral_constant<int, (r) * TN + (j)>{}); }
#define MX_ROW(r) { MX_ONE(r, 0) MX_ONE(r, 1) MX_ONE(r, 2) MX_ONE(r, 3)                                                                     \
                    if constexpr (TN == 8) { MX_ONE(r, TN - 4) MX_ONE(r, TN - 3) MX_ONE(r, TN - 2) MX_ONE(r, TN - 1) } }
        MX_ROW(0) MX_ROW(1) MX_ROW(2) MX_ROW(3) MX_ROW(4) MX_ROW(5) MX_ROW(6) MX_ROW(7)
      };
      step(std::integral_constant<int, 0>{}, f0, f1);
      step(std::integral_constant<int, 1>{}, f1, f0);
      step(std::integral_constant<int, 2>{}, f0, f1);
      step(std::integral_constant<int, 3>{}, f1, f0);
    }
    img += ngr;
    mx_settle();
    // KS = 2: the next tile's steps 1 and 2 have landed before the stores queue up behind them.  No DMA outlives the kernel.
    if (!more) mx_wait<0>(); else if constexpr (KS == 2) mx_wait<PIECES>();
    char* const buf = smem + G::EPI + w * 4096;
    const int em = m0 + wm, en = n0 + wn;
    if (p.act) mx_epilogue_pre<TM, TN, 2>(p, acc, em, en, buf);
    else if (p.bias) mx_epilogue_pre<TM, TN, 1>(p, acc, em, en, buf);
    else mx_epilogue_pre<TM, TN, 0>(p, acc, em, en, buf);
    if (!more) return;
    id = nid;
    m0 = nm0;
    n0 = nn0;
  }
}

// Scales as the K loop reads them: for every quad of row tiles (64 rows, QA of them A's) and 128 k, 256 bytes [q][r] of dwords whose byte t is
// the scale of row 16 t + r, block q.  Row-major, a lane would fetch 4 of every 128 bytes it touches, for every tile anew; rows past the
// end and blocks past K become 2^0 (against zero codes).  One workgroup: a quad x 32 of those 128 k.
__global__ __launch_bounds__(256) void mx4_tile_scales_kernel(const unsigned char* __restrict__ as, const unsigned char* __restrict__ bs,
                                                              unsigned char* __restrict__ ts, int M, int N, int nblk, long ldas, long ldbs, int QA,
                                                              int steps) {
  __shared__ __attribute__((aligned(16))) unsigned char im[32][272];              // (16 bytes of padding: the rows start in different banks)
  const int t = threadIdx.x, st = t & 31, s = blockIdx.y * 32 + st;
  const bool is_a = (int)blockIdx.x < QA;
  const int row0 = ((int)blockIdx.x - (is_a ? 0 : QA)) * 64, rows = is_a ? M : N;
  const unsigned char* const p = is_a ? as : bs;
  const long ld = is_a ? ldas : ldbs;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = (t >> 5) + 8 * h;
    unsigned d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + 16 * i + r;
      d[i] = 0x7f7f7f7fu;
      if (row < rows) {
        const unsigned char* c = p + row * ld + 4 * s;
        if (4 * s + 4 <= nblk) __builtin_memcpy(&d[i], c, 4);                     // any alignment
        else
          for (int e = 0; 4 * s + e < nblk; ++e) d[i] = (d[i] & ~(255u << (8 * e))) | (unsigned)c[e] << (8 * e);
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const unsigned sel = 0x0c0c0400u + q * 0x0101u;
      *reinterpret_cast<unsigned*>(&im[st][q * 64 + r * 4]) = __builtin_amdgcn_perm(d[1], d[0], sel) | __builtin_amdgcn_perm(d[3], d[2], sel) << 16;
    }
  }
  __syncthreads();
  const int left = min(32, steps - (int)blockIdx.y * 32);
  unsigned char* o = ts + ((long)blockIdx.x * steps + blockIdx.y * 32) * 256;
  for (int c = t; c < left * 16; c += 256) *reinterpret_cast<u32x4*>(o + c * 16) = *reinterpret_cast<const u32x4*>(&im[c >> 4][(c & 15) * 16]);
}

__global__ __launch_bounds__(256, 1) void gemm_mxfp4_256_kernel(Mx4Args p) { gemm_mxfp4_body<256, 256, 1>(p); }
__global__ __launch_bounds__(256, 1) void gemm_mxfp4_128_kernel(Mx4Args p) { gemm_mxfp4_body<128, 128, 2>(p); }

// Two shapes of tile.  A workgroup takes about 0.62 us per 128 k of a 256 x 256 tile and 3 us to write it, 0.6 us per 256 k of a 128 x 128 tile
// and 1 us to write that; filling and draining cost 7 and 5 us once.  Rounds of 256 workgroups decide (256 / 128, microseconds measured):
// 867 x 12288 x 4096 35.4 / 36.1, 867 x 22016 x 4096 60 / 56, 867 x 4096 x 11008 65 / 33, 2000 x 2000 x 2048 22.7 / 13.4,
// 25700 x 4096 x 1024 92 / 109, 13872 x 22016 x 4096 610 / 760.
struct Mx4Plan {
  int tile, qa, qb, steps;                 // quads of row tiles of A and B, 128-k steps of a row (whole groups)
  size_t ws;
};
Mx4Plan mx4_plan(int M, int N, int K) {
  Mx4Plan r;
  const long r256 = cdiv((long)cdiv(M, 256) * cdiv(N, 256), MX_CUS), r128 = cdiv((long)cdiv(M, 128) * cdiv(N, 128), MX_CUS);
  const long t256 = 700 + r256 * (62L * cdiv(K, 128) + 300), t128 = 500 + r128 * (60L * cdiv(K, 256) + 100);
  r.tile = t256 < t128 ? 256 : 128;
  const int ks = r.tile == 256 ? 1 : 2;
  r.qa = cdiv(M, r.tile) * (r.tile / 64);
  r.qb = cdiv(N, r.tile) * (r.tile / 64);
  r.steps = cdiv(K, 512 * ks) * 4 * ks;
  r.ws = (size_t)(r.qa + r.qb) * r.steps * 256;
  return r;
}

template <int BM, int BN, int KS>
int mx4_launch(void (*k)(Mx4Args), Mx4Args p, hipStream_t stream) {
  constexpr int lds = Mx4Geo<BM, BN, KS>::LDS;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (attr != hipSuccess) { set_error("gemm_mxfp4: hipFuncSetAttribute: %s", hipGetErrorString(attr)); return HVLM_ERR_LAUNCH; }
  p.tiles_m = cdiv(p.M, BM);
  p.tiles_n = cdiv(p.N, BN);
  const int tiles = p.tiles_m * p.tiles_n;
  hipLaunchKernelGGL(k, dim3((unsigned)std::min(cdiv(tiles, 8) * 8, MX_CUS)), dim3(256), lds, stream, p);
  return check_launch("gemm_mxfp4_nt");
}

}  // namespace
}  // namespace hvlm

using namespace hvlm;

extern "C" size_t hvlm_gemm_mxfp4_ws_bytes(int M, int N, int K) { return M > 0 && N > 0 && K > 0 ? mx4_plan(M, N, K).ws : 0; }

extern "C" int hvlm_gemm_mxfp4_nt(const void* A, const void* a_scale, const void* B, const void* b_scale, void* C, int M, int N, int K, long lda,
                                  long ldas, long ldb, long ldbs, long ldc, const void* bias, const void* residual, long ldr, int act, int out_f32,
                                  void* ws, void* stream) {
  HVLM_REQUIRE(A && a_scale && B && b_scale && C && ws, "gemm_mxfp4_nt: null pointer");
  HVLM_REQUIRE(M > 0 && N > 0 && K > 0 && K % MX_BLOCK == 0, "gemm_mxfp4_nt: M=%d, N=%d must be positive, K=%d a positive multiple of 32", M, N, K);
  HVLM_REQUIRE(lda >= K / 2 && ldb >= K / 2 && lda % 16 == 0 && ldb % 16 == 0 && ((uintptr_t)A & 15) == 0 && ((uintptr_t)B & 15) == 0,
               "gemm_mxfp4_nt: rows of codes must be 16-byte aligned");
  HVLM_REQUIRE(lda < (1L << 22) && ldb < (1L << 22), "gemm_mxfp4_nt: leading dimensions of the codes must be below 4 MiB");
  HVLM_REQUIRE(ldas >= K / MX_BLOCK && ldbs >= K / MX_BLOCK, "gemm_mxfp4_nt: leading dimensions of the scales");
  HVLM_REQUIRE(ldc >= N && ldc < (1L << 26) && (!residual || (ldr >= N && ldr < (1L << 26))), "gemm_mxfp4_nt: leading dimensions of C / residual");
  HVLM_REQUIRE(act == HVLM_ACT_NONE || act == HVLM_ACT_QUICK_GELU, "gemm_mxfp4_nt: unknown act %d", act);
  HVLM_REQUIRE((long)cdiv(M, 128) * cdiv(N, 128) < (1L << 30), "gemm_mxfp4_nt: too many tiles");
  HVLM_REQUIRE(((uintptr_t)ws & 15) == 0, "gemm_mxfp4_nt: the workspace must be 16-byte aligned");
  const Mx4Plan plan = mx4_plan(M, N, K);
  HVLM_REQUIRE(plan.ws < (1UL << 31), "gemm_mxfp4_nt: the scales of %d + %d rows of %d are too many for one call", M, N, K);
  Mx4Args p{};
  p.A = (const unsigned char*)A; p.B = (const unsigned char*)B; p.ts = (const unsigned char*)ws;
  p.C = C; p.bias = (const bf16_t*)bias; p.res = (const bf16_t*)residual;
  p.M = M; p.N = N; p.K = K; p.lda = lda; p.ldb = ldb; p.ldc = ldc; p.ldr = ldr; p.act = act; p.out_f32 = out_f32;
  hipLaunchKernelGGL(mx4_tile_scales_kernel, dim3((unsigned)(plan.qa + plan.qb), (unsigned)cdiv(plan.steps, 32)), dim3(256), 0, as_stream(stream),
                     (const unsigned char*)a_scale, (const unsigned char*)b_scale, (unsigned char*)ws, M, N, K / MX_BLOCK, ldas, ldbs, plan.qa, plan.steps);
  const int rc = check_launch("gemm_mxfp4_nt");
  if (rc) return rc;
  return plan.tile == 256 ? mx4_launch<256, 256, 1>(gemm_mxfp4_256_kernel, p, as_stream(stream))
                          : mx4_launch<128, 128, 2>(gemm_mxfp4_128_kernel, p, as_stream(stream));
}
