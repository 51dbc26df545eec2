// KV cache held in MXFP4 (format: mxfp4.h) and single-token attention over it.
//
// Layout, per K and V: codes [B, Hkv, max_len, dh / 2], scales [B, Hkv, max_len, dh / 32] — the rows of one head are contiguous (a
// 128-wide key is 64 + 4 bytes), blocks run along the head dimension, so a token is appended without touching its neighbours.
//
// Attention: out[b, h] = sum_t softmax_t(scale * q[b, h] . k[b, h / G, t]) v[b, h / G, t] over the lens[b] first rows (G = H / Hkv).
// A wave takes 32 keys at a time of one (sample, KV head) with all G <= 16 query heads of the group as the columns of its MFMAs
// (v_mfma_f32_16x16x32_bf16; K and V are de-quantised to bf16 in registers, which is exact):
//   S^T [16 keys x heads] = K Q^T: lane (r = l & 15, g = l >> 4) holds key 4 (r & 3) + (r >> 2) and the dh / 4 dims of quarter g in one read;
//     the lane's four results are then keys 4 i + g of head r;
//   O^T [dh x heads] += V^T P^T: the same lane supplies the probabilities of the keys 4 i + g — where they already are, nothing is
//     exchanged — and V is read in that order too: one read covers four whole rows, lane r its dh / 16 dims of them; the pairs
//     of adjacent dims that the conversion yields are turned into pairs of keys by v_perm.
// The codes of a tile (K 2 KB, V 2 KB) come by LDS-DMA, 1 KB of consecutive rows an instruction, into a ring of the wave's own, three tiles ahead
// and without a barrier; loaded into registers in fragment order a tile would take 20 instructions instead of 6 and the address units
// would bound the kernel.  A tile's scales are two more.
// Softmax: running maximum and sum per wave in fp32.  P enters the second product as two bf16 terms, its rounding and the rounded rest, 2^-16 relative
// in all: with the first alone keys of equal scores would all be off by the same up to 2^-8, as much as the result's own rounding.  Up to eight heads
// leave half of the sixteen columns free: column r + 8 repeats head r and carries the rests, so that the second term costs no product; nine to sixteen
// heads have it in products of its own.  The waves of a workgroup take alternate tiles and merge in LDS; the
// workgroups of a split sample write (max, sum, unnormalised row) in fp32 and a second kernel joins them in order: no atomics.
// Rows at and past lens[b] are never read.
//
// Bound by the read of the cache when there are many keys: 32 samples x 32 heads, 98 MB, 32 - 34 us; 8 samples x 8 KV
// heads of up to 32768 keys, 214 MB, 52 us and 4.6 us to join (from HBM at the rate of a copy, 4.79 TB/s, these take 20 and 45 us; what earlier
// calls left in the last-level cache comes faster).  Short caches by latency: one sample x 32 heads x 967 keys 9.6 us.  (Medians.  Of these the second term of P is
// 0.5 to 1.7 us, 5 % at most.)
#include "mxfp4.h"

namespace hvlm {
namespace {

constexpr int KV4_WAVES = 4;                // of a workgroup of the attention
constexpr int KV4_WIDE = 8;                 // of its form for short caches
constexpr int KV4_TILE = 32;               // keys per wave and step

// ---- append -----------------------------------------------------------------------------------------------------------------------
// item = 8 elements (one dword of codes); four adjacent lanes share a block
template <int DH>
__global__ __launch_bounds__(256) void kv4_append_kernel(const bf16_t* __restrict__ qkv, long ld, unsigned char* __restrict__ kc,
                                                         unsigned char* __restrict__ ks, unsigned char* __restrict__ vc,
                                                         unsigned char* __restrict__ vs, const int32_t* __restrict__ start,
                                                         const int32_t* __restrict__ count, int B, int S, long max_len, int H, int Hkv) {
  constexpr int CH = DH / 8;
  const long per_row = 2L * Hkv * CH, total = (long)B * S * per_row;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long row = i / per_row;
    const int r = (int)(i - row * per_row), hh = r / CH, c = r % CH;          // hh: 0 .. Hkv - 1 keys, Hkv .. 2 Hkv - 1 values
    const int b = (int)(row / S), s = (int)(row - (long)b * S);
    const long pos = (start ? start[b] : 0) + (long)s;
    if (pos < 0 || pos >= max_len || (count && s >= count[b])) continue;       // (whole quads: a quad is one block of one row)
    const u32x4 v = *reinterpret_cast<const u32x4*>(qkv + row * ld + (long)(H + hh) * DH + c * 8);
    const unsigned sc = mx_scale_code<false>(mx_quad_max(mx_amax8(v)));
    const bool is_v = hh >= Hkv;
    const long slot = ((long)b * Hkv + (is_v ? hh - Hkv : hh)) * max_len + pos;
    *reinterpret_cast<unsigned*>((is_v ? vc : kc) + slot * (DH / 2) + c * 4) = mx_quant8<false>(v, sc);
    if ((c & 3) == 0) (is_v ? vs : ks)[slot * (DH / 32) + (c >> 2)] = (unsigned char)sc;
  }
}

// ---- attention ----------------------------------------------------------------------------------------------------------------------
struct Kv4Args {
  const bf16_t* q;
  const unsigned char *kc, *ks, *vc, *vs;
  const int32_t* lens;
  bf16_t* out;
  float* ws;
  long ldq, ldo, max_len;
  int H, Hkv, G, splits;
  float scale_log2;                       // softmax scale * log2(e)
};

__device__ __forceinline__ float quarter_max(float v) {                       // over the four lanes that share a head column
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float quarter_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

__device__ __forceinline__ float kv4_other_half(float v) {                    // of the lane eight columns away
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, true));     // row_ror:8
}

typedef __attribute__((address_space(3))) void* lds_ptr_t;
constexpr int KV4_RING = 4;                // tiles in a wave's LDS ring

// vmcnt(V), and lgkmcnt(0): the wave's reads of LDS are back too, so a slot that they read may be filled again
template <int V>
__device__ __forceinline__ void kv4_wait() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((V & 15) | ((V >> 4) << 14) | 0x070);
  asm volatile("" ::: "memory");
}

// (a __device__ template under plain __global__ wrappers, as in gemm_pp.hip)
template <int DH, int WAVES>
__device__ __forceinline__ void attn_decode_kv4_body(const Kv4Args& p) {
  constexpr int KD = DH / 4;              // dims of a key per lane: KD / 2 bytes
  constexpr int VD = DH / 16;             // dims of a value row per lane: VD / 2 bytes
  constexpr int CB = DH / 2, SB = DH / 32;
  constexpr int TB = KV4_TILE * CB, ND = TB / 1024, LOADS = 2 * ND + 2;       // bytes of a tile's K, its DMA instructions, those of a tile
  constexpr int SLOT = 2 * TB + 512;                                          // K, V, a dword of scales per row of K, of V (each twice as long)
  extern __shared__ __attribute__((aligned(16))) float sm[];                  // the rings; afterwards [waves][G][DH] rows, [waves][G] max, [waves][G] sum
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), l = t & 63, r16 = l & 15, g = l >> 4;
  const int bh = blockIdx.x / p.splits, split = blockIdx.x - bh * p.splits;
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const long len = min((long)max(p.lens[b], 0), p.max_len);
  // keys of this split: a whole number of rounds of the workgroup
  const long round = WAVES * KV4_TILE;
  const long per = ((len + p.splits - 1) / p.splits + round - 1) / round * round;
  const long k0 = min(per * split, len), k1 = min(k0 + per, len);
  const long base = (long)bh * p.max_len;
  const unsigned char *kc = p.kc + base * CB, *vc = p.vc + base * CB, *ks = p.ks + base * SB, *vs = p.vs + base * SB;

  bf16x8 qf[KD / 8];
  f32x4 o[VD];
#pragma unroll
  for (int j = 0; j < VD; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float mx = -INFINITY, sum = 0.f;
  const bool second = p.G <= 8 && r16 >= 8;                                    // a column of the second terms

  char* const ring = reinterpret_cast<char*>(sm) + w * (KV4_RING * SLOT);
  const int krow = 4 * (r16 & 3) + (r16 >> 2);
  const long first = k0 + w * KV4_TILE;
  const int tiles = first < k1 ? (int)((k1 - first + round - 1) / round) : 0;
  // LDS image of K at dh = 128: 16-byte chunks at c ^ (key >> 2 & 3): the keys 4 apart of a fragment read fall into different banks.  The
  // descriptors of a tile end with the last key of the split: what lies behind it is not touched and comes as zeros (at scale 2^-127).
  unsigned off_k[ND], off_v[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    constexpr int LPR = CB / 16;                                               // lanes of a row
    const int key = (64 / LPR) * i + l / LPR, c = l % LPR;
    off_k[i] = key * CB + (LPR == 4 ? c ^ ((key >> 2) & 3) : c) * 16;
    off_v[i] = key * CB + c * 16;
  }
  auto rsrc = [](const unsigned char* at, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(at), 0, (unsigned)bytes, 0x00020000);
  };
  auto fetch = [&](int n, int slot) {
    const long kt = first + (long)n * round;
    const int left = (int)min(k1 - kt, (long)KV4_TILE);
    char* d = ring + slot * SLOT;
    const __amdgpu_buffer_rsrc_t rk = rsrc(kc + kt * CB, left * CB), rv = rsrc(vc + kt * CB, left * CB);
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_ptr_t)(d + i * 1024), 16, off_k[i], 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_ptr_t)(d + TB + i * 1024), 16, off_v[i], 0, 0, 0);
    }
    const __amdgpu_buffer_rsrc_t rks = rsrc(ks + kt * SB, left * SB), rvs = rsrc(vs + kt * SB, left * SB);
    if constexpr (SB == 4) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rks, (lds_ptr_t)(d + 2 * TB), 4, (unsigned)l * 4u, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rvs, (lds_ptr_t)(d + 2 * TB + 256), 4, (unsigned)l * 4u, 0, 0, 0);
    } else {                                                                   // (two bytes a row: a dword all the same, zero-extended)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rks, (lds_ptr_t)(d + 2 * TB), 2, (unsigned)l * 2u, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rvs, (lds_ptr_t)(d + 2 * TB + 256), 2, (unsigned)l * 2u, 0, 0, 0);
    }
  };
  auto compute = [&](int n, int slot) {
    const long kt = first + (long)n * round;
    const int left = (int)min(k1 - kt, (long)KV4_TILE);                        // valid keys of this tile
    const char* d = ring + slot * SLOT;
    // scores: lane holds keys 16 u + 4 i + g of head r16
    float s[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key = 16 * u + krow;
      unsigned kq[KD / 8];
      if constexpr (KD == 32) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(d + key * CB + (g ^ ((key >> 2) & 3)) * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) kq[j] = x[j];
      } else {
        const u32x2 x = *reinterpret_cast<const u32x2*>(d + key * CB + g * 8);
        kq[0] = x[0]; kq[1] = x[1];
      }
      const float ksc = mx_scale((unsigned char)d[2 * TB + key * 4 + g * KD / 32]);
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KD / 8; ++j) a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_bf16x8(kq[j], ksc), qf[j], a, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * u + i] = 16 * u + 4 * i + g < left ? a[i] * p.scale_log2 : -INFINITY;
    }
    float tm = s[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) tm = fmaxf(tm, s[e]);
    const float nm = fmaxf(mx, quarter_max(tm));
    const float off = nm == -INFINITY ? 0.f : nm;                              // nothing but -inf so far: every p is 0
    const float fac = __builtin_amdgcn_exp2f(mx - off);
    mx = nm;
    float pr[8], ps = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) { pr[e] = __builtin_amdgcn_exp2f(s[e] - off); ps += pr[e]; }
    sum = sum * fac + ps;                                                      // (this lane's quarter of the keys; joined at the end)
    u32x4 pw, rest;                                                            // two probabilities a dword; p less its rounding
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned h = pack_bf2(pr[2 * i], pr[2 * i + 1]);
      rest[i] = pack_bf2(pr[2 * i] - bf_lo(h), pr[2 * i + 1] - bf_hi(h));
      pw[i] = second ? rest[i] : h;
    }
    const bf16x8 pf = __builtin_bit_cast(bf16x8, pw);
#pragma unroll
    for (int j = 0; j < VD; ++j) o[j] *= fac;
    // values: dims r16 * VD + j of the keys of quarter g (a key past the end: p = 0 against zeros)
    unsigned vp[VD / 2][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int key = 16 * (e >> 2) + 4 * (e & 3) + g;
      const float vsc = mx_scale((unsigned char)d[2 * TB + 256 + key * 4 + r16 * VD / 32]);
      unsigned vq;
      if constexpr (VD == 8) vq = *reinterpret_cast<const unsigned*>(d + TB + key * CB + r16 * 4);
      else vq = *reinterpret_cast<const unsigned short*>(d + TB + key * CB + r16 * 2);
      vp[0][e] = mx_pair_bf16<0>(vq, vsc);
      vp[1][e] = mx_pair_bf16<1>(vq, vsc);
      if constexpr (VD == 8) { vp[2][e] = mx_pair_bf16<2>(vq, vsc); vp[3][e] = mx_pair_bf16<3>(vq, vsc); }
    }
#pragma unroll
    for (int j = 0; j < VD; ++j) {
      u32x4 f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = __builtin_amdgcn_perm(vp[j >> 1][2 * e + 1], vp[j >> 1][2 * e], (j & 1) ? 0x07060302u : 0x05040100u);
      o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, f), pf, o[j], 0, 0, 0);
      if (p.G > 8) o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, f), __builtin_bit_cast(bf16x8, rest), o[j], 0, 0, 0);
    }
  };
#pragma unroll
  for (int n = 0; n < KV4_RING - 1; ++n)
    if (n < tiles) fetch(n, n);
  {
    const int head = min(p.G > 8 ? r16 : r16 & 7, p.G - 1);                    // of this column (those past G repeat the last head)
    const bf16_t* qp = p.q + (long)b * p.ldq + (long)(hk * p.G + head) * DH + g * KD;
#pragma unroll
    for (int j = 0; j < KD / 8; ++j) qf[j] = *reinterpret_cast<const bf16x8*>(qp + j * 8);
  }
  kv4_wait<0>();                                                               // (the query, too: a load still out at the loop's entry is waited for in every round)
  for (int n0 = 0; n0 < tiles; n0 += KV4_RING) {
#pragma unroll
    for (int u = 0; u < KV4_RING; ++u) {
      const int n = n0 + u;
      if (n >= tiles) break;
      // tile n has landed when no more than the tiles behind it are out
      const int behind = min(tiles - 1 - n, KV4_RING - 2);
      if (behind == 2) kv4_wait<2 * LOADS>(); else if (behind == 1) kv4_wait<LOADS>(); else kv4_wait<0>();
      if (n + KV4_RING - 1 < tiles) fetch(n + KV4_RING - 1, (u + KV4_RING - 1) % KV4_RING);     // (tile n - 1's slot, whose reads the wait has seen back)
      compute(n, u);
    }
  }
  sum = quarter_sum(sum);
  __syncthreads();                                                             // the rings become the rows to merge

  if (p.G <= 8) {
#pragma unroll
    for (int j = 0; j < VD; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] += kv4_other_half(o[j][i]);
  }
  // merge: lane holds dims (4 g + i) VD + j of head r16
  float* sm_m = sm + WAVES * p.G * DH;
  float* sm_l = sm_m + WAVES * p.G;
  if (r16 < p.G) {
    float* row = sm + (w * p.G + r16) * DH + 4 * g * VD;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < VD; ++j) row[i * VD + j] = o[j][i];
    if (g == 0) { sm_m[w * p.G + r16] = mx; sm_l[w * p.G + r16] = sum; }
  }
  __syncthreads();
  for (int i = t; i < p.G * DH; i += WAVES * 64) {
    const int h = i / DH, d = i - h * DH;
    float m = sm_m[h];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) m = fmaxf(m, sm_m[v * p.G + h]);
    const float off = m == -INFINITY ? 0.f : m;
    float acc = 0.f, den = 0.f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) {
      const float f = __builtin_amdgcn_exp2f(sm_m[v * p.G + h] - off);
      acc += f * sm[(v * p.G + h) * DH + d];
      den += f * sm_l[v * p.G + h];
    }
    const long head = (long)b * p.H + hk * p.G + h;
    if (p.splits == 1) {
      p.out[(long)b * p.ldo + (hk * p.G + h) * DH + d] = f2bf(len == 0 ? 0.f : acc / den);     // (keys whose scores are all -inf: 0 / 0, as the definition has it)
    } else {
      float* rec = p.ws + (head * p.splits + split) * (DH + 2);
      rec[d] = acc;
      if (d == 0) { rec[DH] = m; rec[DH + 1] = den; }
    }
  }
}

__global__ __launch_bounds__(KV4_WAVES * 64, 2) void attn_decode_kv4_128_kernel(Kv4Args p) { attn_decode_kv4_body<128, KV4_WAVES>(p); }
__global__ __launch_bounds__(KV4_WAVES * 64, 2) void attn_decode_kv4_64_kernel(Kv4Args p) { attn_decode_kv4_body<64, KV4_WAVES>(p); }
__global__ __launch_bounds__(KV4_WIDE * 64, 2) void attn_decode_kv4_128_wide_kernel(Kv4Args p) { attn_decode_kv4_body<128, KV4_WIDE>(p); }
__global__ __launch_bounds__(KV4_WIDE * 64, 2) void attn_decode_kv4_64_wide_kernel(Kv4Args p) { attn_decode_kv4_body<64, KV4_WIDE>(p); }

// Joins the splits of one head: KV4_JOIN groups of DH threads take every KV4_JOIN-th split, all of a group's loads at once up to eight, and merge
// in LDS, in order.
constexpr int KV4_JOIN = 4;
template <int DH>
__global__ __launch_bounds__(KV4_JOIN * DH) void kv4_combine_kernel(const float* __restrict__ ws, const int32_t* __restrict__ lens, bf16_t* __restrict__ out, long ldo,
                                                                   int H, int splits) {
  __shared__ float sa[KV4_JOIN][DH], sm[KV4_JOIN], sl[KV4_JOIN];
  const long head = blockIdx.x;
  const float* rec = ws + head * splits * (DH + 2);
  const int d = threadIdx.x % DH, grp = threadIdx.x / DH;
  float m = -INFINITY, acc = 0.f, den = 0.f;
  for (int s0 = grp; s0 < splits; s0 += 8 * KV4_JOIN) {
    float ms[8], ls[8], as[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float* r = rec + (long)min(s0 + KV4_JOIN * i, splits - 1) * (DH + 2);
      ms[i] = r[DH];
      ls[i] = r[DH + 1];
      as[i] = r[d];
    }
    float nm = m;
#pragma unroll
    for (int i = 0; i < 8; ++i) if (s0 + KV4_JOIN * i < splits) nm = fmaxf(nm, ms[i]);
    const float off = nm == -INFINITY ? 0.f : nm, fac = __builtin_amdgcn_exp2f(m - off);
    acc *= fac;
    den *= fac;
    m = nm;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (s0 + KV4_JOIN * i >= splits) break;
      const float f = __builtin_amdgcn_exp2f(ms[i] - off);
      acc += f * as[i];
      den += f * ls[i];
    }
  }
  sa[grp][d] = acc;
  if (d == 0) { sm[grp] = m; sl[grp] = den; }
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int i = 1; i < KV4_JOIN; ++i) m = fmaxf(m, sm[i]);
  const float off = m == -INFINITY ? 0.f : m;
  acc = den = 0.f;
#pragma unroll
  for (int i = 0; i < KV4_JOIN; ++i) {
    const float f = __builtin_amdgcn_exp2f(sm[i] - off);
    acc += f * sa[i][d];
    den += f * sl[i];
  }
  const long b = head / H;
  out[b * ldo + (head % H) * DH + d] = f2bf(lens[b] <= 0 ? 0.f : acc / den);
}

// Splits of the key axis, waves of a workgroup, by the number of (sample, KV head) pairs and the length of the cache.  Two workgroups fit a CU.
//   Up to 256 pairs, short caches: a workgroup of eight waves reads all of a head's keys and nothing is joined.  Longer ones: one round of splits (512
//   workgroups), joined by a second kernel; where samples may differ by many thousands of keys two rounds, so that the short ones make room.
//   Beyond 256 pairs: no split, but for long caches, whose last round would be long.
// Measured (us, in a graph; all keys used, dh = 128): 32 pairs x 256 keys one kernel 5.5, two 7.2; x 512 7.0 / 7.5; x 967 9.6 / 8.2: from about 600 keys on the
// second launch costs a graph less than it gains, but a call that is issued by itself some 3 us of the host.  x 8192 8, 16, 32 splits 17.0, 16.9, 20.0;
// 128 pairs x 2048 one kernel 16.9, two 16.2, x 4096 28.0 / 22.8; 64 pairs x 32768 8, 16 splits 68.7, 74.3, and 42.5, 42.6 with lengths spread from 1000 to
// 32768; 520 pairs x 967 1, 2 splits 26.3, 27.8, x 4096 82.8, 74.9; 1024 pairs x 1131 38.5, 47.1.
struct Kv4Plan {
  int waves, splits;
};
Kv4Plan kv4_plan(int B, int Hkv, long max_len) {
  const long pairs = (long)B * Hkv, rounds = (max_len + KV4_WAVES * KV4_TILE - 1) / (KV4_WAVES * KV4_TILE);
  if (pairs > 256) return {KV4_WAVES, max_len <= 2048 ? 1 : (int)((1024 + pairs - 1) / pairs)};
  if (max_len <= (pairs > 51 ? 20 * pairs : 1024)) return {KV4_WIDE, 1};
  const long s = (B == 1 || max_len <= 8192 ? 512 : 1024) / pairs;
  return {KV4_WAVES, (int)(s > rounds ? rounds : s > 256 ? 256 : s)};
}

}  // namespace
}  // namespace hvlm

using namespace hvlm;

static int kv4_check(const char* what, const void* kc, const void* ks, const void* vc, const void* vs, int B, long max_len, int H, int Hkv, int dh) {
  HVLM_REQUIRE(kc && ks && vc && vs, "%s: null pointer", what);
  HVLM_REQUIRE(B > 0 && max_len > 0 && H > 0 && Hkv > 0, "%s: B=%d, max_len=%ld, H=%d, Hkv=%d must be positive", what, B, max_len, H, Hkv);
  HVLM_REQUIRE(dh == 64 || dh == 128, "%s: head dimension %d (64 or 128)", what, dh);
  HVLM_REQUIRE(max_len < (1L << 31) && (long)B * Hkv < (1L << 22), "%s: cache too large", what);
  HVLM_REQUIRE((((uintptr_t)kc | (uintptr_t)vc) & 15) == 0, "%s: codes must be 16-byte aligned", what);
  HVLM_REQUIRE((((uintptr_t)ks | (uintptr_t)vs) & (dh / 32 - 1)) == 0, "%s: scales must be aligned to a row's %d bytes", what, dh / 32);
  return HVLM_OK;
}

extern "C" int hvlm_kv4_append(const void* qkv, long ld, void* k_codes, void* k_scales, void* v_codes, void* v_scales, const int32_t* start,
                               const int32_t* count, int B, int S, long max_len, int H, int Hkv, int dh, void* stream) {
  const int rc = kv4_check("kv4_append", k_codes, k_scales, v_codes, v_scales, B, max_len, H, Hkv, dh);
  if (rc) return rc;
  HVLM_REQUIRE(qkv && S > 0, "kv4_append: null rows or S=%d", S);
  HVLM_REQUIRE(ld >= (long)(H + 2 * Hkv) * dh && ld % 8 == 0 && ((uintptr_t)qkv & 15) == 0, "kv4_append: rows must be 16-byte aligned");
  const long total = (long)B * S * 2 * Hkv * (dh / 8), g = (total + 255) / 256;
  const auto k = dh == 128 ? kv4_append_kernel<128> : kv4_append_kernel<64>;
  hipLaunchKernelGGL(k, dim3((unsigned)(g < 8192 ? g : 8192)), dim3(256), 0, as_stream(stream), (const bf16_t*)qkv, ld, (unsigned char*)k_codes,
                     (unsigned char*)k_scales, (unsigned char*)v_codes, (unsigned char*)v_scales, start, count, B, S, max_len, H, Hkv);
  return check_launch("kv4_append");
}

extern "C" size_t hvlm_attn_decode_kv4_ws_bytes(int B, int H, int Hkv, int dh, long max_len) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || dh <= 0 || max_len <= 0) return 0;
  const int s = kv4_plan(B, Hkv, max_len).splits;
  return s == 1 ? 0 : (size_t)B * H * s * (dh + 2) * 4;
}

extern "C" int hvlm_attn_decode_kv4(const void* q, long ldq, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                                    const int32_t* lens, void* out, long ldo, int B, long max_len, int H, int Hkv, int dh, float scale, void* ws,
                                    void* stream) {
  const int rc = kv4_check("attn_decode_kv4", k_codes, k_scales, v_codes, v_scales, B, max_len, H, Hkv, dh);
  if (rc) return rc;
  HVLM_REQUIRE(q && lens && out, "attn_decode_kv4: null pointer");
  HVLM_REQUIRE(H % Hkv == 0 && H / Hkv <= 16, "attn_decode_kv4: H=%d must be 1 to 16 times Hkv=%d", H, Hkv);
  HVLM_REQUIRE(ldq >= (long)H * dh && ldq % 8 == 0 && ((uintptr_t)q & 15) == 0, "attn_decode_kv4: rows of q must be 16-byte aligned");
  HVLM_REQUIRE(ldo >= (long)H * dh, "attn_decode_kv4: leading dimension of out");
  const Kv4Plan plan = kv4_plan(B, Hkv, max_len);
  const int splits = plan.splits, waves = plan.waves, G = H / Hkv;
  HVLM_REQUIRE(splits == 1 || (ws && ((uintptr_t)ws & 15) == 0), "attn_decode_kv4: a 16-byte aligned workspace of hvlm_attn_decode_kv4_ws_bytes() is needed");
  Kv4Args p{};
  p.q = (const bf16_t*)q; p.kc = (const unsigned char*)k_codes; p.ks = (const unsigned char*)k_scales; p.vc = (const unsigned char*)v_codes;
  p.vs = (const unsigned char*)v_scales; p.lens = lens; p.out = (bf16_t*)out; p.ws = (float*)ws; p.ldq = ldq; p.ldo = ldo; p.max_len = max_len;
  p.H = H; p.Hkv = Hkv; p.G = G; p.splits = splits; p.scale_log2 = scale * 1.4426950408889634f;
  const size_t merge = (size_t)waves * G * (dh + 2) * 4, rings = (size_t)waves * KV4_RING * (KV4_TILE * dh + 512);
  const size_t lds = merge > rings ? merge : rings;                           // a wave's ring is 18 KB at dh = 128, 10 KB at dh = 64
  const auto k = dh == 128 ? (waves == KV4_WIDE ? attn_decode_kv4_128_wide_kernel : attn_decode_kv4_128_kernel)
                           : (waves == KV4_WIDE ? attn_decode_kv4_64_wide_kernel : attn_decode_kv4_64_kernel);
  const auto set = [](void (*f)(Kv4Args), int bytes) { return hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, bytes); };
  static const hipError_t a1 = set(attn_decode_kv4_128_kernel, 73728), a2 = set(attn_decode_kv4_128_wide_kernel, 147456), a3 = set(attn_decode_kv4_64_wide_kernel, 81920);
  if (a1 != hipSuccess || a2 != hipSuccess || a3 != hipSuccess) {
    set_error("attn_decode_kv4: hipFuncSetAttribute: %s", hipGetErrorString(a1 != hipSuccess ? a1 : a2 != hipSuccess ? a2 : a3));
    return HVLM_ERR_LAUNCH;
  }
  hipLaunchKernelGGL(k, dim3((unsigned)(B * Hkv * splits)), dim3((unsigned)waves * 64), lds, as_stream(stream), p);
  const int rc2 = check_launch("attn_decode_kv4");
  if (rc2 || splits == 1) return rc2;
  const auto c = dh == 128 ? kv4_combine_kernel<128> : kv4_combine_kernel<64>;
  hipLaunchKernelGGL(c, dim3((unsigned)(B * H)), dim3(KV4_JOIN * dh), 0, as_stream(stream), (const float*)ws, lens, (bf16_t*)out, ldo, H, splits);
  return check_launch("attn_decode_kv4");
}
