// OCP Microscaling FP4 (MXFP4) on gfx950: blocks of 32 consecutive elements share one power-of-two scale (E8M0 byte s, value
// 2^(s - 127), 255 = NaN), elements are E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two per byte, the even element in the low
// nibble.  A block is quantised with s - 127 = floor(log2 max|x|) - 2 (6 = 1.5 * 2^2 is the largest element: values between 6 and 8 of a
// block saturate, as the format's specification has it) and round-to-nearest-even; a block with an infinity or a NaN becomes NaN.
// v_cvt_scalef32_pk_* does the scaling and the rounding of a pair in one instruction; it agrees with the definition for every finite
// bf16 / fp16 value at every scale code, and for every code back to bf16 / fp16 / fp32, subnormal results included (4 and 6 at scale code 253, 2 and
// more at 254 are past the range of bf16 and fp32 and become infinities; no quantised block has a scale code above 252).
#pragma once
#include "common.h"

namespace hvlm {

constexpr int MX_BLOCK = 32;

// E8M0 byte -> the fp32 scale operand of v_cvt_scalef32_*: it reads the exponent field alone, 0 as 2^-127 and 255 as NaN
__device__ __forceinline__ float mx_scale(unsigned s) { return __uint_as_float(s << 23); }

// largest magnitude bits of a block (sign cleared: ordered like the magnitudes, infinities and NaNs on top) -> its E8M0 byte
template <bool F16>
__device__ __forceinline__ unsigned mx_scale_code(unsigned amax) {
  if constexpr (!F16) {
    const int e = (int)(amax >> 7);                  // biased exponent; a subnormal block (e = 0) is below 2^-126: clamped to 2^-127
    return e == 255 ? 255u : (unsigned)max(e - 2, 0);
  } else {
    const int e = (int)(amax >> 10);
    if (e == 31) return 255u;
    if (e) return (unsigned)(e - 15 - 2 + 127);
    return amax ? (unsigned)(31 - __builtin_clz(amax) - 24 - 2 + 127) : 0u;
  }
}

// max over the 8 magnitudes of a 16-byte chunk
__device__ __forceinline__ unsigned mx_amax8(u32x4 v) {
  unsigned r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r = max(r, max(v[i] & 0x7fffu, (v[i] >> 16) & 0x7fffu));
  return r;
}
// max over the four adjacent lanes that hold one block (every lane gets it)
__device__ __forceinline__ unsigned mx_quad_max(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));    // quad_perm [1,0,3,2]
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));  // quad_perm [2,3,0,1]
}
// eight 16-bit floats -> eight codes (one dword) at scale code s
template <bool F16>
__device__ __forceinline__ unsigned mx_quant8(u32x4 v, unsigned s) {
  const float sc = mx_scale(s);
  unsigned r = 0;
  if constexpr (F16) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, (unsigned)v[0]), sc, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, (unsigned)v[1]), sc, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, (unsigned)v[2]), sc, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, (unsigned)v[3]), sc, 3);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (unsigned)v[0]), sc, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (unsigned)v[1]), sc, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (unsigned)v[2]), sc, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (unsigned)v[3]), sc, 3);
  }
  return s == 255u ? 0u : r;                         // a NaN block holds zeros under its NaN scale
}
// byte I of a dword of codes -> a bf16 pair (exact but for overflow)
template <int I>
__device__ __forceinline__ unsigned mx_pair_bf16(unsigned codes, float sc) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, sc, I));
}
// eight codes -> eight bf16
__device__ __forceinline__ bf16x8 mx_bf16x8(unsigned codes, float sc) {
  const u32x4 r = {mx_pair_bf16<0>(codes, sc), mx_pair_bf16<1>(codes, sc), mx_pair_bf16<2>(codes, sc), mx_pair_bf16<3>(codes, sc)};
  return __builtin_bit_cast(bf16x8, r);
}

}  // namespace hvlm
