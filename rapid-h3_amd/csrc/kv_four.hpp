// The 4-bit format of the paged cache (RH3_KV_FP4): what its kernels share.
//
// A row of a head is groups of 32 channels: codes e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign bit), two to a byte, the lower
// channel in the low half; a group has one power of two 2^(byte - 127), the least that brings its largest magnitude to 7 or under:
// what lies over 5 rounds to 6, off by 1 at most, as what lies between 4 and 6 is. 4.25 bits a value. The bytes that writing
// leaves are 2 to 252 (no value underflows or overflows fp32); 255 in a key's bytes marks a position whose key or value holds an
// infinity or a NaN.
// A code times its power of two is exact in bf16 (2 significant bits, fp32's exponents), so attention takes keys and values to the
// bf16 MFMA as they are, scale included, two to an instruction. (The MFMA that reads e2m1 codes and their scale bytes itself keeps
// its sums to 2^-13 of their terms' magnitudes, measured on random operands; the bf16 one to fp32's rounding.)
#pragma once

#include <type_traits>

#include "kv_attn.hpp"

namespace rh3 {
namespace kv {

typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));

constexpr int GROUP4 = 32;                              // channels to a scale

// the scale byte of a group by the bits of its largest magnitude (finite): e with amax <= 7 * 2^e, within +-125
__device__ __forceinline__ uint32_t scale4(uint32_t amax) {
  const int e = static_cast<int>(amax >> 23) - 2 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(min(max(e, 2), 252));
}
// 8 values to codes; the conversion takes the scale's exponent, rounds to the nearest code, ties to the even one, and saturates
__device__ __forceinline__ uint32_t codes4(const float* x, uint32_t byte) {
  const float s = __uint_as_float(byte << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  return w;
}
// two values of byte I of a word; of the scale only the exponent's bits count (its sign and mantissa may be anything)
template <int I>
__device__ __forceinline__ uint32_t pair4(uint32_t w, float s) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, I));
}
__device__ __forceinline__ uint4 words4(uint32_t w, float s) {
  return make_uint4(pair4<0>(w, s), pair4<1>(w, s), pair4<2>(w, s), pair4<3>(w, s));
}
__device__ __forceinline__ b8_t bf16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __builtin_bit_cast(b8_t, make_uint4(a, b, c, d)); }
__device__ __forceinline__ b8_t values4(uint32_t w, float s) { return __builtin_bit_cast(b8_t, words4(w, s)); }

// A query row's 8 values in bf16: as they are, or, of fp16 (11 significant bits), in two terms, which hold them exactly
template <bool FINE>
__device__ __forceinline__ void query8(const uint4 raw, b8_t& hi, b8_t& lo) {
  if constexpr (!FINE) {
    hi = __builtin_bit_cast(b8_t, raw);
  } else {
    float x[8];
    row8<RH3_DTYPE_F16>(raw, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi[e] = static_cast<__bf16>(x[e]);
      lo[e] = static_cast<__bf16>(x[e] - static_cast<float>(hi[e]));
    }
  }
}

// Probabilities are 2^(score - reference), base 2, with the reference OVER over the row's running maximum, moved where a score comes
// to less than -STALE under it: with bf16's exponents their size costs nothing. Of equal scores 2^16 make a lane's sum, of scores that
// rose just so far that the reference stayed 2^4; at SUM_MOST it moves up by LATER. So a row's sum over the 16 lanes that share it in
// a workgroup is under 0.1, its values' sum, not yet divided, under 0.1 of the largest of them, and fp32 holds both, and the join of all
// workgroups' times PART, up to the largest value there is (1.5 * 2^127) for any number of keys. Values down to 2^-94 keep their bits
// (2^-82 after one LATER: 2^17 equal scores and more). (From 2^28 on, a score's last place is more than OVER: the reference is then
// the maximum itself, or the next number, and does not move for a sum's sake.)
constexpr float OVER = 24.0f;
constexpr float STALE = -12.0f;
constexpr float SUM_MOST = 0x1p-8f;
constexpr float LATER = 12.0f;
constexpr float NO_REF = -0x1.fffffep127f;   // reference of a row that has seen no key: any score moves it
__device__ __forceinline__ float reference_over(float top) { return top + OVER; }
// a row's reference for keys whose largest score is `top`; sum: of its probabilities so far, over all lanes
__device__ __forceinline__ float next_reference(float ref, float top, float sum, float stale = STALE) {
  return top - ref > stale ? reference_over(top) : sum > SUM_MOST ? ref + LATER : ref;
}
// parts are kept against a reference 2^24 lower (their sums times PART, as the join takes them)
constexpr float PART_UP = 0x1p24f;

// host: launches of the two kernels for their checked arguments
void launch_token4(const AttnArgs& a, int dim, int rows, hipStream_t st);
void launch_chunk4(const AttnArgs& a, int dim, int rows, hipStream_t st);

}  // namespace kv
}  // namespace rh3
