// Attention over the paged cache: what its kernels share. kv_token.hip runs few query rows to a K/V head (bound by the cache's
// bytes), kv_chunk.hip many (bound by the matrix units), kv_attn.hip joins the parts that either leaves and holds the entry points.
//
// For a query row i of a sequence of n rows and `len` cached positions: o_i = sum_j p_ij v_j / sum_j p_ij with
// p_ij = exp(scale q_i.k_j) over j < len, and j <= len - n + i if causal. A K/V head's query rows are its group's heads of every
// token of the sequence, numbered token * group + head in the group, so that the group shares each key and value that is read.
//
// Arithmetic. Codes are small integers (int8) or 4-bit significands (e4m3): exact in f16. A query row is scaled by the power of
// two that brings its largest magnitude to [2^7, 2^8): bf16 and fp16 values are exact in f16 after it (those 2^21 below the row's
// largest lose low bits, 2^-33 of it at most). So q.k is a sum of exact products in fp32 on the f16 MFMA, times the key's scale,
// in fp32. Probabilities are taken against a reference 10 to 15 under the row's running maximum (base 2), so that in f16 they use
// its range from 2^15 down, rounded to nearest (2^-11 relative at most); products of probability and value scale keep that
// precision down to 2^-24 of the largest. Their sum is fp32.
#pragma once

#include "kv_common.hpp"

namespace rh3 {
namespace kv {

// A part: the unnormalised sum of a query row over some of its keys, with the fp32 sum of its probabilities and their reference
// (base 2). Slots of parts hold R rows each: part_o [slot][R][dim], part_ml [slot][R][2] (reference, sum).
struct AttnArgs {
  Cache c;
  Seqs s;
  const void* q;
  int64_t q_st, q_sh;
  int fp16, group, causal;
  float scale_log2;          // softmax scale * log2(e)
  void* out;
  int64_t o_st, o_sh;
  float* lse;                // [rows][q heads] or null
  float* part_o;
  float* part_ml;
  int64_t items;             // slots of completed items
  int wgs;                   // token kernel: workgroups
  int keep;                  // token kernel: leave a part for every item, also for those that one workgroup completes
  int splits, tiles;         // chunk kernel: key ranges of an item, row tiles in the grid
};

// ---------------------------------------------------------------- the token kernel's work, the same on every wave that asks
// Items: (sequence, K/V head, R query rows of it). Units: 32 keys of an item. The units of all items in order (sequences, then
// K/V heads, then row tiles) are dealt to the workgroups in equal contiguous ranges, so that uneven histories, which only the
// device knows, load the workgroups evenly. UNIT_MIN units at least make a workgroup worth starting: one for each of its waves.
constexpr int UNIT_KEYS = 32;
constexpr int UNIT_MIN = 4;

struct Work {
  int64_t units;             // of all sequences
  int wgs;                   // workgroups that have a share
};
RH3_HD int64_t share_begin(const Work& w, int wg) { return w.units * wg / w.wgs; }
// the workgroup whose share holds unit u
RH3_HD int share_of(const Work& w, int64_t u) { return static_cast<int>(((u + 1) * w.wgs - 1) / w.units); }

struct SeqWork {
  int row_tiles, key_tiles;
  int64_t units;
};
RH3_HD SeqWork work_of(const AttnArgs& a, const Seq& q, int R) {
  SeqWork w;
  w.row_tiles = static_cast<int>((static_cast<int64_t>(q.n) * a.group + R - 1) / R);
  const int kt = (q.len + UNIT_KEYS - 1) / UNIT_KEYS;
  w.key_tiles = kt < 1 ? 1 : kt;
  // no memory holds 2^36 units (2^41 keys); offsets in cu that fall can count rows many times, and must not overflow the sums
  const int64_t u = static_cast<int64_t>(a.c.heads) * w.row_tiles;
  w.units = u < (int64_t{1} << 36) / w.key_tiles ? u * w.key_tiles : int64_t{1} << 36;
  return w;
}
__device__ __forceinline__ int64_t wave_scan(int64_t v) {   // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t t = __shfl_up(v, d);
    if (lane >= d) v += t;
  }
  return v;
}
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  return (static_cast<int64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32))) << 32) |
         static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v)));
}

// units of all sequences; and, for the sequence b >= 0, those of the sequences before it and their items
__device__ __forceinline__ Work all_work(const AttnArgs& a, int R, int b, int64_t& before, int64_t& items_before) {
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  before = items_before = 0;
  for (int at = 0; at < a.s.batch; at += 64) {
    int64_t u = 0, it = 0;
    if (at + lane < a.s.batch) {
      const SeqWork w = work_of(a, seq_at(a.s, at + lane), R);
      u = w.units;
      it = static_cast<int64_t>(a.c.heads) * w.row_tiles;
    }
    const bool pre = at + lane < b;
    int64_t ub = pre ? u : 0, ib = pre ? it : 0;
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      u += __shfl_xor(u, d);
      if (b > at) {
        ub += __shfl_xor(ub, d);
        ib += __shfl_xor(ib, d);
      }
    }
    total += u;
    before += ub;
    items_before += ib;
  }
  Work w;
  w.units = uniform64(total);
  before = uniform64(before);
  items_before = uniform64(items_before);
  const int64_t most = (w.units + UNIT_MIN - 1) / UNIT_MIN;
  w.wgs = static_cast<int>(most < a.wgs ? (most > 0 ? most : 1) : a.wgs);
  return w;
}

// the sequence that holds unit u, the units and items before it
struct UnitAt {
  int b;
  int64_t before, items_before;
};
__device__ __forceinline__ UnitAt seq_of_unit(const AttnArgs& a, int R, int64_t u) {
  const int lane = threadIdx.x & 63;
  int64_t base = 0, ibase = 0;
  for (int at = 0; at < a.s.batch; at += 64) {
    int64_t n = 0, it = 0;
    if (at + lane < a.s.batch) {
      const SeqWork w = work_of(a, seq_at(a.s, at + lane), R);
      n = w.units;
      it = static_cast<int64_t>(a.c.heads) * w.row_tiles;
    }
    const int64_t s = wave_scan(n), si = wave_scan(it);
    const unsigned long long m = __builtin_amdgcn_ballot_w64(base + s > u);
    if (m) {
      const int l = __builtin_ctzll(m);
      UnitAt r;
      r.b = __builtin_amdgcn_readfirstlane(at + l);
      r.before = uniform64(base + __shfl(s - n, l));
      r.items_before = uniform64(ibase + __shfl(si - it, l));
      return r;
    }
    base += __shfl(s, 63);
    ibase += __shfl(si, 63);
  }
  return UnitAt{-1, 0, 0};
}

// ---------------------------------------------------------------- query rows
// 8 values of a query row at offset `at` as floats
__device__ __forceinline__ void load_q8(const AttnArgs& a, int64_t at, float* v) {
  if (a.fp16) load_row8<RH3_DTYPE_F16>(a.q, at, v);
  else load_row8<RH3_DTYPE_BF16>(a.q, at, v);
}
// the exponent that brings a magnitude to [2^7, 2^8) (zero, infinite or NaN: none)
__device__ __forceinline__ int q_exponent(float amax) {
  const int e = static_cast<int>(__float_as_uint(amax) >> 23) & 255;
  return e == 0 || e == 255 ? 0 : 134 - e;
}
__device__ __forceinline__ h8_t q_f16(const float* v, int e) {
  h8_t r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = static_cast<_Float16>(__builtin_amdgcn_ldexpf(v[i], e));
  return r;
}
// max and sum over lanes l, l ^ 32 and (QUAD) l ^ 16
template <bool QUAD>
__device__ __forceinline__ float across_max(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  v = fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
  if constexpr (QUAD) {
    r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
  }
  return v;
}
template <bool QUAD>
__device__ __forceinline__ float across_sum(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  v = __int_as_float(r[0]) + __int_as_float(r[1]);
  if constexpr (QUAD) {
    r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = __int_as_float(r[0]) + __int_as_float(r[1]);
  }
  return v;
}

// ---------------------------------------------------------------- the softmax reference and the values' scale
constexpr float REF_UNDER = 10.0f;   // a new reference lies this far under the maximum: probabilities up to 2^10
constexpr float REF_STALE = 15.0f;   // a score this far over the reference moves it: probabilities up to 2^15

// the power of two over a scale (the largest finite one for an infinity; NaN never gets here)
__device__ __forceinline__ float pow2_over(float v) {
  const uint32_t e = (__float_as_uint(v) >> 23) & 255u;
  return __uint_as_float(min(e + 1u, 253u) << 23);
}

__device__ __forceinline__ uint32_t pack_out(const AttnArgs& a, float x, float y) { return a.fp16 ? pack_h2(x, y) : pack_bf2(x, y); }

// host: launches of the two kernels for their checked arguments
void launch_token(const AttnArgs& a, int fmt, int dim, int rows, hipStream_t st);
void launch_chunk(const AttnArgs& a, int fmt, int dim, int rows, int64_t grid, hipStream_t st);

}  // namespace kv
}  // namespace rh3
