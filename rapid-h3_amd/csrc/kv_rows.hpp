// Rows of keys and values on their way into the paged cache: where a row of a call lies, and its codes and scales (kv_cache.hip,
// kv_rope.hip).
#pragma once

#include "kv_four.hpp"

namespace rh3 {
namespace kv {

constexpr int NT = 256;

// where a row of the call lies in the cache: offsets of its codes and scale without the head's part; false if it lies nowhere
// (no sequence has the row, its position is before the first or past the table, its page is absent). `mine`: a sequence has the row.
struct Place {
  int64_t code, scale;
  int64_t pos;      // of a row that is `mine`, wherever that is: a sequence's rows have their positions past the table's end too
  bool mine, there;
};
template <int FMT, int D>
__device__ __forceinline__ Place place_of(const Seqs& s, const Cache& c, int row) {
  Place p{0, 0, 0, false, false};
  Seq q;
  int64_t row0;
  const int b = seq_of_row<D / 8 == 16 ? 16 : 8>(s, min(row, s.rows - 1), q, row0);
  if (b < 0 || row >= s.rows) return p;
  p.mine = true;
  p.pos = row0 + row;
  if (p.pos < 0 || p.pos >= s.cap) return p;
  const int pos = static_cast<int>(p.pos), pg = page_of(s, c, b, pos);
  if (pg < 0) return p;
  const int off = pos & ((1 << c.log2page) - 1);
  p.code = pg * c.page_stride + off * (FMT == FP4 ? D / 2 : D);
  p.scale = pg * c.spage_stride + off * (FMT == FP4 ? D / GROUP4 : 1);
  p.there = true;
  return p;
}

__device__ __forceinline__ uint32_t max_with(uint32_t v, int lane_xor) { return max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), lane_xor))); }
// the largest magnitude of 8 values by its bits: they order like the values, infinities and NaN last
__device__ __forceinline__ uint32_t magnitude8(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
  return m;
}
// max over the D / 8 lanes of a row
template <int D>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max_with(max_with(max_with(v, 1), 2), 4);
  if constexpr (D == 128) v = max_with(v, 8);
  return v;
}

template <int FMT, int D>
__device__ __forceinline__ void put8(const float* x, uint8_t* codes, float* scale, bool first) {
  const uint32_t m = row_max<D>(magnitude8(x));
  uint2 q = make_uint2(0u, 0u);
  float s = __uint_as_float(0x7fc00000u);
  if (m < 0x7f800000u) {
    s = fmaxf(__uint_as_float(m) / (FMT == INT8 ? 127.0f : 448.0f), 1e-12f);
    const float inv = 1.0f / s;
    if constexpr (FMT == INT8)
      q = quant8_i8(x, s, inv);
    else
      q = quant8_fp8(x, s, inv, fp8_odd(__uint_as_float(m), 0.0f, s));
  }
  *reinterpret_cast<uint2*>(codes) = q;
  if (first) *scale = s;
}

// lane l of a row's D / 8: its 8 values of a key (x) and value (y) of head h to their codes
template <int FMT, int D>
__device__ __forceinline__ void put(const Cache& c, const Place& p, int h, int l, const float* x, const float* y) {
  if constexpr (FMT != FP4) {
    const int64_t code = p.code + h * c.head_stride + 8 * l, scale = p.scale + h * c.shead_stride;
    put8<FMT, D>(x, c.k + code, c.ks + scale, l == 0);
    put8<FMT, D>(y, c.v + code, c.vs + scale, l == 0);
  } else {
    // 4 lanes are a group. An infinity or a NaN anywhere in the two rows marks the position: key scales 255, all else 0
    const uint32_t mk = max_with(max_with(magnitude8(x), 1), 2), mv = max_with(max_with(magnitude8(y), 1), 2);
    uint32_t all = max_with(max(mk, mv), 4);
    if constexpr (D == 128) all = max_with(all, 8);
    uint32_t sk = 255, sv = 0, wk = 0, wv = 0;
    if (all < 0x7f800000u) {
      sk = scale4(mk);
      sv = scale4(mv);
      wk = codes4(x, sk);
      wv = codes4(y, sv);
    }
    const int64_t code = p.code + h * c.head_stride + 4 * l, scale = p.scale + h * c.shead_stride + l / 4;
    *reinterpret_cast<uint32_t*>(c.k + code) = wk;
    *reinterpret_cast<uint32_t*>(c.v + code) = wv;
    if (l % 4 == 0) {
      reinterpret_cast<uint8_t*>(c.ks)[scale] = static_cast<uint8_t>(sk);
      reinterpret_cast<uint8_t*>(c.vs)[scale] = static_cast<uint8_t>(sv);
    }
  }
}

// A lane's 8 values of a row as they lie
template <int DT>
struct Raw {
  uint4 w[DT == RH3_DTYPE_F32 ? 2 : 1];
};
// once: 16-bit rows that are best kept out of the last cache
template <int DT>
__device__ __forceinline__ Raw<DT> load_raw(const void* p, int64_t at, bool once = false) {
  Raw<DT> r;
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + at * (DT == RH3_DTYPE_F32 ? 4 : 2));
  if constexpr (DT == RH3_DTYPE_F32) {
    r.w[0] = src[0];
    r.w[1] = src[1];
  } else {
    r.w[0] = once ? ld_stream16(src) : src[0];
  }
  return r;
}
template <int DT>   // bf16 or fp16
__device__ __forceinline__ void store_row8_once(void* p, int64_t at, const float* v) {
  uint4 r;
  store_row8<DT>(&r, 0, v);
  const u32x4_t t = {r.x, r.y, r.z, r.w};
  __builtin_nontemporal_store(t, reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(p) + at));
}
constexpr int64_t LAST_CACHE = int64_t{256} << 20;
template <int DT>
__device__ __forceinline__ void values_of(const Raw<DT>& r, float* x) {
  if constexpr (DT == RH3_DTYPE_F32) {
    const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
  } else {
    row8<DT>(r.w[0], x);
  }
}

// Workgroups for `rows` rows: along x the rows, along y as many heads side by side as it takes for 8 workgroups to a CU, or 32 where
// that leaves a workgroup 8 heads (22,332 rows x 56 heads in int8: written in 218 and 208 us, read in 202 and 193; in 4 bits 157
// and 159, 128 and 127; 24,009 x 8: 28.2 and 29.8, 24.9 and 24.1); the other heads are the workgroup's loop, which resolves a row's
// page once for all of them.
inline dim3 grid_of(int64_t rows, int heads, int dim) {
  const int64_t gx = (rows + NT / (dim / 8) - 1) / (NT / (dim / 8));
  const int64_t cus = device_cus() > 0 ? device_cus() : 256;
  int64_t few = (8 * cus + gx - 1) / gx, many = (32 * cus + gx - 1) / gx;
  many = many > heads / 8 ? heads / 8 : many;
  int64_t gy = few > many ? few : many;
  gy = gy < 1 ? 1 : gy > heads ? heads : gy;
  return dim3(static_cast<uint32_t>(gx), static_cast<uint32_t>(gy));
}

}  // namespace kv
}  // namespace rh3
