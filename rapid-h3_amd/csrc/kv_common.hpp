// Shared by the kernels of the paged key / value cache (kv_cache.hip, kv_token.hip, kv_chunk.hip, their 4-bit forms,
// kv_attn.hip): where a sequence's rows and positions lie, page lookups, and the conversion of 8-bit codes to f16.
//
// A cache is pages of `page` positions: codes [P][heads][page][dim], one fp32 scale per code row [P][heads][page] (4-bit format:
// bytes of two codes [..][dim / 2], scale bytes [..][dim / 32], kv_four.hpp). Position p of sequence b lies in page
// table[b][p / page]; an entry outside [0, P) is an absent page, whose positions hold nothing.
// Everything that comes from device memory (lengths, row offsets, page numbers) is clamped before it addresses anything, so no
// content of these arrays can make an access leave the caller's buffers.
#pragma once

#include "rh3_common.hpp"

#define RH3_HD __host__ __device__ __forceinline__

namespace rh3 {
namespace kv {

constexpr int INT8 = RH3_KV_INT8;
constexpr int E4M3 = RH3_KV_E4M3;
constexpr int FP4 = RH3_KV_FP4;

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f16_t __attribute__((ext_vector_type(16)));

struct Cache {
  uint8_t *k, *v;
  float *ks, *vs;
  int64_t page_stride, head_stride;     // of codes, in bytes
  int64_t spage_stride, shead_stride;   // of scales, in floats (4-bit format: in bytes)
  int pages, heads, log2page;
};

// batch sequences: `rows` packed rows, those of sequence b at cu[b] .. cu[b + 1] (cu null: `per` each); lens[b] cached
// positions. The rows of a sequence are its last positions, row cu[b + 1] - 1 the last of all, whether the call has that row or not.
struct Seqs {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* cu;
  int width, batch, rows, per, cap;   // cap: width * page
};

struct Seq {
  int first, n, len;   // rows [first, first + n), cached positions that the table has
  int pos;             // of row `first`: negative or past len where it has no place
};

constexpr int64_t MAX_ROWS = int64_t{1} << 30;   // of a call, and positions of a table

RH3_HD int clamped(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
// row0: the position that row 0 of the call would have in the sequence, not clamped as `pos` is (to what the table can hold)
RH3_HD Seq seq_at(const Seqs& s, int b, int64_t& row0) {
  Seq r;
  int64_t end;
  if (s.cu) {
    end = s.cu[b + 1];
    r.first = clamped(s.cu[b], 0, s.rows);
    r.n = clamped(static_cast<int>(end), r.first, s.rows) - r.first;
  } else {
    r.first = b * s.per;
    r.n = s.per;
    end = r.first + r.n;
  }
  const int64_t len = s.lens[b], pos = len - end + r.first;
  row0 = len - end;
  r.len = clamped(static_cast<int>(len), 0, s.cap);
  r.pos = static_cast<int>(pos < -MAX_ROWS ? -MAX_ROWS : pos > s.cap ? s.cap : pos);
  return r;
}
RH3_HD Seq seq_at(const Seqs& s, int b) {
  int64_t row0;
  return seq_at(s, b, row0);
}

// The sequence of a row: the last b with cu[b] <= row, by a search over LANES (8, 16 or 64) lanes that hold the same
// row, or -1 for a row that no sequence has (behind the last one, or in a cu that does not rise).
template <int LANES>
__device__ __forceinline__ int seq_of_row(const Seqs& s, int row, Seq& q, int64_t& row0) {
  int b;
  if (!s.cu) {
    b = row / s.per;
    if (b >= s.batch) return -1;
  } else {
    const int lane = threadIdx.x & 63, l = lane & (LANES - 1);
    int lo = 0, n = s.batch;             // the answer is in [lo, lo + n)
    while (n > 1) {
      const int step = (n + LANES - 1) / LANES;
      const int at = lo + l * step;
      const bool le = at < lo + n && s.cu[at] <= row;
      unsigned long long m = __builtin_amdgcn_ballot_w64(le);
      if constexpr (LANES < 64) m = (m >> (lane & ~(LANES - 1))) & ((1ull << LANES) - 1);
      const int c = max(static_cast<int>(__popcll(m)), 1) - 1;   // none: a row in front of cu[lo]
      n = min(step, lo + n - (lo + c * step));
      lo += c * step;
    }
    b = lo;
  }
  q = seq_at(s, b, row0);
  return row >= q.first && row < q.first + q.n ? b : -1;
}
template <int LANES>
__device__ __forceinline__ int seq_of_row(const Seqs& s, int row, Seq& q) {
  int64_t row0;
  return seq_of_row<LANES>(s, row, q, row0);
}

// page of a position of sequence b (pos < cap), or -1
RH3_HD int page_of(const Seqs& s, const Cache& c, int b, int pos) {
  const int p = s.table[b * s.table_stride + (pos >> c.log2page)];
  return p >= 0 && p < c.pages ? p : -1;
}

// a table entry by the scalar cache: the same address in all lanes, and nothing that a kernel of this call writes
__device__ __forceinline__ int scalar_load(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)(p);
}

// ---------------------------------------------------------------- codes to f16, exact
// int8: the byte c + 128 beside 0x64 is the f16 1024 + (c + 128), from which one packed subtraction takes 1152
// (a permute, an xor and a packed add per two codes). e4m3: the hardware conversion (its scale operand 1).
__device__ __forceinline__ h2_t f16_of_spread(uint32_t w) {   // codes in bytes 0 and 2, the others 0
  const h2_t m = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
  return __builtin_bit_cast(h2_t, w ^ 0x64806480u) - m;
}
__device__ __forceinline__ h8_t join(h2_t a, h2_t b, h2_t c, h2_t d) {
  h8_t r;
  r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1];
  r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
  return r;
}
// 8 consecutive codes (two words) to f16
template <int FMT>
__device__ __forceinline__ h8_t f16x8(uint32_t lo, uint32_t hi) {
  if constexpr (FMT == INT8) {
    return join(f16_of_spread(__builtin_amdgcn_perm(0u, lo, 0x0c010c00u)), f16_of_spread(__builtin_amdgcn_perm(0u, lo, 0x0c030c02u)),
                f16_of_spread(__builtin_amdgcn_perm(0u, hi, 0x0c010c00u)), f16_of_spread(__builtin_amdgcn_perm(0u, hi, 0x0c030c02u)));
  } else {
    return join(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true),
                __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
  }
}
// w[0 .. 7]: words of 4 channels at 8 positions -> for each of the channels, its 8 positions as f16
template <int FMT>
__device__ __forceinline__ void f16x8_across(const uint32_t (&w)[8], h8_t (&o)[4]) {
  if constexpr (FMT == INT8) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t sel = 0x0c040c00u + static_cast<uint32_t>(c) * 0x00010001u;
      o[c] = join(f16_of_spread(__builtin_amdgcn_perm(w[1], w[0], sel)), f16_of_spread(__builtin_amdgcn_perm(w[3], w[2], sel)),
                  f16_of_spread(__builtin_amdgcn_perm(w[5], w[4], sel)), f16_of_spread(__builtin_amdgcn_perm(w[7], w[6], sel)));
    }
  } else {
#pragma unroll
    for (int p = 0; p < 2; ++p) {      // channels 2p and 2p + 1
      const uint32_t sel = p ? 0x07030602u : 0x05010400u;
      const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], sel), b = __builtin_amdgcn_perm(w[3], w[2], sel);
      const uint32_t c = __builtin_amdgcn_perm(w[5], w[4], sel), d = __builtin_amdgcn_perm(w[7], w[6], sel);
      o[2 * p] = f16x8<E4M3>(__builtin_amdgcn_perm(b, a, 0x05040100u), __builtin_amdgcn_perm(d, c, 0x05040100u));
      o[2 * p + 1] = f16x8<E4M3>(__builtin_amdgcn_perm(b, a, 0x07060302u), __builtin_amdgcn_perm(d, c, 0x07060302u));
    }
  }
}

// ---------------------------------------------------------------- rows of bf16 / fp16 / fp32
template <int DT>   // bf16 or fp16
__device__ __forceinline__ void row8(const uint4 r, float* v) {
  if constexpr (DT == RH3_DTYPE_BF16) {
    unpack8(r, v);
  } else {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const h2_t h = __builtin_bit_cast(h2_t, w[i]);
      v[2 * i] = static_cast<float>(h[0]);
      v[2 * i + 1] = static_cast<float>(h[1]);
    }
  }
}
template <int DT>
__device__ __forceinline__ void load_row8(const void* p, int64_t at, float* v) {
  if constexpr (DT == RH3_DTYPE_F32) {
    const float4 a = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at)[0];
    const float4 b = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    row8<DT>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at), v);
  }
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {   // round to nearest even
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t{a, b}), h2_t));
}
template <int DT>
__device__ __forceinline__ void store_row8(void* p, int64_t at, const float* v) {
  if constexpr (DT == RH3_DTYPE_F32) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    o[0] = make_float4(v[0], v[1], v[2], v[3]);
    o[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint4 r;
    if constexpr (DT == RH3_DTYPE_BF16)
      r = make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
    else
      r = make_uint4(pack_h2(v[0], v[1]), pack_h2(v[2], v[3]), pack_h2(v[4], v[5]), pack_h2(v[6], v[7]));
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) = r;
  }
}

// ---------------------------------------------------------------- host: the checks that every entry point shares
// fills c and s; RH3_EINVAL with a message if the call cannot be run
int check_cache(const char* name, const rh3_kv_cache* cache, Cache& c);
int check_seqs(const char* name, const Cache& c, const int32_t* table, int64_t table_stride, int64_t width, const int32_t* lens,
               const int32_t* cu, int64_t batch, int64_t rows, Seqs& s);

}  // namespace kv
}  // namespace rh3
