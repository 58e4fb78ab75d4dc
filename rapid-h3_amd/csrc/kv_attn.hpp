// Attention over the paged cache: what its kernels share. kv_token.hip runs few query rows to a K/V head (bound by the cache's
// bytes), kv_chunk.hip many (bound by the matrix units), kv_attn.hip joins the parts that either leaves and holds the entry points.
//
// For a query row i of a sequence of n rows and `len` cached positions: o_i = sum_j p_ij v_j / sum_j p_ij with
// p_ij = exp(scale q_i.k_j) over j < len, and j <= pos + i (pos = len - n) if causal. A K/V head's query rows are its group's heads
// of every token of the sequence, numbered token * group + head in the group, so that the group shares each key and value that is
// read.
//
// Arithmetic. Codes are small integers (int8) or 4-bit significands (e4m3): exact in f16. A query row is scaled by the power of
// two that brings its largest magnitude to [2^14, 2^15) (the chunk kernel: the largest of all rows of its tile, where none is far
// below it): bf16 and fp16 values are exact in f16 after it (those 2^28 below lose low bits, 2^-40 of it at most). So q.k is a sum
// of exact products in fp32 on the f16 MFMA, times the key's scale, in fp32. Probabilities are taken against a reference 10 to 15
// under the row's running maximum (base 2), so that in f16 they use its range from 2^15 down, rounded to nearest (2^-11 relative at
// most); where they are multiplied by value scales first, the products keep that precision down to 2^-24 of the row's largest.
// Their sum is fp32.
#pragma once

#include "kv_common.hpp"

namespace rh3 {
namespace kv {

// A part: the unnormalised sum of a query row over some of its keys, times PART (probabilities of up to 2^15 of very many keys with
// values near fp32's largest), with the fp32 sum of its probabilities and their reference (base 2). Slots of parts hold R rows
// each: part_o [slot][R][dim], part_ml [slot][R][2] (reference, sum).
constexpr float PART = 0x1p-32f;

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
  // A prefix that all sequences' rows see, taken as the first sequence (those rows its own, no causal limit) by the launch that
  // also does the others, or by one for it alone; or null
  const int32_t* prefix;
  int prefix_len, prefix_width, alone;
  int64_t items;             // slots of completed items
  int wgs;
  int keep;                  // leave a part for every item, also for those that one workgroup completes
};

// ---------------------------------------------------------------- the kernels' work, the same on every wave that asks
// Items: (sequence, K/V head, R query rows of it). Units: KEYS keys of an item. The units of all items in order (sequences, then
// K/V heads, then row tiles) are dealt to the workgroups in equal contiguous ranges, so that uneven histories, which only the
// device knows, load the workgroups evenly. `least` units at least make a workgroup worth starting.
// An item counts `extra` units before its keys, about what beginning one takes: without them a workgroup with several short items
// would have as many keys as one with a long one, and take longer.
struct Tiling {
  int rows, keys, extra, least;
};
constexpr int TOKEN_KEYS = 32, CHUNK_KEYS = 64;
RH3_HD Tiling tiling(bool chunk, int rows) { return chunk ? Tiling{rows, CHUNK_KEYS, 4, 8} : Tiling{rows, TOKEN_KEYS, 4, 4}; }

// Units are counted in 64 bits; a division of what fits 32 bits is done there (a 64-bit one takes some hundred instructions).
RH3_HD int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 31) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
struct Work {
  int wgs;                   // workgroups that have a share
  int64_t each, more;        // the first `more` of them have each + 1 units, the others each
};
RH3_HD Work dealt(int64_t units, int wgs, const Tiling& g) {
  Work w;
  const int64_t most = (units + g.least - 1) / g.least;
  w.wgs = static_cast<int>(most < wgs ? (most > 0 ? most : 1) : wgs);
  w.each = quotient(units, w.wgs);
  w.more = units - w.each * w.wgs;
  return w;
}
RH3_HD int64_t share_begin(const Work& w, int wg) { return w.each * wg + (wg < w.more ? wg : w.more); }
// the workgroup whose share holds unit u
RH3_HD int share_of(const Work& w, int64_t u) {
  const int64_t head = w.more * (w.each + 1);
  return static_cast<int>(u < head ? quotient(u, w.each + 1) : w.more + quotient(u - head, w.each));
}

// a sequence of the launch: the prefix, if there is one, before the batch's
RH3_HD int sequences(const AttnArgs& a) { return (a.alone ? 0 : a.s.batch) + (a.prefix != nullptr); }
RH3_HD Seq sequence(const AttnArgs& a, int i) {
  if (a.prefix) {
    if (i == 0) {
      const int first = a.s.cu ? clamped(a.s.cu[0], 0, a.s.rows) : 0;
      return Seq{first, (a.s.cu ? clamped(a.s.cu[a.s.batch], first, a.s.rows) : a.s.rows) - first, a.prefix_len, 0};
    }
    --i;
  }
  return seq_at(a.s, i);
}

struct SeqWork {
  int row_tiles, span;       // span: units of an item
  int64_t units;
};
RH3_HD SeqWork work_of(const AttnArgs& a, const Seq& q, const Tiling& g) {
  SeqWork w;
  w.row_tiles = static_cast<int>((static_cast<int64_t>(q.n) * a.group + g.rows - 1) / g.rows);
  const int kt = (q.len + g.keys - 1) / g.keys;
  w.span = (kt < 1 ? 1 : kt) + g.extra;
  // no memory holds 2^36 units (2^41 keys); offsets in cu that fall can count rows many times, and must not overflow the sums
  const int64_t u = static_cast<int64_t>(a.c.heads) * w.row_tiles;
  w.units = u < (int64_t{1} << 36) / w.span ? u * w.span : int64_t{1} << 36;
  return w;
}

// Sums over the lanes before and at each one, by lane moves within rows of 16 and two broadcasts over them
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t scan_step(int64_t v) {
  const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, true);
  return v + ((static_cast<int64_t>(hi) << 32) | static_cast<uint32_t>(lo));
}
__device__ __forceinline__ int64_t wave_scan(int64_t v) {   // inclusive
  v = scan_step<0x111, 0xf>(v);   // row_shr:1, 2, 4, 8
  v = scan_step<0x112, 0xf>(v);
  v = scan_step<0x114, 0xf>(v);
  v = scan_step<0x118, 0xf>(v);
  v = scan_step<0x142, 0xa>(v);   // row_bcast:15 into rows 1 and 3
  v = scan_step<0x143, 0xc>(v);   // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int64_t lane64(int64_t v, int lane) {
  return (static_cast<int64_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane)) << 32) |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

// 64 sequences, one to a lane, and the units and items (row tiles of all K/V heads) up to each
struct Block {
  int at;                          // the first of them
  int64_t base, items_base;        // units and items before it
  Seq seq;
  int64_t units, items;            // running sums within the block, this lane's included
  int row_tiles, span;
  __device__ __forceinline__ int64_t end() const { return base + lane64(units, 63); }
};
__device__ __forceinline__ void load_block(const AttnArgs& a, const Tiling& g, int at, int64_t base, int64_t items_base, Block& b) {
  const int i = at + (threadIdx.x & 63);
  b.at = at;
  b.base = base;
  b.items_base = items_base;
  b.seq = Seq{0, 0, 0, 0};
  SeqWork w{0, 1, 0};
  if (i < sequences(a)) {
    b.seq = sequence(a, i);
    w = work_of(a, b.seq, g);
  }
  b.row_tiles = w.row_tiles;
  b.span = w.span;
  b.units = wave_scan(w.units);
  b.items = a.keep ? wave_scan(static_cast<int64_t>(a.c.heads) * w.row_tiles) : 0;
}
// the first block, and the units of all
__device__ __forceinline__ int64_t load_blocks(const AttnArgs& a, const Tiling& g, Block& b) {
  load_block(a, g, 0, 0, 0, b);
  int64_t total = b.end();
  for (int at = 64; at < sequences(a); at += 64) {
    Block next;
    load_block(a, g, at, 0, 0, next);
    total += next.end();
  }
  return total;
}
__device__ __forceinline__ void next_block(const AttnArgs& a, const Tiling& g, Block& b) {
  load_block(a, g, b.at + 64, b.end(), b.items_base + lane64(b.items, 63), b);
}

// a sequence of the block by its lane, the same in all lanes
struct SeqItems {
  Seq seq;
  int row_tiles, span;
  int64_t before, items_before;    // units, items of the sequences before it
};
__device__ __forceinline__ SeqItems seq_in(const AttnArgs& a, const Block& b, int l) {
  SeqItems r;
  r.seq.first = __builtin_amdgcn_readlane(b.seq.first, l);
  r.seq.n = __builtin_amdgcn_readlane(b.seq.n, l);
  r.seq.len = __builtin_amdgcn_readlane(b.seq.len, l);
  r.seq.pos = __builtin_amdgcn_readlane(b.seq.pos, l);
  r.row_tiles = __builtin_amdgcn_readlane(b.row_tiles, l);
  r.span = __builtin_amdgcn_readlane(b.span, l);
  r.before = b.base + (l ? lane64(b.units, l - 1) : 0);
  r.items_before = b.items_base + (l ? lane64(b.items, l - 1) : 0);
  return r;
}

// The chunk kernel's causal row tiles are taken from both ends in turn (0, n - 1, 1, n - 2, ..), so that the long and short ones
// of a share even out: the tile at a place, and the place of a tile
RH3_HD int tile_at_place(int at, int n) { return at & 1 ? n - 1 - (at >> 1) : at >> 1; }
RH3_HD int place_of_tile(int rt, int n) { return rt < (n + 1) / 2 ? 2 * rt : 2 * (n - 1 - rt) + 1; }

// A value that is the same in all lanes, as a scalar: a division is done by vector instructions, and what depends on its result
// (loop bounds, addresses) would stay in vector registers
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t scalar(int64_t v) { return lane64(v, 0); }

// ---------------------------------------------------------------- query rows
// the exponent that brings a magnitude to [2^14, 2^15) (zero, infinite or NaN: none)
__device__ __forceinline__ int q_exponent(float amax) {
  const int e = static_cast<int>(__float_as_uint(amax) >> 23) & 255;
  return e == 0 || e == 255 ? 0 : 141 - e;
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
// (from 2^27 on a score's last place is 16: a reference that would come to lie that far under the maximum is the maximum itself)
__device__ __forceinline__ float reference_under(float top) {
  const float r = top - REF_UNDER;
  return top - r > REF_STALE ? top : r;
}

// the power of two over a scale, at least 2^-111 (NaN never gets here)
__device__ __forceinline__ float pow2_over(float v) {
  const uint32_t e = (__float_as_uint(v) >> 23) & 255u;
  return __uint_as_float(min(max(e + 1u, 16u), 253u) << 23);
}

// The unit of a row's weights (probability times value scale, in f16) where its probabilities so far are scaled by f (at most 1)
// and the largest weight of the next keys is w base: a power of two. The weights so far are in fp32 sums and may lie under it.
constexpr float WEIGHT_MOST = 0x1p15f;
__device__ __forceinline__ float weight_unit(float unit, float f, float w, float base) {
  const float kept = unit * __uint_as_float(__float_as_uint(f) & 0x7f800000u);
  return fmaxf(fmaxf(kept, base * (pow2_over(w) * 0x1p-11f)), 0x1p-120f);
}

// 1 over a power of two given by its bits (exponents 1 to 253)
__device__ __forceinline__ float pow2_inverse(int bits) { return __int_as_float((254 << 23) - bits); }

__device__ __forceinline__ uint32_t pack_out(const AttnArgs& a, float x, float y) { return a.fp16 ? pack_h2(x, y) : pack_bf2(x, y); }

// host: launches of the two kernels for their checked arguments
void launch_token(const AttnArgs& a, int fmt, int dim, int rows, hipStream_t st);
void launch_chunk(const AttnArgs& a, int fmt, int dim, int rows, hipStream_t st);

}  // namespace kv
}  // namespace rh3
