// Attention over the paged cache: joining the parts that the token and chunk kernels leave, and the entry points.
#include "kv_attn.hpp"

namespace rh3 {
namespace kv {
namespace {

// A launch that has left parts
struct Source {
  AttnArgs a;
  int chunk, rows;    // kernel, rows of its tiles
};

// the parts of one query row: slot(i), i < count, and the row in each slot
struct Parts {
  int64_t first, next;
  int count, row;
  __device__ __forceinline__ int64_t slot(int i) const { return i == 0 ? first : next + 2 * (i - 1); }
};
// of row r of a K/V head of the launch's sequence b
__device__ __forceinline__ Parts parts_of(const Source& s, const Work& w, const SeqItems& sw, const Tiling& g, bool causal, int64_t r, int kvh) {
  Parts p;
  const int rt = scalar(static_cast<int>(quotient(r, s.rows)));
  p.row = static_cast<int>(r - static_cast<int64_t>(rt) * s.rows);
  const int64_t item = static_cast<int64_t>(kvh) * sw.row_tiles + (s.chunk && causal ? place_of_tile(rt, sw.row_tiles) : rt);
  const int64_t u = sw.before + item * sw.span;
  const int w0 = share_of(w, u + g.extra), w1 = share_of(w, u + sw.span - 1);
  p.next = 2 * (static_cast<int64_t>(w0) + 1);
  p.first = 2 * static_cast<int64_t>(w0) + 1;
  p.count = w1 - w0 + 1;
  if (w0 == w1) {
    p.first = 2 * static_cast<int64_t>(s.a.wgs) + sw.items_before + item;
    p.count = s.a.keep && sw.items_before + item < s.a.items ? 1 : 0;   // (a cu that falls can count rows more than once)
  }
  return p;
}

// Sums of a row's parts on WPR waves, each of which takes every WPR-th part: lane l has channels EPL l .. of them
template <int D>
struct Sums {
  static constexpr int EPL = D / 64;
  float o[EPL], sum;
  __device__ __forceinline__ void add(const AttnArgs& a, int64_t at, float top) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
    const float f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - top);
    sum += f * ml.y;
    const float* po = a.part_o + at * D + EPL * (threadIdx.x & 63);
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] += f * po[e];
  }
  __device__ __forceinline__ void store(const AttnArgs& a, int tok, int hd, float top) const {
    const int lane = threadIdx.x & 63;
    const float inv = sum == 0.0f ? 0.0f : (1.0f / PART) / sum;
    uint16_t* dst = static_cast<uint16_t*>(a.out) + tok * a.o_st + hd * a.o_sh + EPL * lane;
    if constexpr (EPL == 2) *reinterpret_cast<uint32_t*>(dst) = pack_out(a, o[0] * inv, o[1] * inv);
    else *dst = static_cast<uint16_t>(pack_out(a, o[0] * inv, 0.0f));
    if (a.lse && lane == 0)
      a.lse[static_cast<int64_t>(tok) * a.c.heads * a.group + hd] = sum == 0.0f ? -INFINITY : (__builtin_amdgcn_logf(sum) + top) * 0.6931471805599453f;
  }
};

// Every query row of the call, WPR waves to one: where a row has many parts (few items on all workgroups), or a prefix's beside its
// own (of the same launch, or of `prefix`). Bound by latency: a row's parts are a few KB to some hundred (4 rows x 56 heads in 16
// parts 5.7 us; 64 x 32 with a prefix's 33 parts each, 38 MB, 14.5).
template <int D, int WPR>
__global__ void __launch_bounds__(WPR > 4 ? WPR * 64 : 256) join_rows_kernel(Source own, Source prefix, int has_prefix) {
  constexpr int WAVES = WPR > 4 ? WPR : 4, EPL = D / 64;
  __shared__ float so[WAVES][D];
  __shared__ float sl[WAVES];
  const int lane = threadIdx.x & 63;
  const int wave = scalar(static_cast<int>(threadIdx.x >> 6));
  const int heads = own.a.c.heads * own.a.group;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (WAVES / WPR) + wave / WPR;
  const int tok = scalar(static_cast<int>(quotient(id, heads))), hd = static_cast<int>(id - static_cast<int64_t>(tok) * heads);
  if (tok >= own.a.s.rows) return;             // WPR > 1: the whole workgroup, before its barrier
  const int kvh = scalar(hd / own.a.group), ig = hd - kvh * own.a.group;
  Seq q;
  const int b = scalar(seq_of_row<64>(own.a.s, tok, q));
  if (b < 0) return;                           // a row that no sequence has stays as it is
  Parts p[2];
  p[1].count = 0;
  {
    Block blk;
    const Tiling g = tiling(own.chunk, own.rows);
    const Work w = dealt(load_blocks(own.a, g, blk), own.a.wgs, g);
    const int64_t all = static_cast<int64_t>(tok) * own.a.group + ig;
    int at = b;
    auto of_prefix = [&](const Source& s, const Work& w, const Tiling& g) {
      const SeqItems sw = seq_in(s.a, blk, 0);
      const int64_t r = all - static_cast<int64_t>(sw.seq.first) * own.a.group;
      if (r >= 0 && tok < sw.seq.first + sw.seq.n) p[1] = parts_of(s, w, sw, g, false, r, kvh);   // (not so where a cu falls)
    };
    if (own.a.prefix) {
      of_prefix(own, w, g);
      ++at;
    }
    while (at >= blk.at + 64) next_block(own.a, g, blk);
    p[0] = parts_of(own, w, seq_in(own.a, blk, at - blk.at), g, own.a.causal, all - static_cast<int64_t>(q.first) * own.a.group, kvh);
    if (has_prefix) {
      const Tiling gp = tiling(prefix.chunk, prefix.rows);
      const Work wp = dealt(load_blocks(prefix.a, gp, blk), prefix.a.wgs, gp);
      of_prefix(prefix, wp, gp);
    }
  }
  if (p[0].count + p[1].count == 0) return;    // one workgroup completed it
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const Source& s = k && has_prefix ? prefix : own;
    for (int i = lane; i < p[k].count; i += 64) top = fmaxf(top, s.a.part_ml[(p[k].slot(i) * s.rows + p[k].row) * 2]);
  }
  top = wave_max(top);
  Sums<D> r{};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const Source& s = k && has_prefix ? prefix : own;
#pragma unroll 4
    for (int i = wave % WPR; i < p[k].count; i += WPR) r.add(s.a, p[k].slot(i) * s.rows + p[k].row, top);
  }
  if constexpr (WPR > 1) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) so[wave][EPL * lane + e] = r.o[e];
    if (lane == 0) sl[wave] = r.sum;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) r.o[e] += so[w][EPL * lane + e];
      r.sum += sl[w];
    }
  }
  r.store(own.a, tok, hd, top);
}

// Only the items that shares divide, at most one to a boundary of two shares: workgroup (w, y) joins rows 16 y .. of the item that
// begins in share w and goes on behind it, if there is one. Measured: 32 rows 4.8 us, 2,048 x 32 heads 7.4, 1,560 x 56 heads 20.
template <int D>
__global__ void __launch_bounds__(256) join_shares_kernel(Source own) {
  const AttnArgs& a = own.a;
  const Tiling g = tiling(own.chunk, own.rows);
  Block blk;
  const Work work = dealt(load_blocks(a, g, blk), a.wgs, g);
  const int w = blockIdx.x;
  if (w + 1 >= work.wgs) return;
  const int64_t end = scalar(share_begin(work, w + 1));
  while (end > blk.end()) {
    if (blk.at + 64 >= sequences(a)) return;
    next_block(a, g, blk);
  }
  const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(blk.base + blk.units >= end));   // the share's last unit is its
  const SeqItems sw = seq_in(a, blk, l);
  const int item = scalar(static_cast<int>(quotient(end - 1 - sw.before, sw.span)));
  const int64_t last = sw.before + (static_cast<int64_t>(item) + 1) * sw.span;               // end of the item
  const int64_t begin = last - sw.span + g.extra;                                            // its first key's unit
  if (last == end || begin >= end || begin < share_begin(work, w)) return;
  const int parts = scalar(share_of(work, last - 1)) - w + 1;
  const int kvh = scalar(item / sw.row_tiles), at = item - kvh * sw.row_tiles;
  const int rt = own.chunk && a.causal ? tile_at_place(at, sw.row_tiles) : at;
  const int wave = scalar(static_cast<int>(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  const int rows = sw.seq.n * a.group;
  // a wave's 4 rows side by side: their loads do not wait for each other
  const int row0 = 16 * blockIdx.y + 4 * wave;
  if (rt * own.rows + row0 >= rows) return;
  auto slot = [&](int j) { return (2 * static_cast<int64_t>(w + j) + (j == 0)) * own.rows + row0; };
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  for (int j = lane; j < parts; j += 64)
#pragma unroll
    for (int i = 0; i < 4; ++i) top[i] = fmaxf(top[i], a.part_ml[2 * (slot(j) + i)]);
#pragma unroll
  for (int i = 0; i < 4; ++i) top[i] = wave_max(top[i]);
  Sums<D> r[4] = {};
#pragma unroll 2
  for (int j = 0; j < parts; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i].add(a, slot(j) + i, top[i]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rw = rt * own.rows + row0 + i;
    if (rw >= rows) return;
    const int tok = scalar(rw / a.group);
    r[i].store(a, sw.seq.first + tok, kvh * a.group + rw - tok * a.group, top[i]);
  }
}

// ---------------------------------------------------------------- host: how a call runs
struct Plan {
  int chunk, rows;        // kernel, query rows of its tiles
  int wgs;
  int64_t items;          // slots for items that one workgroup completes
  int64_t slots;          // parts it may leave
};

// rows: of a call; per sequence they are counted as even. keep: a part for every item.
// The token kernel reads the keys once for every 16 (dim 64: 32) query rows of a K/V head, at some 6.8 TB/s, mostly from L2 from
// the second time on; the chunk kernel once for 128 or 256, as 3 TB/s at most (it is bound by its arithmetic), after some 34 us
// that its longer beginning, end and joins take. The lengths are the device's: the table's width stands for them. Measured (us a
// call, token / chunk, 8 K/V heads of 128, rows of a K/V head): 1 sequence of 16,384 keys: 32 rows 24 / 39, 96 41 / 49, 128 45 / 53,
// 192 58 / 47, 256 67 / 53; 16 of 4,096: 32 50 / 66, 48 68 / 71, 64 82 / 73, 96 121 / 80; 4 of 65,536: 32 140 / 188, 48 285 / 197;
// 4 of 1,024: 16 16 / 37, 256 24 / 49. Heads of 64: 1 of 65,536: 128 60 / 70, 192 81 / 80, 256 103 / 87; 4: 96 150 / 158, 128 186 / 169.
Plan plan_of(int64_t rows, int64_t batch, bool even, int64_t group, int64_t heads, int64_t dim, int64_t cap, bool keep, int form) {
  const int64_t cus = device_cus() > 0 ? device_cus() : 256;
  const int64_t mean = (rows * group + batch - 1) / batch;    // query rows of a sequence's K/V head
  const int small = dim == 64 && mean > 16 ? 32 : 16;
  const double mb = 2e-6 * static_cast<double>(dim + 4) * static_cast<double>(batch * heads) * static_cast<double>(cap);
  Plan p{};
  p.chunk = form != RH3_KV_BY_SIZE ? form == RH3_KV_CHUNK : static_cast<double>((mean + small - 1) / small) * mb / 6.8 > 34.0 + static_cast<double>((mean + 127) / 128) * mb / 3.0;
  p.rows = !p.chunk ? small : mean <= 128 ? 128 : 256;
  p.wgs = static_cast<int>(p.rows == 256 ? cus : 2 * cus);
  p.items = !keep ? 0 : heads * (even ? batch * ((rows / batch * group + p.rows - 1) / p.rows) : rows * group / p.rows + batch);
  p.slots = 2 * static_cast<int64_t>(p.wgs) + p.items;
  return p;
}
int64_t bytes_of(const Plan& p, int64_t dim) { return p.slots * p.rows * (dim + 2) * 4; }

struct Call {
  Plan own, prefix;
  bool joined;            // the prefix is a sequence of the one launch
  int64_t bytes;
};
Call call_of(int64_t rows, int64_t q_heads, int64_t heads, int64_t dim, int64_t cap, int64_t batch, bool even, int64_t prefix_len, int form) {
  Call c{};
  const int64_t group = q_heads / heads;
  c.own = plan_of(rows, batch, even, group, heads, dim, cap, prefix_len > 0, form);
  if (prefix_len > 0) {
    c.prefix = plan_of(rows, 1, true, group, heads, dim, prefix_len, true, form);
    c.joined = c.own.chunk == c.prefix.chunk;   // the prefix's rows then go by the sequences' tiles
    if (c.joined) {
      const int64_t items = heads * ((rows * group + c.own.rows - 1) / c.own.rows);
      c.own.items += items;
      c.own.slots += items;
    } else {
      c.bytes += bytes_of(c.prefix, dim);
    }
  }
  c.bytes += bytes_of(c.own, dim);
  return c;
}

void launch(const AttnArgs& a, const Plan& p, int fmt, int dim, hipStream_t st) {
  if (p.chunk) launch_chunk(a, fmt, dim, p.rows, st);
  else launch_token(a, fmt, dim, p.rows, st);
}

}  // namespace
}  // namespace kv
}  // namespace rh3

using namespace rh3;
using namespace rh3::kv;

extern "C" int64_t rh3_kv_attention_workspace_bytes(int64_t q_heads, int64_t heads, int64_t dim, int64_t rows, int64_t capacity,
                                                    int64_t batch, int even, int64_t prefix_len, int form) {
  if (heads < 1 || heads > 65535 || q_heads < heads || q_heads % heads || rows < 1 || rows > MAX_ROWS || q_heads / heads > MAX_ROWS / rows ||
      batch < 1 || batch > 65536 || capacity < 1 || capacity > MAX_ROWS || prefix_len < 0 || prefix_len > MAX_ROWS || (dim != 64 && dim != 128))
    return 0;
  return call_of(rows, q_heads, heads, dim, capacity, batch, even != 0, prefix_len, form).bytes;
}

extern "C" int rh3_kv_attention(const rh3_kv_cache* cache, const void* q, int64_t q_st, int64_t q_sh, int64_t q_heads, int dtype,
                                int64_t rows, const int32_t* table, int64_t table_stride, int64_t width, const int32_t* lens,
                                const int32_t* cu, int64_t batch, int causal, float scale, void* out, int64_t o_st, int64_t o_sh,
                                float* lse, const int32_t* prefix, int64_t prefix_len, int form, void* workspace,
                                int64_t workspace_bytes, hipStream_t stream) {
  clear_error();
  AttnArgs a{};
  if (const int e = check_cache("kv_attention", cache, a.c)) return e;
  if (const int e = check_seqs("kv_attention", a.c, table, table_stride, width, lens, cu, batch, rows, a.s)) return e;
  if (rows == 0) return RH3_OK;
  RH3_REQUIRE(dtype == RH3_DTYPE_BF16 || dtype == RH3_DTYPE_F16, "kv_attention: query type %d (bf16 or fp16)", dtype);
  RH3_REQUIRE(q_heads >= a.c.heads && q_heads % a.c.heads == 0, "kv_attention: %lld query heads do not divide over %d K/V heads",
              static_cast<long long>(q_heads), a.c.heads);
  RH3_REQUIRE(q_heads / a.c.heads <= MAX_ROWS / rows, "kv_attention: %lld rows of %lld heads", static_cast<long long>(rows),
              static_cast<long long>(q_heads));
  RH3_REQUIRE(q && out, "kv_attention: null q or out");
  RH3_REQUIRE(aligned16(q) && aligned16(out) && q_st % 8 == 0 && q_sh % 8 == 0 && o_st % 8 == 0 && o_sh % 8 == 0,
              "kv_attention: q and out must be 16-byte aligned with strides that are multiples of 8");
  RH3_REQUIRE((rows == 1 || o_st != 0) && (q_heads == 1 || o_sh != 0), "kv_attention: rows or heads of out share memory");
  RH3_REQUIRE(prefix_len >= 0 && prefix_len <= MAX_ROWS && (prefix_len == 0 || prefix), "kv_attention: prefix of %lld positions without pages",
              static_cast<long long>(prefix_len));
  RH3_REQUIRE(form >= RH3_KV_BY_SIZE && form <= RH3_KV_CHUNK, "kv_attention: form %d", form);
  const int dim = static_cast<int>(cache->dim), fmt = static_cast<int>(cache->format);
  const Call call = call_of(rows, q_heads, a.c.heads, dim, width * cache->page, batch, cu == nullptr, prefix_len, form);
  RH3_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= call.bytes,
              "kv_attention: workspace of %lld bytes needed, %lld given", static_cast<long long>(call.bytes), static_cast<long long>(workspace_bytes));
  // Parts that a row may have: the workgroups over the least count of items, no more than the keys make. Measured (kernel us, by
  // shares / rows on 4 waves / on 16): 8 parts of 32 rows 5.1 / 4.7 / 5.7, 16 of 224 rows - / 6.3 / 7.7. Waves of one row each find
  // their way through the shares themselves, so many rows, which fill the chip, have one (us, rows on 1 wave / on 4): 192 rows
  // behind a prefix 7.9 / 6.1, 512 21.2 / 20.8 (whole calls, as those that follow), 768 21.6 / 22.1, 1,024 24.8 / 26.2, 1,536 29.5 /
  // 32.4; 2,048 of 33 parts 13.5 / 19.2; 4,096 of 16 parts 72 / 78 (whole calls).
  const int64_t ids = rows * q_heads, cap = width * cache->page + prefix_len;
  const int64_t tiles = (rows * (q_heads / a.c.heads) / batch + call.own.rows - 1) / call.own.rows;
  const int64_t shared = call.own.wgs / (batch * a.c.heads * (tiles > 0 ? tiles : 1));
  const int64_t most = cap / (call.own.chunk ? 8 * CHUNK_KEYS : 4 * TOKEN_KEYS), parts = shared < most ? shared : most;
  const bool by_shares = prefix_len == 0 && parts <= 8;
  const int wpr = parts > 32 ? 16 : ids <= 2 * device_cus() ? 4 : 1;
  const int64_t waves = wpr == 1 ? (ids + 3) / 4 : ids;   // workgroups of the join by rows
  RH3_REQUIRE(by_shares || waves * (wpr == 16 ? 4 : 1) <= MAX_GRID_256, "kv_attention: %lld rows of %lld heads behind a prefix in one call",
              static_cast<long long>(rows), static_cast<long long>(q_heads));
  a.q = q;
  a.q_st = q_st;
  a.q_sh = q_sh;
  a.fp16 = dtype == RH3_DTYPE_F16;
  a.group = static_cast<int>(q_heads / a.c.heads);
  a.causal = causal != 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = out;
  a.o_st = o_st;
  a.o_sh = o_sh;
  a.lse = lse;
  a.keep = prefix_len > 0;

  float* ws = static_cast<float*>(workspace);
  auto source = [&](AttnArgs x, const Plan& p) {
    x.items = p.items;
    x.wgs = p.wgs;
    x.part_o = ws;
    x.part_ml = ws + p.slots * p.rows * dim;
    ws += p.slots * p.rows * (dim + 2);
    return Source{x, p.chunk, p.rows};
  };
  auto with_prefix = [&](AttnArgs x) {
    x.prefix = prefix;
    x.prefix_len = static_cast<int>(prefix_len);
    x.prefix_width = static_cast<int>((prefix_len + cache->page - 1) / cache->page);
    return x;
  };
  const Source own = source(call.joined ? with_prefix(a) : a, call.own);
  Source pre{};
  if (prefix_len > 0 && !call.joined) {
    AttnArgs x = with_prefix(a);
    x.alone = 1;
    pre = source(x, call.prefix);
    launch(pre.a, call.prefix, fmt, dim, stream);
    if (const int e = launch_status("kv_attention (prefix)")) return e;
  }
  launch(own.a, call.own, fmt, dim, stream);
  if (const int e = launch_status("kv_attention")) return e;
  const int has = prefix_len > 0 && !call.joined;
  if (by_shares) {
    const dim3 grid(static_cast<uint32_t>(call.own.wgs), static_cast<uint32_t>(call.own.rows / 16));
    if (dim == 128) hipLaunchKernelGGL((join_shares_kernel<128>), grid, dim3(256), 0, stream, own);
    else hipLaunchKernelGGL((join_shares_kernel<64>), grid, dim3(256), 0, stream, own);
    return launch_status("kv_attention (join)");
  }
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(waves)), dim3(wpr == 16 ? 1024 : 256), 0, stream, own, pre, has);
  };
  if (dim == 128) wpr == 16 ? go(join_rows_kernel<128, 16>) : wpr == 4 ? go(join_rows_kernel<128, 4>) : go(join_rows_kernel<128, 1>);
  else wpr == 16 ? go(join_rows_kernel<64, 16>) : wpr == 4 ? go(join_rows_kernel<64, 4>) : go(join_rows_kernel<64, 1>);
  return launch_status("kv_attention (join)");
}
