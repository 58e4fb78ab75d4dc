// Attention of few query rows over the 4-bit paged cache: kv_token.hip's way through the work, for codes and scales of kv_four.hpp.
//
// Bound by the cache's bytes: 2 (dim / 2 + dim / 32) per K/V head and position. Measured: 64 sequences of up to 16,381 keys x 8 K/V heads
// of 128 (0.38 GB) in 77 us, 4.9 TB/s (a large copy moves 5.1, reading alone 5.8), the vector units 47 % busy, the matrix units 17 %.
//
// A wave takes 32 keys at a time, for 16 query rows of the K/V head or 32 (4 sequences x 65,536 keys, 32 rows: 76 us, in two turns of
// 16 92), straight from memory to registers:
//   S^T = K Q^T (16x16x32 bf16): lane l holds key l % 16 of each 16, and of it at dim 128 one group of 32 channels (16 bytes), at 64
//   half of one: its group's power of two goes into the conversion. The channel order this gives each MFMA step is given to Q as well.
//   O^T = V^T P^T: the keys are the 8 whose probabilities a lane now has, dim / 16 channels each, all of one group; pairs of channels
//   are converted with the key's scale, then pairs of keys put together by permutes.
// Probabilities are taken in two bf16 terms, 2^-16 relative at most: the matrix units have the time (with one term the same 84 us).
//
// What mattered (the first size, whole call): a tile's page looked up once and its loads from buffer bases without vector arithmetic, the
// loads of the next tile unconditional (a load that is only sometimes there is waited for at once), 12 waves to a CU in workgroups of 4
// (84 us; 8 waves with two tiles' registers each 86; 12 waves in workgroups of 6, of which only one fits a CU, 112 to 121; 16 waves of
// 128 registers, which spill, 108).
#include "kv_four.hpp"

namespace rh3 {
namespace kv {
namespace {

constexpr int WAVES = 4, NT = WAVES * 64;

template <int D>
struct Tile {
  uint32_t k[2][D / 32];      // of key l % 16 of each half
  uint32_t ks[2];             // its scale byte
  uint2 v[2][D / 64];         // 16 codes of one of keys 4 (l / 16) + 0 .. 3, at 128 of one of the first two and of the others (values())
  uint32_t vs[2][D / 32];     // scale bytes of 4 keys
};

// The page of a 32-key tile, -1 where absent; with pages of 16 (SMALL) the two of its 16-key halves
template <bool SMALL>
struct Pages {
  int p[SMALL ? 2 : 1];
  __device__ __forceinline__ int of(int half) const { return p[SMALL ? half : 0]; }
};
template <bool SMALL>
__device__ __forceinline__ Pages<SMALL> pages_of(const AttnArgs& a, const int32_t* row, int width, int tile) {
  Pages<SMALL> r;
#pragma unroll
  for (int h = 0; h < (SMALL ? 2 : 1); ++h) {
    const int i = min((tile * TOKEN_KEYS + 16 * h) >> a.c.log2page, width - 1);
    const int p = scalar_load(row + i);
    r.p[h] = p >= 0 && p < a.c.pages ? p : -1;
  }
  return r;
}

// A tile's loads: scalar bases (a buffer's, which takes them without vector arithmetic), and offsets that the lane keeps. head: the
// K/V head's codes and scales of keys and of values in page 0.
template <int D, bool SMALL>
struct Bases {
  __amdgpu_buffer_rsrc_t codes[SMALL ? 2 : 1], scales[SMALL ? 2 : 1];
};
template <int D, bool SMALL>
__device__ __forceinline__ Bases<D, SMALL> bases_of(const AttnArgs& a, const uint8_t* codes, const uint8_t* scales, int tile, const Pages<SMALL>& pg) {
  auto buffer = [](const uint8_t* p) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, 0x7fffffff, BUF_RSRC_WORD3); };
  const int off = (tile * TOKEN_KEYS) & ((1 << a.c.log2page) - 1);
  Bases<D, SMALL> b;
#pragma unroll
  for (int h = 0; h < (SMALL ? 2 : 1); ++h) {
    const int64_t p = max(pg.p[h], 0);
    b.codes[h] = buffer(codes + (p * a.c.page_stride + off * (D / 2)));
    b.scales[h] = buffer(scales + (p * a.c.spage_stride + off * (D / 32)));
  }
  return b;
}
template <int D, bool SMALL>
__device__ __forceinline__ void load_keys(const AttnArgs& a, const uint8_t* const (&head)[4], int tile, const Pages<SMALL>& pg, Tile<D>& t) {
  const uint32_t lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const Bases<D, SMALL> b = bases_of<D, SMALL>(a, head[0], head[1], tile, pg);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int w = SMALL ? h : 0, key = SMALL ? 0 : 16 * h;
    const uint32_t codes = l16 * (D / 2) + g * (D / 8) + key * (D / 2);
    if constexpr (D == 128) {
      const u32x4_t x = __builtin_amdgcn_raw_buffer_load_b128(b.codes[w], codes, 0, 0);
      t.k[h][0] = x[0]; t.k[h][1] = x[1]; t.k[h][2] = x[2]; t.k[h][3] = x[3];
    } else {
      const u32x2_t x = __builtin_amdgcn_raw_buffer_load_b64(b.codes[w], codes, 0, 0);
      t.k[h][0] = x[0]; t.k[h][1] = x[1];
    }
    t.ks[h] = __builtin_amdgcn_raw_buffer_load_b8(b.scales[w], l16 * (D / 32) + (g * D / 4) / GROUP4 + key * (D / 32), 0, 0);
  }
}
template <int D, bool SMALL>
__device__ __forceinline__ void load_values(const AttnArgs& a, const uint8_t* const (&head)[4], int tile, const Pages<SMALL>& pg, Tile<D>& t) {
  const uint32_t lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const Bases<D, SMALL> b = bases_of<D, SMALL>(a, head[2], head[3], tile, pg);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int w = SMALL ? h : 0, key = SMALL ? 0 : 16 * h;
    const uint32_t scales = 4 * g * (D / 32) + key * (D / 32);
    if constexpr (D == 128) {
      const u32x4_t x = __builtin_amdgcn_raw_buffer_load_b128(b.scales[w], scales, 0, 0);
      t.vs[h][0] = x[0]; t.vs[h][1] = x[1]; t.vs[h][2] = x[2]; t.vs[h][3] = x[3];
    } else {
      const u32x2_t x = __builtin_amdgcn_raw_buffer_load_b64(b.scales[w], scales, 0, 0);
      t.vs[h][0] = x[0]; t.vs[h][1] = x[1];
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const u32x2_t x = __builtin_amdgcn_raw_buffer_load_b64(b.codes[w], 128 * (D / 64) * g + 8 * l16 + (128 * i + key * (D / 2)), 0, 0);
      t.v[h][i] = make_uint2(x[0], x[1]);
    }
  }
}

// The loads of values are whole lines of 128 bytes to 16 lanes: a load brings a lane 16 channels of one key, and lanes 8 apart (at 64
// also 4 apart) exchange what the other one's channels are. A lane then has, of each of its 4 keys, the dim / 16 channels that begin
// at channel_of(l % 16).
template <int D>
RH3_HD int channel_of(int m) { return D == 128 ? 16 * (m & 7) + 8 * (m >> 3) : 16 * (m & 3) + 8 * (m >> 3) + 4 * ((m >> 2) & 1); }
template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
// codes of 4 keys: 128: a word each; 64: a half word each, in two words
template <int D>
__device__ __forceinline__ void exchange(const uint2 (&v)[D / 64], uint32_t (&w)[D / 32]) {
  const uint32_t lane = threadIdx.x & 63;
  const bool up = lane & 8;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const uint32_t got = moved<0x128>(up ? v[i].x : v[i].y);   // row_ror:8: from lane ^ 8
    w[2 * i] = up ? got : v[i].x;
    w[2 * i + 1] = up ? v[i].y : got;
  }
  if constexpr (D == 64) {
    const uint32_t sel = lane & 4 ? 0x03020706u : 0x05040100u;
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = __builtin_amdgcn_perm(moved<0x1B>(moved<0x141>(w[i])), w[i], sel);   // from lane ^ 4
  }
}

// one wave's running state for MT x 16 query rows (row l % 16 of each)
template <int D, int MT>
struct State {
  f4_t o[MT][D / 16];   // o[m][i][r]: channel channel_of(4 (l / 16) + r) + i
  float ref[MT], sum[MT];
};

// One tile. FINE: fp16 queries, in two terms. The wave's next tile (nt, pages pn) is loaded into the same registers, its keys as soon
// as these are used, its values as soon as theirs are. (The last turn loads its own tile again: loads that are only sometimes there
// would be waited for at once.)
template <int D, int MT, bool FINE, bool SMALL>
__device__ __forceinline__ void compute(const AttnArgs& a, Tile<D>& t, int tile, const Pages<SMALL>& pg, const b8_t (&q)[MT][D / 32],
                                        const b8_t (&ql)[MT][D / 32], const int (&lim)[MT], int low, int len, const uint8_t* const (&head)[4], int nt,
                                        const Pages<SMALL>& pn, State<D, MT>& st) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int kb = tile * TOKEN_KEYS;
  // low: keys that every row sees
  const bool edge = kb + TOKEN_KEYS > low || pg.of(0) < 0 || pg.of(1) < 0;
  f4_t acc[MT][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m][h] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const float s = __uint_as_float(t.ks[h] << 23);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const b8_t k = values4(t.k[h][c], s);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        acc[m][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[m][c], acc[m][h], 0, 0, 0);
        if constexpr (FINE) acc[m][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, ql[m][c], acc[m][h], 0, 0, 0);
      }
    }
  }
  load_keys<D, SMALL>(a, head, nt, pn, t);
  auto key = [&](int j) { return kb + 16 * (j >> 2) + 4 * g + (j & 3); };
  auto hidden = [&](int j, int end) { return key(j) >= end || pg.of(j >> 2) < 0; };
  b8_t p[MT], rest[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    // scores less the reference, which is finite: before a row's first key it is the lowest number
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = fmaf(acc[m][j >> 2][j & 3], a.scale_log2, -st.ref[m]);
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = hidden(j, lim[m]) ? -INFINITY : y[j];
    }
    float top = st.sum[m] + (STALE - SUM_MOST);   // over STALE where the sum is over SUM_MOST
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, y[j]);
    if (__builtin_amdgcn_ballot_w64(top > STALE)) {
      float n = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = edge && hidden(j, lim[m]) ? -INFINITY : acc[m][j >> 2][j & 3] * a.scale_log2;
        n = fmaxf(n, y[j]);
      }
      n = across_max<true>(n);
      const float to = next_reference(st.ref[m], n, across_sum<true>(st.sum[m]));
      const float f = __builtin_amdgcn_exp2f(st.ref[m] - to);
      st.ref[m] = to;
      st.sum[m] *= f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) st.o[m][i] *= f;
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] -= to;
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float e0 = __builtin_amdgcn_exp2f(y[j]), e1 = __builtin_amdgcn_exp2f(y[j + 1]);
      st.sum[m] += e0 + e1;
      hi[j / 2] = pack_bf2(e0, e1);
      lo[j / 2] = pack_bf2(e0 - __uint_as_float(hi[j / 2] << 16), e1 - __uint_as_float(hi[j / 2] & 0xffff0000u));
    }
    p[m] = bf16x8(hi[0], hi[1], hi[2], hi[3]);
    rest[m] = bf16x8(lo[0], lo[1], lo[2], lo[3]);
  }

  // the scale byte of the lane's group to where a float's exponent is; what lies beside it is not looked at
  const int group = channel_of<D>(l16) / GROUP4;
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t w = D == 128 ? t.vs[j >> 2][j & 3] : t.vs[j >> 2][(j & 3) >> 1];
    const int byte = D == 128 ? group : 2 * (j & 1) + group;
    s[j] = __uint_as_float(__builtin_amdgcn_alignbit(w, w, (8 * byte + 9) & 31));
  }
  uint32_t v[2][D / 32];
#pragma unroll
  for (int h = 0; h < 2; ++h) exchange<D>(t.v[h], v[h]);
  if (edge) {   // what lies behind the sequence or in an absent page may be anything
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (hidden(j, len)) {
        if constexpr (D == 128) v[j >> 2][j & 3] = 0;
        else v[j >> 2][(j & 3) >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
        s[j] = 1.0f;
      }
    }
  }
  auto channels = [&](auto C) __attribute__((always_inline)) {   // 2 c and 2 c + 1
    constexpr int c = decltype(C)::value;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (D == 128) w[j] = pair4<c>(v[j >> 2][j & 3], s[j]);
      else w[j] = j & 1 ? pair4<(c + 2) & 3>(v[j >> 2][(j & 3) >> 1], s[j]) : pair4<c>(v[j >> 2][(j & 3) >> 1], s[j]);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t sel = e ? 0x07060302u : 0x05040100u;
      const b8_t x = bf16x8(__builtin_amdgcn_perm(w[1], w[0], sel), __builtin_amdgcn_perm(w[3], w[2], sel),
                            __builtin_amdgcn_perm(w[5], w[4], sel), __builtin_amdgcn_perm(w[7], w[6], sel));
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        st.o[m][2 * c + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, p[m], st.o[m][2 * c + e], 0, 0, 0);
        st.o[m][2 * c + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, rest[m], st.o[m][2 * c + e], 0, 0, 0);
      }
    }
  };
  load_values<D, SMALL>(a, head, nt, pn, t);
  channels(std::integral_constant<int, 0>());
  channels(std::integral_constant<int, 1>());
  if constexpr (D == 128) {
    channels(std::integral_constant<int, 2>());
    channels(std::integral_constant<int, 3>());
  }
}

// The block of 64 sequences at hand (kv_attn.hpp), kept in LDS: in registers it would take what the loop's loads need
struct SharedList {
  int first[64], n[64], len[64], pos[64], row_tiles[64], span[64];
  int64_t units[64], items[64];
};
struct Listed {
  int at;
  int64_t base, items_base, end;
  __device__ __forceinline__ void put(const Block& b, SharedList& s) {
    const int lane = threadIdx.x & 63;
    at = b.at;
    base = scalar(b.base);
    items_base = scalar(b.items_base);
    end = b.end();
    __syncthreads();
    if (threadIdx.x < 64) {
      s.first[lane] = b.seq.first;
      s.n[lane] = b.seq.n;
      s.len[lane] = b.seq.len;
      s.pos[lane] = b.seq.pos;
      s.row_tiles[lane] = b.row_tiles;
      s.span[lane] = b.span;
      s.units[lane] = b.units;
      s.items[lane] = b.items;
    }
    __syncthreads();
  }
  __device__ __forceinline__ Work begin(const AttnArgs& a, const Tiling& g, SharedList& s) {
    Block b;
    const Work w = dealt(load_blocks(a, g, b), a.wgs, g);
    put(b, s);
    return w;
  }
  __device__ __forceinline__ void next(const AttnArgs& a, const Tiling& g, SharedList& s) {
    Block b;
    load_block(a, g, at + 64, end, items_base + scalar(s.items[63]), b);
    put(b, s);
  }
  __device__ __forceinline__ int lane_of(const SharedList& s, int64_t u) const {
    return __builtin_ctzll(__builtin_amdgcn_ballot_w64(base + s.units[threadIdx.x & 63] > u));
  }
  __device__ __forceinline__ SeqItems sequence(const SharedList& s, int l) const {
    SeqItems r;
    r.seq = Seq{scalar(s.first[l]), scalar(s.n[l]), scalar(s.len[l]), scalar(s.pos[l])};
    r.row_tiles = scalar(s.row_tiles[l]);
    r.span = scalar(s.span[l]);
    r.before = base + (l ? scalar(s.units[l - 1]) : 0);
    r.items_before = items_base + (l ? scalar(s.items[l - 1]) : 0);
    return r;
  }
};

template <int D, int MT, bool FINE, bool SMALL>
__global__ void __launch_bounds__(NT, MT == 1 ? 3 : 2) token_kernel(AttnArgs a) {
  constexpr int R = 16 * MT, PAD = D + 4;
  const Tiling TILING = tiling(false, R);
  __shared__ float so[WAVES][R][PAD];
  __shared__ float sm[WAVES][R], sl[WAVES][R];
  __shared__ SharedList shared_list;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Listed list;
  const Work work = list.begin(a, TILING, shared_list);
  const int wg = blockIdx.x;
  if (wg >= work.wgs) return;
  int64_t u = scalar(share_begin(work, wg));
  const int64_t end = scalar(share_begin(work, wg + 1));

  while (u < end) {
    while (u >= list.end) {
      if (list.at + 64 >= sequences(a)) return;
      list.next(a, TILING, shared_list);
    }
    const int l = list.lane_of(shared_list, u);
    const SeqItems sw = list.sequence(shared_list, l);
    const Seq sq = sw.seq;
    const int64_t local = u - sw.before;
    const int item = scalar(static_cast<int>(quotient(local, sw.span)));
    const int u0 = static_cast<int>(local - static_cast<int64_t>(item) * sw.span);
    const int u1 = static_cast<int>(end - u < sw.span - u0 ? u0 + (end - u) : sw.span);
    u += u1 - u0;
    const int t0 = max(u0 - TILING.extra, 0), t1 = u1 - TILING.extra;
    if (t1 <= 0) continue;
    const bool pre = a.prefix && list.at + l == 0, causal = a.causal && !pre;
    const int32_t* row = pre ? a.prefix : a.s.table + (list.at + l - (a.prefix != nullptr)) * a.s.table_stride;
    const int width = pre ? a.prefix_width : a.s.width;
    const int kvh = scalar(item / sw.row_tiles), rt = item - kvh * sw.row_tiles;
    const int rows = sq.n * a.group;

    // query rows: lane l holds row l % 16, channels (dim / 4) (l / 16) + 8 c + 0 .. 7 in step c
    int t = t0 + wave;
    Pages<SMALL> pg = pages_of<SMALL>(a, row, width, t), pn = pages_of<SMALL>(a, row, width, t + WAVES);
    uint4 raw[MT][D / 32];
    int lim[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int mine = rt * R + 16 * m + l16, rr = mine < rows ? mine : 0;
      const int tok = rr / a.group, hd = kvh * a.group + rr - tok * a.group;
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + (sq.first + tok) * a.q_st + hd * a.q_sh + (D / 4) * g;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) raw[m][c] = *reinterpret_cast<const uint4*>(src + 8 * c);
      lim[m] = causal ? min(sq.len, sq.pos + tok + 1) : sq.len;
    }
    // the first keys and values are on their way while the query rows come in
    Tile<D> tile;
    const int64_t codes = kvh * a.c.head_stride, scales = kvh * a.c.shead_stride;
    const uint8_t* const head[4] = {a.c.k + codes, reinterpret_cast<const uint8_t*>(a.c.ks) + scales, a.c.v + codes,
                                    reinterpret_cast<const uint8_t*>(a.c.vs) + scales};
    if (t < t1) {
      load_keys<D, SMALL>(a, head, t, pg, tile);
      load_values<D, SMALL>(a, head, t, pg, tile);
    }
    b8_t q[MT][D / 32], ql[MT][D / 32];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) query8<FINE>(rt * R + 16 * m + l16 < rows ? raw[m][c] : make_uint4(0, 0, 0, 0), q[m][c], ql[m][c]);
    const int low = causal ? min(sq.len, sq.pos + scalar((rt * R) / a.group) + 1) : sq.len;

    State<D, MT> st;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      st.ref[m] = NO_REF;
      st.sum[m] = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) st.o[m][i] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    while (t < t1) {
      const Pages<SMALL> p2 = pages_of<SMALL>(a, row, width, t + 2 * WAVES);
      const bool more = t + WAVES < t1;
      compute<D, MT, FINE, SMALL>(a, tile, t, pg, q, ql, lim, low, sq.len, head, more ? t + WAVES : t, more ? pn : pg, st);
      pg = pn;
      pn = p2;
      t += WAVES;
    }
    // join the waves
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float sum = across_sum<true>(st.sum[m]);
      if (g == 0) {
        sm[wave][16 * m + l16] = st.ref[m];
        sl[wave][16 * m + l16] = sum;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < D / 16; i += 4)
          *reinterpret_cast<float4*>(&so[wave][16 * m + l16][channel_of<D>(4 * g + r) + i]) =
              make_float4(st.o[m][i][r], st.o[m][i + 1][r], st.o[m][i + 2][r], st.o[m][i + 3][r]);
    }
    __syncthreads();
    const bool whole = t0 == 0 && u1 == sw.span;
    constexpr int TPR = NT / R, EPT = D / TPR;   // threads to a row, channels to a thread
    const int rl = threadIdx.x / TPR, d0 = (threadIdx.x % TPR) * EPT;
    const int rw = rt * R + rl;
    if (rw < rows) {
      float top = sm[0][rl];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) top = fmaxf(top, sm[w][rl]);
      float sum = 0.0f, o[EPT] = {};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = __builtin_amdgcn_exp2f(sm[w][rl] - top);
        sum += f * sl[w][rl];
#pragma unroll
        for (int e = 0; e < EPT; ++e) o[e] += f * so[w][rl][d0 + e];
      }
      if (whole && !a.keep) {
        const int tok = rw / a.group, hd = kvh * a.group + rw - tok * a.group;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        uint16_t* dst = static_cast<uint16_t*>(a.out) + (sq.first + tok) * a.o_st + hd * a.o_sh + d0;
        uint32_t w[EPT / 2];
#pragma unroll
        for (int e = 0; e < EPT; e += 2) w[e / 2] = pack_out(a, o[e] * inv, o[e + 1] * inv);
#pragma unroll
        for (int e = 0; e < EPT / 2; e += 2) *reinterpret_cast<uint2*>(dst + 2 * e) = make_uint2(w[e], w[e + 1]);
        if (a.lse && d0 == 0)
          a.lse[static_cast<int64_t>(sq.first + tok) * a.c.heads * a.group + hd] =
              sum == 0.0f ? -INFINITY : (__builtin_amdgcn_logf(sum) + top) * 0.6931471805599453f;
      } else if (!whole || sw.items_before + item < a.items) {   // (a cu that falls can count rows more than once)
        // slots: two to a workgroup (the item that it goes on with, the one that it begins), then one to an item that it completes
        const int64_t slot = whole ? 2 * static_cast<int64_t>(a.wgs) + sw.items_before + item : 2 * static_cast<int64_t>(wg) + (t0 == 0);
        float* po = a.part_o + (slot * R + rl) * D + d0;
#pragma unroll
        for (int e = 0; e < EPT; e += 4)
          *reinterpret_cast<float4*>(po + e) = make_float4(o[e] * (PART * PART_UP), o[e + 1] * (PART * PART_UP), o[e + 2] * (PART * PART_UP), o[e + 3] * (PART * PART_UP));
        if (d0 == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * R + rl) * 2) = make_float2(sum == 0.0f ? -INFINITY : sum == sum ? top - OVER : 0.0f, sum * PART_UP);
      }
    }
    if (u < end) __syncthreads();
  }
}

}  // namespace

void launch_token4(const AttnArgs& a, int dim, int rows, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(a.wgs)), dim3(NT), 0, st, a); };
  auto by_page = [&](auto small, auto large) { a.c.log2page == 4 ? go(small) : go(large); };
  auto by_type = [&](auto D, auto MT) {
    constexpr int d = decltype(D)::value, m = decltype(MT)::value;
    if (a.fp16) by_page(token_kernel<d, m, true, true>, token_kernel<d, m, true, false>);
    else by_page(token_kernel<d, m, false, true>, token_kernel<d, m, false, false>);
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  if (dim == 128) rows == 16 ? by_type(std::integral_constant<int, 128>(), One()) : by_type(std::integral_constant<int, 128>(), Two());
  else rows == 16 ? by_type(std::integral_constant<int, 64>(), One()) : by_type(std::integral_constant<int, 64>(), Two());
}

}  // namespace kv
}  // namespace rh3
