// Attention of few query rows over the 4-bit paged cache: kv_token.hip's way through the work, for codes and scales of kv_four.hpp.
//
// Bound by the cache's bytes: 2 (dim / 2 + dim / 32) per K/V head and position.
//
// A wave takes 32 keys at a time, for 16 query rows of the K/V head, straight from memory to registers:
//   S^T = K Q^T (16x16x32 bf16): lane l holds key l % 16 of each 16, and of it at dim 128 one group of 32 channels (16 bytes), at 64
//   half of one: its group's power of two goes into the conversion. The channel order this gives each MFMA step is given to Q as well.
//   O^T = V^T P^T: the keys are the 8 whose probabilities a lane now has, dim / 16 channels each, all of one group; pairs of channels
//   are converted with the key's scale, then pairs of keys put together by permutes.
// Probabilities are taken in two bf16 terms, 2^-16 relative at most: the matrix units have the time.
#include "kv_four.hpp"

namespace rh3 {
namespace kv {
namespace {

constexpr int WAVES = 8, NT = WAVES * 64, R = 16;

template <int D>
struct Tile {
  uint32_t k[2][D / 32];      // of key l % 16 of each half
  uint32_t ks[2];             // its scale byte
  uint32_t v[8];              // dim / 16 codes of keys 4 (l / 16) + 0 .. 3 of each half
  uint32_t vs[2][D / 32];     // scale bytes of 4 keys
};

// the two pages of a 32-key tile (two 16-key halves), -1 where absent
struct Pages {
  int p[2];
};
__device__ __forceinline__ Pages pages_of(const AttnArgs& a, const int32_t* row, int width, int tile) {
  Pages r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = min((tile * TOKEN_KEYS + 16 * h) >> a.c.log2page, width - 1);
    const int p = scalar_load(row + i);
    r.p[h] = p >= 0 && p < a.c.pages ? p : -1;
  }
  return r;
}

template <int D>
__device__ __forceinline__ void load_keys(const AttnArgs& a, int kvh, int tile, const Pages& pg, Tile<D>& t) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const uint8_t* scales = reinterpret_cast<const uint8_t*>(a.c.ks);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t p = max(pg.p[h], 0);
    const int off = (tile * TOKEN_KEYS + 16 * h) & ((1 << a.c.log2page) - 1);
    const uint8_t* kb = a.c.k + p * a.c.page_stride + kvh * a.c.head_stride + off * (D / 2) + l16 * (D / 2) + g * (D / 8);
    if constexpr (D == 128) {
      const uint4 w = *reinterpret_cast<const uint4*>(kb);
      t.k[h][0] = w.x; t.k[h][1] = w.y; t.k[h][2] = w.z; t.k[h][3] = w.w;
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(kb);
      t.k[h][0] = w.x; t.k[h][1] = w.y;
    }
    t.ks[h] = scales[p * a.c.spage_stride + kvh * a.c.shead_stride + off * (D / 32) + l16 * (D / 32) + (g * D / 4) / GROUP4];
  }
}
template <int D>
__device__ __forceinline__ void load_values(const AttnArgs& a, int kvh, int tile, const Pages& pg, Tile<D>& t) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const uint8_t* scales = reinterpret_cast<const uint8_t*>(a.c.vs);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t p = max(pg.p[h], 0);
    const int off = (tile * TOKEN_KEYS + 16 * h) & ((1 << a.c.log2page) - 1);
    const uint8_t* vb = a.c.v + p * a.c.page_stride + kvh * a.c.head_stride + off * (D / 2) + 4 * g * (D / 2) + l16 * (D / 32);
    const uint8_t* sb = scales + p * a.c.spage_stride + kvh * a.c.shead_stride + off * (D / 32) + 4 * g * (D / 32);
    if constexpr (D == 128) {
      const uint4 s = *reinterpret_cast<const uint4*>(sb);
      t.vs[h][0] = s.x; t.vs[h][1] = s.y; t.vs[h][2] = s.z; t.vs[h][3] = s.w;
#pragma unroll
      for (int j = 0; j < 4; ++j) t.v[4 * h + j] = *reinterpret_cast<const uint32_t*>(vb + j * (D / 2));
    } else {
      const uint2 s = *reinterpret_cast<const uint2*>(sb);
      t.vs[h][0] = s.x; t.vs[h][1] = s.y;
#pragma unroll
      for (int j = 0; j < 4; ++j) t.v[4 * h + j] = *reinterpret_cast<const uint16_t*>(vb + j * (D / 2));
    }
  }
}

// one wave's running state for 16 query rows (row l % 16)
template <int D>
struct State {
  f4_t o[D / 16];   // o[i][r]: channel (D / 16) (4 (l / 16) + r) + i
  float ref, sum;
};

// One tile. FINE: fp16 queries, in two terms. MORE: the wave's next tile (pages `pn`) is loaded into the same registers, its keys as
// soon as these are used, its values at the end.
template <int D, bool FINE, bool MORE>
__device__ __forceinline__ void compute(const AttnArgs& a, Tile<D>& t, int kvh, int tile, const Pages& pg, const Pages& pn,
                                        const b8_t (&q)[D / 32], const b8_t (&ql)[D / 32], int lim, int low, int len, State<D>& st) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int kb = tile * TOKEN_KEYS;
  // low: keys that every row sees
  const bool edge = kb + TOKEN_KEYS > low || pg.p[0] < 0 || pg.p[1] < 0;
  f4_t acc[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    acc[h] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const float s = __uint_as_float(t.ks[h] << 23);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const b8_t k = values4(t.k[h][c], s);
      acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[c], acc[h], 0, 0, 0);
      if constexpr (FINE) acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, ql[c], acc[h], 0, 0, 0);
    }
  }
  if constexpr (MORE) load_keys<D>(a, kvh, tile + WAVES, pn, t);
  auto key = [&](int j) { return kb + 16 * (j >> 2) + 4 * g + (j & 3); };
  float x[8], top = -INFINITY;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = acc[j >> 2][j & 3] * a.scale_log2;
  if (edge) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = key(j) >= lim || pg.p[j >> 2] < 0 ? -INFINITY : x[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);
  if (__builtin_amdgcn_ballot_w64(top - st.ref > STALE)) {
    const float n = across_max<true>(top);
    if (n - st.ref > STALE) {
      const float to = reference_over(n);
      const float f = __builtin_amdgcn_exp2f(st.ref - to);   // from no keys yet: 2^-inf = 0
      st.ref = to;
      st.sum *= f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) st.o[i] *= f;
    }
  }
  // a row that has seen no key yet has only -inf here: any finite reference gives it zeros
  const float ref = st.ref == -INFINITY ? 0.0f : st.ref;
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float e0 = __builtin_amdgcn_exp2f(x[j] - ref), e1 = __builtin_amdgcn_exp2f(x[j + 1] - ref);
    st.sum += e0 + e1;
    hi[j / 2] = pack_bf2(e0, e1);
    lo[j / 2] = pack_bf2(e0 - __uint_as_float(hi[j / 2] << 16), e1 - __uint_as_float(hi[j / 2] & 0xffff0000u));
  }
  const b8_t p = bf16x8(hi[0], hi[1], hi[2], hi[3]), rest = bf16x8(lo[0], lo[1], lo[2], lo[3]);

  // the scale byte of the lane's group to where a float's exponent is; what lies beside it is not looked at
  const int group = (l16 * (D / 16)) / GROUP4;
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t w = D == 128 ? t.vs[j >> 2][j & 3] : t.vs[j >> 2][(j & 3) >> 1];
    const int byte = D == 128 ? group : 2 * (j & 1) + group;
    s[j] = __uint_as_float(__builtin_amdgcn_alignbit(w, w, (8 * byte + 9) & 31));
  }
  if (edge) {   // what lies behind the sequence or in an absent page may be anything
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (key(j) >= len || pg.p[j >> 2] < 0) {
        t.v[j] = 0;
        s[j] = 1.0f;
      }
    }
  }
  auto channels = [&](auto C) __attribute__((always_inline)) {   // 2 c and 2 c + 1
    constexpr int c = decltype(C)::value;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = pair4<c>(t.v[j], s[j]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t sel = e ? 0x07060302u : 0x05040100u;
      const b8_t v = bf16x8(__builtin_amdgcn_perm(w[1], w[0], sel), __builtin_amdgcn_perm(w[3], w[2], sel),
                            __builtin_amdgcn_perm(w[5], w[4], sel), __builtin_amdgcn_perm(w[7], w[6], sel));
      st.o[2 * c + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p, st.o[2 * c + e], 0, 0, 0);
      st.o[2 * c + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, rest, st.o[2 * c + e], 0, 0, 0);
    }
  };
  channels(std::integral_constant<int, 0>());
  channels(std::integral_constant<int, 1>());
  if constexpr (D == 128) {
    channels(std::integral_constant<int, 2>());
    channels(std::integral_constant<int, 3>());
  }
  if constexpr (MORE) load_values<D>(a, kvh, tile + WAVES, pn, t);
}

template <int D, bool FINE>
__global__ void __launch_bounds__(NT, 4) token_kernel(AttnArgs a) {
  constexpr int PAD = D + 4;
  const Tiling TILING = tiling(false, R);
  __shared__ float so[WAVES][R][PAD];
  __shared__ float sm[WAVES][R], sl[WAVES][R];
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Block blk;
  const Work work = dealt(load_blocks(a, TILING, blk), a.wgs, TILING);
  const int wg = blockIdx.x;
  if (wg >= work.wgs) return;
  int64_t u = scalar(share_begin(work, wg));
  const int64_t end = scalar(share_begin(work, wg + 1));

  while (u < end) {
    while (u >= blk.end()) {
      if (blk.at + 64 >= sequences(a)) return;
      next_block(a, TILING, blk);
    }
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(blk.base + blk.units > u));
    const SeqItems sw = seq_in(a, blk, l);
    const Seq sq = sw.seq;
    const int64_t local = u - sw.before;
    const int item = scalar(static_cast<int>(quotient(local, sw.span)));
    const int u0 = static_cast<int>(local - static_cast<int64_t>(item) * sw.span);
    const int u1 = static_cast<int>(end - u < sw.span - u0 ? u0 + (end - u) : sw.span);
    u += u1 - u0;
    const int t0 = max(u0 - TILING.extra, 0), t1 = u1 - TILING.extra;
    if (t1 <= 0) continue;
    const bool pre = a.prefix && blk.at + l == 0, causal = a.causal && !pre;
    const int32_t* row = pre ? a.prefix : a.s.table + (blk.at + l - (a.prefix != nullptr)) * a.s.table_stride;
    const int width = pre ? a.prefix_width : a.s.width;
    const int kvh = scalar(item / sw.row_tiles), rt = item - kvh * sw.row_tiles;
    const int rows = sq.n * a.group;

    // query rows: lane l holds row l % 16, channels (dim / 4) (l / 16) + 8 c + 0 .. 7 in step c
    int t = t0 + wave;
    Pages pg = pages_of(a, row, width, t), pn = pages_of(a, row, width, t + WAVES);
    const int mine = rt * R + l16, rr = mine < rows ? mine : 0;
    const int tok = rr / a.group, hd = kvh * a.group + rr - tok * a.group;
    uint4 raw[D / 32];
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (sq.first + tok) * a.q_st + hd * a.q_sh + (D / 4) * g;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) raw[c] = *reinterpret_cast<const uint4*>(src + 8 * c);
    const int lim = causal ? min(sq.len, sq.pos + tok + 1) : sq.len;
    // the first keys and values are on their way while the query rows come in
    Tile<D> tile;
    if (t < t1) {
      load_keys<D>(a, kvh, t, pg, tile);
      load_values<D>(a, kvh, t, pg, tile);
    }
    b8_t q[D / 32], ql[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) query8<FINE>(mine < rows ? raw[c] : make_uint4(0, 0, 0, 0), q[c], ql[c]);
    const int low = causal ? min(sq.len, sq.pos + scalar((rt * R) / a.group) + 1) : sq.len;

    State<D> st;
    st.ref = -INFINITY;
    st.sum = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) st.o[i] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (t < t1) {
      for (; t + WAVES < t1; t += WAVES) {
        const Pages p2 = pages_of(a, row, width, t + 2 * WAVES);
        compute<D, FINE, true>(a, tile, kvh, t, pg, pn, q, ql, lim, low, sq.len, st);
        pg = pn;
        pn = p2;
      }
      compute<D, FINE, false>(a, tile, kvh, t, pg, pn, q, ql, lim, low, sq.len, st);
    }
    // join the waves
    const float mysum = across_sum<true>(st.sum);
    if (g == 0) {
      sm[wave][l16] = st.ref;
      sl[wave][l16] = mysum;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < D / 16; i += 4)
        *reinterpret_cast<float4*>(&so[wave][l16][(D / 16) * (4 * g + r) + i]) = make_float4(st.o[i][r], st.o[i + 1][r], st.o[i + 2][r], st.o[i + 3][r]);
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
        // (a wave that has seen nothing but NaN has its sums under no reference)
        const float f = sm[w][rl] == -INFINITY ? (sl[w][rl] == 0.0f ? 0.0f : sl[w][rl]) : __builtin_amdgcn_exp2f(sm[w][rl] - top);
        sum += f * sl[w][rl];
#pragma unroll
        for (int e = 0; e < EPT; ++e) o[e] += f * so[w][rl][d0 + e];
      }
      if (whole && !a.keep) {
        const int tok = rw / a.group, hd = kvh * a.group + rw - tok * a.group;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        uint16_t* dst = static_cast<uint16_t*>(a.out) + (sq.first + tok) * a.o_st + hd * a.o_sh + d0;
        if constexpr (EPT == 4) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack_out(a, o[0] * inv, o[1] * inv), pack_out(a, o[2] * inv, o[3] * inv));
        } else {
          *reinterpret_cast<uint32_t*>(dst) = pack_out(a, o[0] * inv, o[1] * inv);
        }
        if (a.lse && d0 == 0)
          a.lse[static_cast<int64_t>(sq.first + tok) * a.c.heads * a.group + hd] =
              sum == 0.0f ? -INFINITY : (__builtin_amdgcn_logf(sum) + top) * 0.6931471805599453f;
      } else if (!whole || sw.items_before + item < a.items) {   // (a cu that falls can count rows more than once)
        // slots: two to a workgroup (the item that it goes on with, the one that it begins), then one to an item that it completes
        const int64_t slot = whole ? 2 * static_cast<int64_t>(a.wgs) + sw.items_before + item : 2 * static_cast<int64_t>(wg) + (t0 == 0);
        float* po = a.part_o + (slot * R + rl) * D + d0;
#pragma unroll
        for (int e = 0; e < EPT; ++e) po[e] = o[e] * (PART * PART_UP);
        if (d0 == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * R + rl) * 2) = make_float2(sum == sum ? top - OVER : 0.0f, sum * PART_UP);
      }
    }
    if (u < end) __syncthreads();
  }
}

}  // namespace

void launch_token4(const AttnArgs& a, int dim, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(a.wgs)), dim3(NT), 0, st, a); };
  if (dim == 128) a.fp16 ? go(token_kernel<128, true>) : go(token_kernel<128, false>);
  else a.fp16 ? go(token_kernel<64, true>) : go(token_kernel<64, false>);
}

}  // namespace kv
}  // namespace rh3
