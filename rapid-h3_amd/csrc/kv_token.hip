// Attention of few query rows over the paged cache: single tokens of a batch, or a few tokens each.
//
// Bound by the cache's bytes: 2 (dim + 4) per K/V head and position. Measured: 64 sequences of up to 8,190 keys x 8 K/V heads of
// 128 (0.37 GB) in 74 us, 5.0 TB/s; 4 of 131,071 keys (1.1 GB) in 190 us, 5.8 TB/s; a large copy moves 4.8, a fill 6.8.
//
// A wave takes 32 keys at a time, for 16 query rows of the K/V head (32 at dim 64: at 128 their accumulators leave no registers for
// the loads, and 2 x 16 rows, the second time mostly from L2, took 164 us where 32 took 230: 8 sequences of 4 tokens x 56 / 8 heads
// x 32,768 keys), straight from memory to registers, and its matrix instructions' operand order is made to fit what a wide load
// brings, so nothing passes through LDS:
//   S^T = K Q^T: lane l holds key l % 16, two (one) 16-byte pieces of its row; the channel order this gives each MFMA step is
//   given to Q as well. The result has the query row in l % 16 and keys 4 (l / 16) + 0 .. 3 in the registers of both 16-key tiles.
//   O^T = V^T P^T: those keys are the ones whose P a lane now has; it loads the same keys' values, dim / 16 channels each, and
//   turns bytes into channel-major f16 by permutes as it converts.
// Each tile's registers take the next one as they are used up. A workgroup's 4 waves take a share's tiles in turn and join through
// LDS at the end of an item; items that more than one workgroup has worked on are left as parts.
#include "kv_attn.hpp"

namespace rh3 {
namespace kv {
namespace {

constexpr int NT = 256, WAVES = 4;

template <int D>
struct Tile {
  uint4 k[2][D / 64];
  float4 ks[2];
  uint32_t v[8][D / 64];
  float4 vs[2];
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
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t p = max(pg.p[h], 0);
    const int off = (tile * TOKEN_KEYS + 16 * h) & ((1 << a.c.log2page) - 1);
    const uint8_t* kb = a.c.k + p * a.c.page_stride + kvh * a.c.head_stride + off * D;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) t.k[h][c] = *reinterpret_cast<const uint4*>(kb + (l16 * D + 64 * c + 16 * g));
    t.ks[h] = *reinterpret_cast<const float4*>(a.c.ks + p * a.c.spage_stride + kvh * a.c.shead_stride + off + 4 * g);
  }
}
template <int D>
__device__ __forceinline__ void load_values(const AttnArgs& a, int kvh, int tile, const Pages& pg, Tile<D>& t) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t p = max(pg.p[h], 0);
    const int off = (tile * TOKEN_KEYS + 16 * h) & ((1 << a.c.log2page) - 1);
    const uint8_t* vb = a.c.v + p * a.c.page_stride + kvh * a.c.head_stride + off * D;
    t.vs[h] = *reinterpret_cast<const float4*>(a.c.vs + p * a.c.spage_stride + kvh * a.c.shead_stride + off + 4 * g);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint8_t* vr = vb + ((4 * g + j) * D + l16 * (D / 16));
      if constexpr (D == 128) {
        const uint2 w = *reinterpret_cast<const uint2*>(vr);
        t.v[4 * h + j][0] = w.x;
        t.v[4 * h + j][1] = w.y;
      } else {
        t.v[4 * h + j][0] = *reinterpret_cast<const uint32_t*>(vr);
      }
    }
  }
}

// one wave's running state for MT x 16 query rows (row l % 16 of each)
template <int D, int MT>
struct State {
  f4_t o[MT][D / 16];   // o[mt][i][r]: channel (D / 16) (4 (l / 16) + r) + i
  float ref[MT], sum[MT], vref[MT], ivref[MT];   // o is in units of vref, a power of two
};

__device__ __forceinline__ h8_t to_f16(const float (&y)[8]) {
  return join(__builtin_bit_cast(h2_t, pack_h2(y[0], y[1])), __builtin_bit_cast(h2_t, pack_h2(y[2], y[3])),
              __builtin_bit_cast(h2_t, pack_h2(y[4], y[5])), __builtin_bit_cast(h2_t, pack_h2(y[6], y[7])));
}

// One tile. The weights are rounded to f16 (2^-11 at most), or, FINE, to two f16 terms: for fp16 results, whose own rounding is no
// coarser than one (error 4.0e-4 -> 2.1e-4 of the largest, that of the result's rounding; bf16 results round by up to 2^-8). MORE: the
// wave's next tile (pages `pn`) is loaded into the same registers, its keys as soon as these are used, its values at the end: a load
// has about half a tile's work to come in.
// A row's weights are in units of its own, which follow the largest of them as the reference follows the scores: neither values that
// the row does not see nor large values of small probability take bits from the others, down to 2^-24 of the largest product.
template <int FMT, int D, int MT, bool FINE, bool MORE>
__device__ __forceinline__ void compute(const AttnArgs& a, Tile<D>& t, int kvh, int tile, const Pages& pg, const Pages& pn,
                                        const h8_t (&q)[MT][D / 32], const float (&qf)[MT], const int (&lim)[MT], int low, int len,
                                        State<D, MT>& st) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int kb = tile * TOKEN_KEYS;
  // low: keys that every row sees
  const bool edge = kb + TOKEN_KEYS > low || pg.p[0] < 0 || pg.p[1] < 0;
  float ks[8] = {t.ks[0].x, t.ks[0].y, t.ks[0].z, t.ks[0].w, t.ks[1].x, t.ks[1].y, t.ks[1].z, t.ks[1].w};
  float vs[8] = {t.vs[0].x, t.vs[0].y, t.vs[0].z, t.vs[0].w, t.vs[1].x, t.vs[1].y, t.vs[1].z, t.vs[1].w};
#pragma unroll
  for (int j = 0; j < 8; ++j) ks[j] = fmaf(vs[j], 0.0f, ks[j]);   // a NaN value marks the rows that see it as a NaN key does
  int key[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) key[j] = kb + 16 * (j >> 2) + 4 * g + (j & 3);

  f4_t acc[MT][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m][h] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 w = t.k[h][c];
      const h8_t k0 = f16x8<FMT>(w.x, w.y), k1 = f16x8<FMT>(w.z, w.w);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        acc[m][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[m][2 * c], acc[m][h], 0, 0, 0);
        acc[m][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[m][2 * c + 1], acc[m][h], 0, 0, 0);
      }
    }
  }
  if constexpr (MORE) load_keys<D>(a, kvh, tile + WAVES, pn, t);
  if (edge) {
    // what lies behind the sequence or in an absent page may be anything: its scales and, where codes can be NaN, its values go
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (key[j] >= len || pg.p[j >> 2] < 0) {
        vs[j] = 0.0f;
        if constexpr (FMT == E4M3) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c) t.v[j][c] = 0u;
        }
      }
    }
  }
  // a row's largest score and value scale, of the keys that it sees
  float x[MT][8], top[MT], vtop[MT];
  vtop[0] = vs[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) vtop[0] = fmaxf(vtop[0], vs[j]);
  bool move = false;
#pragma unroll
  for (int m = MT - 1; m >= 0; --m) {
    vtop[m] = vtop[0];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[m][j] = acc[m][j >> 2][j & 3] * (ks[j] * qf[m]);
    if (edge) {
      vtop[m] = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool hidden = key[j] >= lim[m] || pg.p[j >> 2] < 0;
        x[m][j] = hidden ? -INFINITY : x[m][j];
        vtop[m] = fmaxf(vtop[m], hidden ? 0.0f : vs[j]);
      }
    }
    top[m] = x[m][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top[m] = fmaxf(top[m], x[m][j]);
    // over 2^15: a probability, or what its product with a value's scale can be
    const float most = __builtin_amdgcn_exp2f(top[m] - (st.ref[m] == -INFINITY ? 0.0f : st.ref[m])) * (vtop[m] * st.ivref[m]);
    move |= top[m] - st.ref[m] > REF_STALE || !(most <= WEIGHT_MOST);
  }
  if (__builtin_amdgcn_ballot_w64(move)) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float n = across_max<true>(top[m]);
      float f = 1.0f;
      if (n - st.ref[m] > REF_STALE) {
        const float to = reference_under(n);
        f = __builtin_amdgcn_exp2f(st.ref[m] - to);   // from no keys yet: 2^-inf = 0
        st.ref[m] = to;
      }
      st.sum[m] *= f;
      // the weights' unit: down with the probabilities so far, up to where the largest weight of these keys is 2^10 to 2^11
      const float base = pow2_over(across_max<true>(vtop[m]));
      const float ibase = pow2_inverse(__float_as_int(base));
      float w = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        w = fmaxf(w, __builtin_amdgcn_exp2f(x[m][j] - (st.ref[m] == -INFINITY ? 0.0f : st.ref[m])) * (vs[j] * ibase));
      const float unit = weight_unit(st.vref[m], f, across_max<true>(w), base);
      st.ivref[m] = pow2_inverse(__float_as_int(unit));
      f *= st.vref[m] * st.ivref[m];
      st.vref[m] = unit;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) st.o[m][i] *= f;
    }
  }
  h8_t p[MT], rest[FINE ? MT : 1];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    // a row that has seen no key yet has only -inf here: any finite reference gives it zeros
    const float ref = st.ref[m] == -INFINITY ? 0.0f : st.ref[m];
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float e = __builtin_amdgcn_exp2f(x[m][j] - ref);
      st.sum[m] += e;
      y[j] = e * (vs[j] * st.ivref[m]);
    }
    if (edge) {   // a key that the row does not see may hold NaN
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (key[j] >= lim[m]) y[j] = 0.0f;
    }
    p[m] = to_f16(y);
    if constexpr (FINE) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] -= static_cast<float>(p[m][j]);
      rest[m] = to_f16(y);
    }
  }
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = t.v[j][c];
    h8_t v[4];
    f16x8_across<FMT>(w, v);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        st.o[m][4 * c + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[i], p[m], st.o[m][4 * c + i], 0, 0, 0);
        if constexpr (FINE) st.o[m][4 * c + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[i], rest[m], st.o[m][4 * c + i], 0, 0, 0);
      }
  }
  if constexpr (MORE) load_values<D>(a, kvh, tile + WAVES, pn, t);
}

template <int FMT, int D, int MT, bool FINE>
__global__ void __launch_bounds__(NT, 2) token_kernel(AttnArgs a) {
  constexpr int R = 16 * MT, PAD = D + 4;
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

    // query rows: lane l holds row l % 16, channels 64 c + 16 (l / 16) + 0 .. 15 in steps 2 c and 2 c + 1
    uint4 raw[MT][D / 32];
    int lim[MT];
    int t = t0 + wave;
    Pages pg = pages_of(a, row, width, t), pn = pages_of(a, row, width, t + WAVES);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = rt * R + 16 * m + l16;
      const int rr = row < rows ? row : 0;
      const int tok = rr / a.group, hd = kvh * a.group + rr - tok * a.group;
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + (sq.first + tok) * a.q_st + hd * a.q_sh + 16 * g;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) raw[m][c] = *reinterpret_cast<const uint4*>(src + 64 * (c >> 1) + 8 * (c & 1));
      lim[m] = causal ? min(sq.len, sq.pos + tok + 1) : sq.len;
    }
    // the first keys and values are on their way while the query rows come in
    Tile<D> tile;
    if (t < t1) {
      load_keys<D>(a, kvh, t, pg, tile);
      load_values<D>(a, kvh, t, pg, tile);
    }
    h8_t q[MT][D / 32];
    float qf[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const bool has = rt * R + 16 * m + l16 < rows;
      float x[D / 32][8], top = 0.0f;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        row8<FINE ? RH3_DTYPE_F16 : RH3_DTYPE_BF16>(raw[m][c], x[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[c][e] = has ? x[c][e] : 0.0f;
          top = fmaxf(top, fabsf(x[c][e]));
        }
      }
      const int e = q_exponent(across_max<true>(top));
#pragma unroll
      for (int c = 0; c < D / 32; ++c) q[m][c] = q_f16(x[c], e);
      qf[m] = __builtin_amdgcn_ldexpf(a.scale_log2, -e);
    }
    const int low = causal ? min(sq.len, sq.pos + scalar((rt * R) / a.group) + 1) : sq.len;

    State<D, MT> st;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      st.ref[m] = -INFINITY;
      st.sum[m] = 0.0f;
      st.vref[m] = 0.0f;
      st.ivref[m] = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) st.o[m][i] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if (t < t1) {
      for (; t + WAVES < t1; t += WAVES) {
        const Pages p2 = pages_of(a, row, width, t + 2 * WAVES);
        compute<FMT, D, MT, FINE, true>(a, tile, kvh, t, pg, pn, q, qf, lim, low, sq.len, st);
        pg = pn;
        pn = p2;
      }
      compute<FMT, D, MT, FINE, false>(a, tile, kvh, t, pg, pn, q, qf, lim, low, sq.len, st);
    }
    // join the 4 waves
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
        for (int i = 0; i < D / 16; i += 4) {
          float4 v = make_float4(st.o[m][i][r], st.o[m][i + 1][r], st.o[m][i + 2][r], st.o[m][i + 3][r]);
          v.x = v.x * PART * st.vref[m];
          v.y = v.y * PART * st.vref[m];
          v.z = v.z * PART * st.vref[m];
          v.w = v.w * PART * st.vref[m];
          *reinterpret_cast<float4*>(&so[wave][16 * m + l16][(D / 16) * (4 * g + r) + i]) = v;
        }
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
      float f[WAVES], sum = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        f[w] = sm[w][rl] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[w][rl] - top);
        sum += f[w] * sl[w][rl];
      }
      float o[EPT];
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        o[e] = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) o[e] += f[w] * so[w][rl][d0 + e];
      }
      if (whole && !a.keep) {
        const int tok = rw / a.group, hd = kvh * a.group + rw - tok * a.group;
        const float inv = sum == 0.0f ? 0.0f : (1.0f / PART) / sum;
        uint32_t w[EPT / 2];
#pragma unroll
        for (int e = 0; e < EPT; e += 2) w[e / 2] = pack_out(a, o[e] * inv, o[e + 1] * inv);
        uint16_t* dst = static_cast<uint16_t*>(a.out) + (sq.first + tok) * a.o_st + hd * a.o_sh + d0;
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
        for (int e = 0; e < EPT; e += 4) *reinterpret_cast<float4*>(po + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        if (d0 == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * R + rl) * 2) = make_float2(top, sum);
      }
    }
    if (u < end) __syncthreads();
  }
}

}  // namespace

void launch_token(const AttnArgs& a, int fmt, int dim, int rows, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(a.wgs)), dim3(NT), 0, st, a); };
  auto by_type = [&](auto bf16, auto fp16) { a.fp16 ? go(fp16) : go(bf16); };
  if (dim == 128 && fmt == INT8) by_type(token_kernel<INT8, 128, 1, false>, token_kernel<INT8, 128, 1, true>);
  else if (dim == 128) by_type(token_kernel<E4M3, 128, 1, false>, token_kernel<E4M3, 128, 1, true>);
  else if (fmt == INT8 && rows == 16) by_type(token_kernel<INT8, 64, 1, false>, token_kernel<INT8, 64, 1, true>);
  else if (fmt == INT8) by_type(token_kernel<INT8, 64, 2, false>, token_kernel<INT8, 64, 2, true>);
  else if (rows == 16) by_type(token_kernel<E4M3, 64, 1, false>, token_kernel<E4M3, 64, 1, true>);
  else by_type(token_kernel<E4M3, 64, 2, false>, token_kernel<E4M3, 64, 2, true>);
}

}  // namespace kv
}  // namespace rh3
