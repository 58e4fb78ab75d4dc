// Attention of many query rows over the 4-bit paged cache: kv_chunk.hip's way through the work, for codes and scales of kv_four.hpp.
//
// 4 dim flops per query row and key, while a key's 2 (dim / 2 + dim / 32) bytes serve all rows of a tile. Measured: 2,048 rows x 32 / 8
// heads at the end of 16,384 keys 460 to 545 us by how far the card's clock falls under it (0.95 to 1.12 PFLOP/s; a large bf16 matrix
// product reaches 1.36 to 1.39); 120 rows x 56 / 8 heads on 24,001 keys 108 us (770 TFLOP/s, 930 of those that it computes: 840 rows
// to a K/V head are 4 tiles of 256). Of the first's cycles, at 1.96 GHz, the matrix units are busy in 50 %, the vector units in 43 %,
// LDS in 37 %, and the waves wait for 28 % of their time.
//
// A workgroup of 4 or 8 waves holds 32 query rows of one K/V head on each and walks its keys 64 at a time. The keys' codes come to
// registers a step ahead, are converted to bf16 (exact, their powers of two included) once for all waves and written to LDS (two
// buffers, one barrier to a step), K and V alike. Per wave
//   S^T = K Q^T (32x32x16 bf16): a lane has one query row (l % 32) and 16 of 32 keys, so a row's softmax is in-lane but for one
//   exchange, and only when its reference moves; the probabilities are the B operand of
//   O^T = V^T P^T as they stand: k-step t of 32 keys takes keys 16 t + 4 (l / 32) + 0 .. 3 and those + 8, and V's operand comes
//   from LDS by transposing loads.
// The keys are taken by halves of 32: while one half's softmax runs, so do the MFMAs of the next half's scores and of the half
// before's values. Where keys are masked, a page is absent or a reference has to move, a plain path does the half.
// Vector work per score: one fma (softmax scale and reference at once), the exponential, the sum and half a conversion.
// Roundings: the probability to bf16, 2^-8 relative at most, as a bf16 result's own: on random rows a result is off by 2.34e-3 (relative
// to all values' norm) for the 1.66e-3 of its own rounding alone. Two terms, which leave 1.66e-3, are a half more matrix work: the first
// size took 668 us for 480. FINE, for fp16 results: the queries, which bf16 does not hold, and the probabilities in two terms each (2^-16).
#include "kv_four.hpp"

namespace rh3 {
namespace kv {
namespace {

constexpr int KT = CHUNK_KEYS;
constexpr float SUM_STALE = 0x1p-12f;        // up to this sum of a half's probabilities none of them is over 2^STALE
// Past it one of 16 is over 2^(STALE - 4): the plain path moves the reference from a little under that on, so that the next halves of
// scores like these pass (with STALE itself, scores 9 to 12 over a share's first ones go both paths half after half until their sum
// moves it; before it did, to the end: 488 us for 266)
constexpr float SLOW_STALE = STALE - 5.0f;

// 16-byte pieces of the LDS rows. Each row has one piece more than it needs, so that 16 rows' pieces of one number lie in all 16
// parts of the banks, and every read of a tile is one lane address with an immediate offset.
template <int D>
constexpr int K_ROW = D / 8 + 1;                               // K: [64 keys][D] bf16
// V: the same, but read by transposing loads (8 bytes a lane, 4 rows x 32 channels to 32 lanes): rows 64 bytes apart in the banks
template <int D>
constexpr int V_ROW = D / 8 + 4;

// 4 rows x 16 channels to 16 lanes: lane i gives the address of row i / 4, channels 4 (i % 4) + 0 .. 3, and gets channel i's 4 rows
typedef __bf16 g4_t __attribute__((__vector_size__(4 * sizeof(__bf16))));
typedef __bf16 b4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ b4_t lds_read_tr(const uint8_t* p) {
  return __builtin_bit_cast(b4_t, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) g4_t*)p));
}

template <int D, int WAVES, bool FINE>
__global__ void __launch_bounds__(WAVES * 64, 2) chunk_kernel(AttnArgs a) {
  constexpr int R = WAVES * 32, KS = D / 16, DT = D / 32;
  const Tiling TILING = tiling(true, R);
  __shared__ uint4 sk[2][KT * K_ROW<D>];
  __shared__ uint4 sv[2][KT * V_ROW<D>];
  __shared__ int sgone[WAVES];
  const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int NP = 8 / WAVES;           // pieces of 8 keys that a wave converts
  const float scale = a.scale_log2;

  // neighbouring shares, which read the same keys, on one XCD (workgroups are dealt to the 8 XCDs in turn)
  const int n8 = a.wgs & ~7;
  const int wg = static_cast<int>(blockIdx.x) < n8 ? (blockIdx.x & 7) * (n8 >> 3) + (blockIdx.x >> 3) : blockIdx.x;
  int64_t u, end;
  {
    Block blk;
    const Work work = dealt(load_blocks(a, TILING, blk), a.wgs, TILING);
    if (wg >= work.wgs) return;
    u = scalar(share_begin(work, wg));
    end = scalar(share_begin(work, wg + 1));
  }

  while (u < end) {
    // the sequences are looked up again for every item: kept, they would take registers from the loop below
    Block blk;
    load_block(a, TILING, 0, 0, 0, blk);
    while (u >= blk.end()) {
      if (blk.at + 64 >= sequences(a)) return;
      next_block(a, TILING, blk);
    }
    const int in_block = __builtin_ctzll(__builtin_amdgcn_ballot_w64(blk.base + blk.units > u));
    const int seq = blk.at + in_block;
    const SeqItems sw = seq_in(a, blk, in_block);
    const Seq sq = sw.seq;
    const int64_t local = u - sw.before;
    const int item = scalar(static_cast<int>(quotient(local, sw.span)));
    const int u0 = static_cast<int>(local - static_cast<int64_t>(item) * sw.span);
    const int u1 = static_cast<int>(end - u < sw.span - u0 ? u0 + (end - u) : sw.span);
    u += u1 - u0;
    const int t0 = max(u0 - TILING.extra, 0), share_t1 = u1 - TILING.extra;
    if (share_t1 <= 0) continue;
    const bool whole = t0 == 0 && u1 == sw.span;
    const bool pre = a.prefix && seq == 0, causal = a.causal && !pre;
    const int32_t* table = pre ? a.prefix : a.s.table + (seq - (a.prefix != nullptr)) * a.s.table_stride;
    const int width = pre ? a.prefix_width : a.s.width;
    const int kvh = scalar(item / sw.row_tiles), at = item - kvh * sw.row_tiles;
    const int rt = causal ? tile_at_place(at, sw.row_tiles) : at;
    const int rows = sq.n * a.group;
    const int tok_last = scalar(min(rows - 1, rt * R + R - 1) / a.group);
    const int seen = causal ? min(sq.len, max(0, sq.pos + tok_last + 1)) : sq.len;   // keys that some row sees
    const int t1 = min(share_t1, (seen + KT - 1) / KT);

    const int row = rt * R + wave * 32 + l32;
    const bool has = row < rows;
    const int rr = has ? row : rows - 1;
    const int tok = rr / a.group, hd = kvh * a.group + rr - tok * a.group;
    const int mask = (1 << a.c.log2page) - 1;
    auto page_in = [&](int entry) { return entry >= 0 && entry < a.c.pages ? entry : -1; };
    const int lim = causal ? min(sq.len, sq.pos + tok + 1) : sq.len;
    // of the wave's rows: keys that all see, keys that some see
    const int r0 = rt * R + wave * 32, r1 = min(rows - 1, r0 + 31);
    const int low = causal ? min(sq.len, sq.pos + scalar(r0 / a.group) + 1) : sq.len;
    const int top_key = r0 >= rows ? 0 : causal ? min(sq.len, sq.pos + scalar(r1 / a.group) + 1) : sq.len;

    f16_t o[DT];
    float ref = NO_REF, sum = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

    // Window w: keys [64 w - 32, 64 w + 32). Stage x in LDS (buffer x & 1) has K of window x + 1 and V of window x. A wave brings 8
    // NP keys of a window, which lie in one page; lane l has 1 / 8 of key l / 8 of each 8, all of one group of channels.
    const int first = 8 * NP * wave;
    auto lookup = [&](int w) {   // the entry of the wave's page; the first window begins before the sequence
      // not by a scalar load: that, on its way, would make every wait for an LDS read a wait for all of them
      return table[min(max(w * KT - 32 + first, 0) >> a.c.log2page, width - 1)];
    };
    uint32_t kraw[NP][D / 64], vraw[NP][D / 64];
    uint32_t ks[NP], vs[NP];               // scale bytes of the lane's group
    int kpage, vpage, entry;               // the wave's pages in the two windows; the entry for K's next one
    auto load_window = [&](const uint8_t* codes, const float* scales, int page, int w, uint32_t (&raw)[NP][D / 64], uint32_t (&s)[NP]) __attribute__((always_inline)) {
      const int off = (w * KT - 32 + first) & mask;
      const uint8_t* at = codes + (max(page, 0) * a.c.page_stride + kvh * a.c.head_stride + off * (D / 2));
      const uint8_t* st = reinterpret_cast<const uint8_t*>(scales) + (max(page, 0) * a.c.spage_stride + kvh * a.c.shead_stride + off * (D / 32));
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if constexpr (D == 128) {
          const uint2 r = *reinterpret_cast<const uint2*>(at + (8 * lane + 8 * (D / 2) * i));
          raw[i][0] = r.x; raw[i][1] = r.y;
        } else {
          raw[i][0] = *reinterpret_cast<const uint32_t*>(at + (4 * lane + 8 * (D / 2) * i));
        }
        s[i] = st[8 * (D / 32) * i + (lane >> 3) * (D / 32) + ((lane & 7) * (D / 8)) / GROUP4];
      }
    };
    if (t0 < t1) {   // the first loads, beside those of the query rows
      kpage = page_in(scalar(lookup(t0)));
      load_window(a.c.k, a.c.ks, kpage, t0, kraw, ks);
      entry = lookup(t0 + 1);
    }
    b8_t q[KS], ql[FINE ? KS : 1];
    {
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + (sq.first + tok) * a.q_st + hd * a.q_sh + 8 * hi;
#pragma unroll
      for (int s = 0; s < KS; ++s) query8<FINE>(*reinterpret_cast<const uint4*>(src + 16 * s), q[s], ql[FINE ? s : 0]);
    }
    bool full;  // no key of the share in an absent page
    {
      bool gone = false;
      for (int i = (t0 * KT >> a.c.log2page) + static_cast<int>(threadIdx.x); i <= (min(t1 * KT, sq.len) - 1) >> a.c.log2page; i += WAVES * 64)
        gone |= page_in(table[min(i, width - 1)]) < 0;
      const int any = __builtin_amdgcn_ballot_w64(gone) != 0;
      if (lane == 0) sgone[wave] = any;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) gone |= sgone[w] != 0;
      full = __builtin_amdgcn_ballot_w64(gone) == 0;
    }
    auto all_there = [&](int s) {   // no key of step s in an absent page
      if (full) return true;
      int bad = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = scalar_load(table + min((s * KT + 16 * i) >> a.c.log2page, width - 1));
        bad |= e < 0 || e >= a.c.pages;
      }
      return bad == 0;
    };
    // Stage x (loaded) to LDS in 2 NP parts of K and 2 NP of V; the loads of stage x + 1
    auto put_k = [&](int x, int part) __attribute__((always_inline)) {
      const int i = part / 2, c = part % 2, key = first + 8 * i + (lane >> 3);
      if (c < D / 64) sk[x & 1][key * K_ROW<D> + (lane & 7) * (D / 64) + c] = words4(kraw[i][c < D / 64 ? c : 0], __uint_as_float(ks[i] << 23));
    };
    auto put_v = [&](int x, int part) __attribute__((always_inline)) {
      const int i = part / 2, c = part % 2, key = first + 8 * i + (lane >> 3);
      // outside the share's keys and in an absent page there may be anything: 0
      const int pos = x * KT - 32 + key;
      const bool here = vpage >= 0 && pos >= t0 * KT && pos < min(sq.len, t1 * KT);
      if (c < D / 64) {
        const uint32_t w = here ? vraw[i][c < D / 64 ? c : 0] : 0u, s = here ? vs[i] << 23 : 0u;
        sv[x & 1][key * V_ROW<D> + (lane & 7) * (D / 64) + c] = words4(w, __uint_as_float(s));
      }
    };
    auto next_v = [&](int x) __attribute__((always_inline)) {   // (before next_k: the window's page is K's of stage x)
      vpage = kpage;
      load_window(a.c.v, a.c.vs, vpage, x + 1, vraw, vs);
    };
    auto next_k = [&](int x) __attribute__((always_inline)) {
      kpage = page_in(scalar(entry));
      entry = lookup(x + 3);
      load_window(a.c.k, a.c.ks, kpage, x + 2, kraw, ks);
    };
    auto stage_v = [&](int x) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2 * NP; ++i) put_v(x, i);
      next_v(x);
    };
    auto stage_k = [&](int x) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2 * NP; ++i) put_k(x, i);
      next_k(x);
    };

    // Half h's softmax runs beside the products of half h + 1 and the values of half h - 1. Step s does halves 2 s and 2 s + 1 with
    // stage s.
    const f16_t zero = {};
    f16_t sa = zero, sb = zero;            // products of the next even and odd half
    b8_t p[2] = {}, pr[2] = {};   // weights of the last half, what their rounding left
    constexpr int AHEAD = 4;
    auto k_at = [&](int b, int half, int ks) { return __builtin_bit_cast(b8_t, sk[b][(32 * half + l32) * K_ROW<D> + hi + 2 * ks]); };
    const uint8_t* v_lane = reinterpret_cast<const uint8_t*>(sv) + (4 * hi + ((lane & 15) >> 2)) * V_ROW<D> * 16 + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    auto v_at = [&](int b, int half, int i) {   // i: k-step * DT + channel tile
      const uint8_t* at = v_lane + ((b * KT + 32 * half + 16 * (i / DT)) * V_ROW<D> * 16 + 64 * (i % DT));
      const b4_t lo = lds_read_tr(at), up = lds_read_tr(at + 8 * V_ROW<D> * 16);
      return __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto scores = [&](b8_t k, int i, f16_t c) __attribute__((always_inline)) {
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[i], c, 0, 0, 0);
      if constexpr (FINE) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, ql[i], c, 0, 0, 0);
      return c;
    };
    auto weigh = [&](b8_t v, int i) __attribute__((always_inline)) {   // i: as v_at's
      o[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, p[i / DT], o[i % DT], 0, 0, 0);
      if constexpr (FINE) o[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, pr[i / DT], o[i % DT], 0, 0, 0);
    };
    // Weights of two keys to bf16; FINE: in two terms
    auto weights = [&](float w0, float w1, uint32_t& rest) __attribute__((always_inline)) {
      const uint32_t w = pack_bf2(w0, w1);
      if constexpr (FINE) rest = pack_bf2(w0 - __uint_as_float(w << 16), w1 - __uint_as_float(w & 0xffff0000u));
      return w;
    };
    auto set2 = [](b8_t (&x)[2], int e, uint32_t w) __attribute__((always_inline)) {
      const b2_t r = __builtin_bit_cast(b2_t, w);
      x[e / 8][e % 8] = r[0];
      x[e / 8][e % 8 + 1] = r[1];
    };
    // Half H of step s, its softmax spread evenly over the half's MFMAs; the sum of its probabilities. `side(i)` goes with MFMA i.
    auto fast = [&](auto H, int b, f16_t& now, f16_t& next, b8_t (&f)[AHEAD], b8_t (&n)[2], b8_t (&nr)[2], auto side) __attribute__((always_inline)) {
      constexpr int HALF = decltype(H)::value, MM = KS + 2 * DT, N = 16 / MM;
      float y[N], w[16], more = 0.0f;
      auto score = [&](int e) __attribute__((always_inline)) { y[e % N] = fmaf(now[e], scale, -ref); };
      auto pair = [&](int e) __attribute__((always_inline)) {
        more = e == 0 ? w[0] + w[1] : more + (w[e] + w[e + 1]);
        uint32_t rest = 0, bits = weights(w[e], w[e + 1], rest);
        if constexpr (FINE) {
          asm volatile("" : "+v"(rest));
          set2(nr, e, rest);
        }
        asm volatile("" : "+v"(bits), "+v"(more));   // done here, not behind the last MFMA
        set2(n, e, bits);
      };
#pragma unroll
      for (int e = 0; e < N; ++e) score(e);
#pragma unroll
      for (int i = 0; i < MM; ++i) {
        const int r = i + AHEAD;
        if (i < KS) next = scores(f[i % AHEAD], i < KS ? i : 0, i ? next : zero);
        else weigh(f[i % AHEAD], i < KS ? 0 : i - KS);
        if (r < KS) f[i % AHEAD] = k_at(b, HALF, r);
        else if (r < MM) f[i % AHEAD] = v_at(b, HALF, r - KS);
        else if (HALF == 0) f[i % AHEAD] = k_at(b, 1, r - MM);
#pragma unroll
        for (int e = i * N; e < i * N + N; ++e) w[e] = __builtin_amdgcn_exp2f(y[e % N]);
        if (i + 1 < MM) {
#pragma unroll
          for (int e = (i + 1) * N; e < (i + 1) * N + N; ++e) score(e);
        }
        if (i * N >= 2 && (i * N) % 2 == 0) pair(i * N - 2);
        side(i);
        __builtin_amdgcn_sched_barrier(0);
      }
      pair(14);
      return more;
    };
    bool there = all_there(t0);   // of the step at hand
    bool begun = false;           // the first step sets the references
    // Any half: keys that a row does not see hidden, the reference moved where it must be
    auto slow = [&](int b, int s, int half, bool made, f16_t& now, f16_t& next) __attribute__((always_inline)) {
      const int h = 2 * s + half;
      if (!made) {
#pragma unroll
        for (int i = 0; i < 2 * DT; ++i) weigh(v_at(b, half, i), i);
        next = zero;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) next = scores(k_at(b, half, ks), ks, next);
      }
      const int key0 = 32 * h + 4 * hi, m = lim - key0;
      uint32_t gone = 0;
      if (!there)
        gone = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(page_in(table[min((32 * h + l32) >> a.c.log2page, width - 1)]) < 0) >> (4 * hi));
      float y[16], top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = 8 * (i >> 2) + (i & 3);
        y[i] = now[i] * scale;
        y[i] = (key >= m) | ((gone >> key) & 1) ? -INFINITY : y[i];
        top = fmaxf(top, y[i]);
      }
      top = across_max<false>(top);
      const float to = next_reference(ref, top, across_sum<false>(sum), SLOW_STALE);
      const float f = __builtin_amdgcn_exp2f(ref - to);
      ref = to;
      sum *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(y[i] - to), e1 = __builtin_amdgcn_exp2f(y[i + 1] - to);
        sum += e0 + e1;
        uint32_t rest = 0;
        set2(p, i, weights(e0, e1, rest));
        if constexpr (FINE) set2(pr, i, rest);
      }
    };
    auto take = [&](const b8_t (&n)[2], const b8_t (&nr)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        p[i] = n[i];
        if constexpr (FINE) pr[i] = nr[i];
      }
    };
    if (t0 < t1) {
      // stage t0 - 1 is only K of window t0
#pragma unroll
      for (int i = 0; i < 2 * NP; ++i) put_k(t0 - 1, i);
      next_v(t0 - 1);
      next_k(t0 - 1);
      __syncthreads();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) sa = scores(k_at((t0 - 1) & 1, 1, ks), ks, sa);
      stage_v(t0);
      stage_k(t0);
    }
    __syncthreads();
    int s = t0;
    while (s < t1) {
      // of the step at hand: V's and K's stage, the even half, the products of the half at hand
      bool staged_v = false, staged_k = false, odd = false, made = false;
      // Steps whose every key every row sees. The accumulators stay in place in a loop of their own; a step's instructions stay
      // in the order written: behind each MFMA an operand's read for the one after next but two, and vector work that it covers.
      while (begun && there && s * KT + KT <= low) {
        const int b = s & 1;
        constexpr int MM = KS + 2 * DT, EACH = MM / (4 * NP);
        b8_t f[AHEAD], n[2], nr[2];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) f[i] = k_at(b, 0, i);
        __builtin_amdgcn_sched_barrier(0);
        float more = fast(std::integral_constant<int, 0>(), b, sa, sb, f, n, nr, [&](int i) __attribute__((always_inline)) {
          if (i >= MM / 2 && i % EACH == 0) put_v(s + 1, (i - MM / 2) / EACH);
          if (i == MM - 1) next_v(s + 1);
        });
        staged_v = made = true;
        if (__builtin_amdgcn_ballot_w64(more > SUM_STALE)) break;   // a reference has to move
        sum += more;
        take(n, nr);
        odd = true;
        more = fast(std::integral_constant<int, 1>(), b, sb, sa, f, n, nr, [&](int i) __attribute__((always_inline)) {
          if (i >= MM / 2 && i % EACH == 0) put_k(s + 1, (i - MM / 2) / EACH);
          if (i == MM - 1) next_k(s + 1);
        });
        staged_k = true;
        if (__builtin_amdgcn_ballot_w64(more > SUM_STALE)) break;
        sum += more;
        take(n, nr);
        __syncthreads();
        staged_v = staged_k = odd = made = false;
        there = all_there(++s);
        if (s >= t1) break;
        // now and then: 8 steps bring a lane's sum 2^-8 further at most
        if ((s & 7) == 0 && __builtin_amdgcn_ballot_w64(sum > SUM_MOST)) break;
      }
      if (s >= t1) break;
      const int b = s & 1;
      if ((s - 1) * KT < top_key) {   // (a step past the last key that a row sees sums its last values)
        if (!odd) slow(b, s, 0, made, sa, sb);
        slow(b, s, 1, made && odd, sb, sa);
      }
      if (!staged_v) stage_v(s + 1);
      if (!staged_k) stage_k(s + 1);
      begun = true;
      __syncthreads();
      there = all_there(++s);
    }
    if (t0 < t1) {   // the last half's values
#pragma unroll
      for (int i = 0; i < 2 * DT; ++i) weigh(v_at(t1 & 1, 0, i), i);
    }
    __syncthreads();   // the next item's tiles go where these are read

    // lane: query row l % 32, channels 32 d + 8 i + 4 (l / 32) + 0 .. 3
    const float total = across_sum<false>(sum);
    if (has) {
      if (whole && !a.keep) {
        const int tok = row / a.group, hd = kvh * a.group + row - tok * a.group;
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        uint16_t* dst = static_cast<uint16_t*>(a.out) + (sq.first + tok) * a.o_st + hd * a.o_sh + 4 * hi;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint2*>(dst + 32 * d + 8 * i) = make_uint2(pack_out(a, o[d][4 * i] * inv, o[d][4 * i + 1] * inv),
                                                                      pack_out(a, o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv));
        if (a.lse && hi == 0)
          a.lse[static_cast<int64_t>(sq.first + tok) * a.c.heads * a.group + hd] =
              total == 0.0f ? -INFINITY : (__builtin_amdgcn_logf(total) + ref) * 0.6931471805599453f;
      } else if (!whole || sw.items_before + item < a.items) {   // (a cu that falls can count rows more than once)
        // slots: two to a workgroup (the item that it goes on with, the one that it begins), then one to an item that it completes
        const int64_t slot = whole ? 2 * static_cast<int64_t>(a.wgs) + sw.items_before + item : 2 * static_cast<int64_t>(wg) + (t0 == 0);
        const int rl = wave * 32 + l32;
        float* po = a.part_o + (slot * R + rl) * D + 4 * hi;
        constexpr float UNIT = PART * PART_UP;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(po + 32 * d + 8 * i) =
                make_float4(o[d][4 * i] * UNIT, o[d][4 * i + 1] * UNIT, o[d][4 * i + 2] * UNIT, o[d][4 * i + 3] * UNIT);
        if (hi == 0)
          *reinterpret_cast<float2*>(a.part_ml + (slot * R + rl) * 2) =
              make_float2(total == 0.0f ? -INFINITY : total == total ? ref - OVER : 0.0f, total * PART_UP);
      }
    }
  }
}

}  // namespace

void launch_chunk4(const AttnArgs& a, int dim, int rows, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(a.wgs)), dim3(static_cast<uint32_t>(2 * rows)), 0, st, a); };
  auto by = [&](auto four, auto eight, auto four_fine, auto eight_fine) {
    if (rows == 128) a.fp16 ? go(four_fine) : go(four);
    else a.fp16 ? go(eight_fine) : go(eight);
  };
  if (dim == 128) by(chunk_kernel<128, 4, false>, chunk_kernel<128, 8, false>, chunk_kernel<128, 4, true>, chunk_kernel<128, 8, true>);
  else by(chunk_kernel<64, 4, false>, chunk_kernel<64, 8, false>, chunk_kernel<64, 4, true>, chunk_kernel<64, 8, true>);
}

}  // namespace kv
}  // namespace rh3
