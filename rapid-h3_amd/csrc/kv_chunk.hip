// Attention of many query rows over the paged cache: a chunk of a prompt, the tokens of a frame, a whole batch against a prefix
// that it shares.
//
// 4 dim flops per query row and key, while a key's 2 (dim + 4) bytes serve all rows of a tile. Measured: 2,048 rows x 32 / 8 heads
// at the end of 16,384 keys, int8, 590 to 660 us (780 to 870 TFLOP/s by how long the card has been busy); 1,560 rows x 56 heads on
// 22,332 keys, e4m3, 1,280 to 1,400 us (710 to 780); 64 x 4 rows x 8 heads on 32,768 keys 71 us (480). A large f16 matrix product
// reaches 1,485. Of the first's cycles, at 2.0 GHz, the matrix units are busy in 37 %, the vector units in 42 %, LDS in 34 %, and the
// waves wait for 37 % of their time: no unit is full, but two waves to a SIMD do not cover each other's way from scores over
// weights to values, and the clock falls as the units fill. The next limit is LDS: 64 keys at dim 128 are 288 KB of reads and
// writes for 8 waves, 2,300 cycles, beside 2,048 of MFMA.
//
// A workgroup of 4 or 8 waves holds 32 query rows of one K/V head on each and walks its keys 64 at a time. The keys' codes come
// to registers a step ahead, are converted to f16 once for all waves and written to LDS (two buffers, one barrier to a step), K
// and V alike. Per wave
//   S^T = K Q^T (32x32x16 f16): a lane has one query row (l % 32) and 16 of 32 keys, so a row's softmax is in-lane but for one
//   exchange, and only when its reference moves; the probabilities are the B operand of
//   O^T = V^T P^T as they stand: k-step t of 32 keys takes keys 16 t + 4 (l / 32) + 0 .. 3 and those + 8, and V's operand comes
//   from LDS by transposing loads.
// The keys are taken by halves of 32: while one half's softmax runs, so do the MFMAs of the next half's scores and of the half
// before's values, one MFMA to every one (dim 64: two) of the lane's 16 scores. Where keys are masked, a page is absent or a
// reference has to move, a plain path does the half.
// Vector work per score: one fma (key scale, softmax scale and reference at once), the exponential, the sum and half a
// conversion. For that, the query rows of a workgroup share one power of two, if each row's largest is within 2^15 of the tile's (an
// element is then off by 2^-24 of its own row's largest at most); rows further apart, as of an idle slot of a batch beside the
// others, have one each, and the plain path does the whole item with a row's own factor in its scores. A value's scale, relative
// to a power of two over the largest of the share's keys (a scan of the scales before the first step), is multiplied into V as it
// is converted, if those scales are within 2^18 of each other (rows of zeros aside). Else a large value would take bits from rows
// that do not see it, or hardly: the plain path takes that item, too, and multiplies the scales into the probabilities, in a unit
// of each row's own (the first size with one query row of 10^12, or values of 10^9, in every tile: 1,290 us; a tile alone as much
// longer). With rows of zeros on every page 617.
// Roundings to f16: the probability, the value's scale, and the product of that with the code; 2^-11 relative at most each, with
// fp32 sums, beside a bf16 result's own 2^-8. FINE, for fp16 results, whose own rounding is no coarser: the scale (within 2^14 of
// the others) is multiplied into the probability, which is kept in two f16 terms (error of 300 rows on 3,000 keys 4.0e-4 ->
// 2.1e-4, that of the result's rounding; the first size above 590 -> 810 us, the last 80 -> 97 with its join).
//
// Tried and slower, or no faster: exponentials only beside the values' MFMAs (703 against 688 us for the first size above), the
// next step's page entries looked up one by one behind the barrier (688 against 670), a load two steps ahead of the next one that
// brings its lines to the L2 (723), the largest score in place of the probabilities' sum to find that a reference must move, 64
// rows to each of 4 waves, which halves the reads of LDS but leaves one wave to a SIMD (915 against 670).
#include <type_traits>

#include "kv_attn.hpp"

namespace rh3 {
namespace kv {
namespace {

constexpr int KT = CHUNK_KEYS;
constexpr float SUM_STALE = 0x1p15f;  // up to this sum of a half's probabilities none of them is over 2^REF_STALE
constexpr float ROWS_APART = 0x1p-15f;  // query rows whose largest is this far below the tile's do not share its power of two
constexpr float LEAST_SCALE = 1e-12f;   // the quantizers' least, that of a row of zeros
constexpr float NO_REF = -0x1.fffffep127f;   // reference of a row that has seen no key: any score moves it

// 16-byte pieces of the LDS rows. Each row has one piece more than it needs, so that 16 rows' pieces of one number lie in all 16
// parts of the banks, and every read of a tile is one lane address with an immediate offset.
template <int D>
constexpr int K_ROW = D / 8 + 1;                               // K: [64 keys][D] f16
// V: the same, but read by transposing loads (8 bytes a lane, 4 rows x 32 channels to 32 lanes): rows 64 bytes apart in the banks
template <int D>
constexpr int V_ROW = D / 8 + 4;

// whether a row of codes has one that is not zero
template <int FMT, int D>
__device__ __forceinline__ bool codes_in(const uint8_t* row) {
  uint32_t any = 0;
#pragma unroll 1
  for (int i = 0; i < D / 16; ++i) {
    const uint4 r = reinterpret_cast<const uint4*>(row)[i];
    any |= r.x | r.y | r.z | r.w;
  }
  return (any & (FMT == INT8 ? 0xffffffffu : 0x7f7f7f7fu)) != 0;
}

// 4 rows x 16 channels to 16 lanes: lane i gives the address of row i / 4, channels 4 (i % 4) + 0 .. 3, and gets channel i's 4 rows
typedef __fp16 g4_t __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ h4_t lds_read_tr(const uint8_t* p) {
  return __builtin_bit_cast(h4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) g4_t*)p));
}

template <int FMT, int D, int WAVES, bool FINE>
__global__ void __launch_bounds__(WAVES * 64, 2) chunk_kernel(AttnArgs a) {
  constexpr int R = WAVES * 32, KS = D / 16, DT = D / 32;
  const Tiling TILING = tiling(true, R);
  __shared__ uint4 sk[2][KT * K_ROW<D>];
  __shared__ uint4 sv[2][KT * V_ROW<D>];
  __shared__ float sks[8][32];            // key scales of 8 half tiles in turn
  __shared__ float svs[8][32];            // value scales of them (where they go to the weights)
  __shared__ float stop[WAVES], sleast[WAVES], sscale[WAVES], ssmall[WAVES];
  __shared__ float srow[WAVES * 32], sunit[WAVES * 32];   // rows or values far apart: a row's factor of its scores, unit of its weights
  __shared__ int sgone[WAVES];
  const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int NP = 8 / WAVES;           // pieces of 8 keys that a wave converts

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
    h8_t q[KS];
    float qf;
    int vref;   // bits of a power of two, the same in all lanes
    bool full;  // no key of the share in an absent page
    bool apart; // query rows with a power of two each, weights with a unit to each row
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
    // NP keys of a window, which lie in one page; lane l has 1 / 8 of key l / 8 of each 8.
    const int first = 8 * NP * wave;
    auto lookup = [&](int w) {   // the entry of the wave's page; the first window begins before the sequence
      // not by a scalar load: that, on its way, would make every wait for an LDS read a wait for all of them
      return table[min(max(w * KT - 32 + first, 0) >> a.c.log2page, width - 1)];
    };
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
    uint32_t kraw[NP][D / 32], vraw[NP][D / 32];
    float ks[NP], kvs[NP], vs[NP];         // scales of the lane's keys: key and value of K's window, value of V's
    int kpage, vpage, entry;               // the wave's pages in the two windows; the entry for K's next one
    auto load_codes = [&](const uint8_t* base, int page, int w, uint32_t (&raw)[NP][D / 32]) __attribute__((always_inline)) {
      const uint8_t* at = base + (max(page, 0) * a.c.page_stride + kvh * a.c.head_stride + ((w * KT - 32 + first) & mask) * D);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if constexpr (D == 128) {
          const uint4 r = *reinterpret_cast<const uint4*>(at + (16 * lane + 8 * D * i));
          raw[i][0] = r.x; raw[i][1] = r.y; raw[i][2] = r.z; raw[i][3] = r.w;
        } else {
          const uint2 r = *reinterpret_cast<const uint2*>(at + (8 * lane + 8 * D * i));
          raw[i][0] = r.x; raw[i][1] = r.y;
        }
      }
    };
    auto load_k = [&](int w) __attribute__((always_inline)) {
      const int64_t at = max(kpage, 0) * a.c.spage_stride + kvh * a.c.shead_stride + ((w * KT - 32 + first) & mask);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        ks[i] = (a.c.ks + at)[8 * i + (lane >> 3)];
        kvs[i] = (a.c.vs + at)[8 * i + (lane >> 3)];
      }
      load_codes(a.c.k, kpage, w, kraw);
    };
    if (t0 < t1) {   // the first loads, beside those of the query rows and the scales
      kpage = page_in(scalar(lookup(t0)));
      load_k(t0);
      entry = lookup(t0 + 1);
    }
    {
      const int64_t qat = (sq.first + tok) * a.q_st + hd * a.q_sh + 8 * hi;
      float x[KS][8], top = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        load_row8<FINE ? RH3_DTYPE_F16 : RH3_DTYPE_BF16>(a.q, qat + 16 * s, x[s]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[s][e]) < INFINITY ? fabsf(x[s][e]) : 0.0f);
      }
      const float mine = across_max<false>(top);   // of the lane's row
      float least = -wave_max(mine > 0.0f ? -mine : -INFINITY);
      top = wave_max(mine);
      // the largest finite scale of the share's values, 4 keys (of one page) to a thread at a time
      float big = 0.0f, small = INFINITY;
      bool gone = false, zeros = false;
#pragma unroll 4
      for (int key = t0 * KT + 4 * static_cast<int>(threadIdx.x); key < min(t1 * KT, sq.len); key += 4 * WAVES * 64) {
        const int page = page_in(table[min(key >> a.c.log2page, width - 1)]);
        const float4 v = *reinterpret_cast<const float4*>(a.c.vs + max(page, 0) * a.c.spage_stride + kvh * a.c.shead_stride + (key & mask));
        const float x[4] = {v.x, v.y, v.z, v.w};
        gone |= page < 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = page >= 0 && key + e < sq.len && x[e] < INFINITY ? x[e] : 0.0f;
          big = fmaxf(big, y);
          small = fminf(small, y > LEAST_SCALE ? y : INFINITY);
          zeros |= y > 0.0f && y <= LEAST_SCALE;
        }
      }
      if (__builtin_amdgcn_ballot_w64(zeros)) {   // rows of zeros take no part
#pragma unroll 1
        for (int key = t0 * KT + static_cast<int>(threadIdx.x); key < min(t1 * KT, sq.len); key += WAVES * 64) {
          const int page = page_in(table[min(key >> a.c.log2page, width - 1)]);
          if (page < 0) continue;
          const float x = a.c.vs[page * a.c.spage_stride + kvh * a.c.shead_stride + (key & mask)];
          if (x > 0.0f && x <= LEAST_SCALE && codes_in<FMT, D>(a.c.v + page * a.c.page_stride + kvh * a.c.head_stride + (key & mask) * D))
            small = fminf(small, x);
        }
      }
      big = wave_max(big);
      small = -wave_max(-small);
      const int any = __builtin_amdgcn_ballot_w64(gone) != 0;
      if (lane == 0) {
        stop[wave] = top;
        sleast[wave] = least;
        sscale[wave] = big;
        ssmall[wave] = small;
        sgone[wave] = any;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        top = fmaxf(top, stop[w]);
        least = fminf(least, sleast[w]);
        big = fmaxf(big, sscale[w]);
        small = fminf(small, ssmall[w]);
        gone |= sgone[w] != 0;
      }
      full = __builtin_amdgcn_ballot_w64(gone) == 0;
      // V's reference: the largest code times its scale comes to 2^14 to 2^15; f16's range down from there is the smaller scales'
      vref = scalar(__float_as_int(pow2_over(big))) - (FINE ? 0 : (FMT == INT8 ? 8 : 6) << 23);
      apart = __builtin_amdgcn_ballot_w64(least < top * ROWS_APART || small < big * (FINE ? 0x1p-14f : 0x1p-18f)) != 0;
      const int e = q_exponent(apart ? mine : top);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        q[s] = q_f16(x[s], e);
      }
      qf = __builtin_amdgcn_ldexpf(a.scale_log2, apart ? 0 : -e);
      if (apart) {
        srow[wave * 32 + l32] = __builtin_amdgcn_ldexpf(1.0f, -e);
        sunit[wave * 32 + l32] = 0.0f;
      }
    }
    // Stage x (loaded) to LDS in 2 NP parts of K and 2 NP of V; the loads of stage x + 1
    const float vinv = apart ? 1.0f : pow2_inverse(vref);
    auto put_k = [&](int x, int part, bool apart) __attribute__((always_inline)) {
      const int i = part / 2, c = part % 2, key = first + 8 * i + (lane >> 3), h = (2 * x + 1 + (key >> 5)) & 7;
      if (c == 0 && (FINE || apart)) svs[h][key & 31] = kvs[i] < INFINITY ? kvs[i] * vinv : 0.0f;
      // a NaN value would reach rows that do not see its key (0 x NaN): its key is made NaN
      if (c == 0) sks[h][key & 31] = fmaf(kvs[i], 0.0f, ks[i] * qf);
      if (c < D / 64)
        sk[x & 1][key * K_ROW<D> + (lane & 7) * (D / 64) + c] = __builtin_bit_cast(uint4, f16x8<FMT>(kraw[i][2 * c], kraw[i][2 * c + 1]));
    };
    auto put_v = [&](int x, int part, bool apart) __attribute__((always_inline)) {
      const int i = part / 2, c = part % 2, key = first + 8 * i + (lane >> 3);
      // outside the share's keys and in an absent page there may be anything: 0 (and codes that can be NaN go)
      const int pos = x * KT - 32 + key;
      const bool here = vpage >= 0 && pos >= t0 * KT && pos < min(sq.len, t1 * KT);
      [[maybe_unused]] const _Float16 f = static_cast<_Float16>(here && vs[i] < INFINITY ? (apart ? 1.0f : vs[i] * vinv) : 0.0f);
      if (c < D / 64) {
        const bool keep = FMT == INT8 || here;
        const h8_t v = f16x8<FMT>(keep ? vraw[i][2 * c] : 0u, keep ? vraw[i][2 * c + 1] : 0u);
        if constexpr (FINE) sv[x & 1][key * V_ROW<D> + (lane & 7) * (D / 64) + c] = __builtin_bit_cast(uint4, v);
        else sv[x & 1][key * V_ROW<D> + (lane & 7) * (D / 64) + c] = __builtin_bit_cast(uint4, v * f);
      }
    };
    auto next_v = [&](int x) __attribute__((always_inline)) {   // (before next_k: the window's scales and page are K's of stage x)
#pragma unroll
      for (int i = 0; i < NP; ++i) vs[i] = kvs[i];
      vpage = kpage;
      load_codes(a.c.v, vpage, x + 1, vraw);
    };
    auto next_k = [&](int x) __attribute__((always_inline)) {
      kpage = page_in(scalar(entry));
      entry = lookup(x + 3);
      load_k(x + 2);
    };
    auto stage_v = [&](int x) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2 * NP; ++i) put_v(x, i, apart);
      next_v(x);
    };
    auto stage_k = [&](int x) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2 * NP; ++i) put_k(x, i, apart);
      next_k(x);
    };

    // Half h's softmax runs beside the products of half h + 1 and the values of half h - 1. Step s does halves 2 s and 2 s + 1 with
    // stage s.
    const f16_t zero = {};
    f16_t sa = zero, sb = zero;            // products of the next even and odd half
    h8_t p[2] = {}, pr[2] = {};   // weights of the last half, what their rounding left
    constexpr int AHEAD = 4;
    auto k_at = [&](int b, int half, int ks) { return __builtin_bit_cast(h8_t, sk[b][(32 * half + l32) * K_ROW<D> + hi + 2 * ks]); };
    const uint8_t* v_lane = reinterpret_cast<const uint8_t*>(sv) + (4 * hi + ((lane & 15) >> 2)) * V_ROW<D> * 16 + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    auto v_at = [&](int b, int half, int i) {   // i: k-step * DT + channel tile
      const uint8_t* at = v_lane + ((b * KT + 32 * half + 16 * (i / DT)) * V_ROW<D> * 16 + 64 * (i % DT));
      const h4_t lo = lds_read_tr(at), up = lds_read_tr(at + 8 * V_ROW<D> * 16);
      return __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    // Weights of two keys to f16; FINE: in two terms
    auto weights = [&](float w0, float w1, uint32_t& rest) __attribute__((always_inline)) {
      const uint32_t w = pack_h2(w0, w1);
      if constexpr (FINE) {
        const h2_t r = __builtin_bit_cast(h2_t, w);
        rest = pack_h2(w0 - static_cast<float>(r[0]), w1 - static_cast<float>(r[1]));
      }
      return w;
    };
    auto set2 = [](h8_t (&x)[2], int e, uint32_t w) __attribute__((always_inline)) {
      const h2_t r = __builtin_bit_cast(h2_t, w);
      x[e / 8][e % 8] = r[0];
      x[e / 8][e % 8 + 1] = r[1];
    };
    // Half H of step s, its softmax spread evenly over the half's MFMAs; the sum of its probabilities. `side(i)` goes with MFMA i.
    auto fast = [&](auto H, int b, int s, f16_t& now, f16_t& next, h8_t (&f)[AHEAD], float4 (&k0)[2], h8_t (&n)[2], h8_t (&nr)[2],
                    auto side) __attribute__((always_inline)) {
      constexpr int HALF = decltype(H)::value, MM = KS + 2 * DT, N = 16 / MM;
      float4 k1[2];
      [[maybe_unused]] float4 v4;   // value scales of the 4 keys at hand
      float y[N], w[16], more = 0.0f;
      auto score = [&](int e) __attribute__((always_inline)) {
        const float4 k = e < 8 ? k0[e / 4] : k1[e / 4 - 2];
        y[e % N] = fmaf(now[e], e % 4 == 0 ? k.x : e % 4 == 1 ? k.y : e % 4 == 2 ? k.z : k.w, -ref);
      };
      auto pair = [&](int e) __attribute__((always_inline)) {
        more = e == 0 ? w[0] + w[1] : more + (w[e] + w[e + 1]);
        uint32_t rest = 0;
        if constexpr (FINE) {
          if (e % 4 == 0) v4 = *reinterpret_cast<const float4*>(&svs[(2 * s + HALF) & 7][2 * e + 4 * hi]);
        }
        uint32_t bits = FINE ? weights(w[e] * (e % 4 ? v4.z : v4.x), w[e + 1] * (e % 4 ? v4.w : v4.y), rest) : weights(w[e], w[e + 1], rest);
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
        const int j = i - KS, r = i + AHEAD;
        if (i < KS) next = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i % AHEAD], q[i < KS ? i : 0], i ? next : zero, 0, 0, 0);
        else o[j & (DT - 1)] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i % AHEAD], p[(j < 0 ? 0 : j) / DT], o[j & (DT - 1)], 0, 0, 0);
        if constexpr (FINE) {
          if (i >= KS)
            o[j & (DT - 1)] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i % AHEAD], pr[(j < 0 ? 0 : j) / DT], o[j & (DT - 1)], 0, 0, 0);
        }
        if (r < KS) f[i % AHEAD] = k_at(b, HALF, r);
        else if (r < MM) f[i % AHEAD] = v_at(b, HALF, r - KS);
        else if (HALF == 0) f[i % AHEAD] = k_at(b, 1, r - MM);
        if (i == MM / 8) {
#pragma unroll
          for (int c = 0; c < 2; ++c) k1[c] = *reinterpret_cast<const float4*>(&sks[(2 * s + HALF) & 7][8 * (c + 2) + 4 * hi]);
        }
        if (HALF == 0 && i == 5 * MM / 8) {
#pragma unroll
          for (int c = 0; c < 2; ++c) k0[c] = *reinterpret_cast<const float4*>(&sks[(2 * s + 1) & 7][8 * c + 4 * hi]);
        }
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
    bool begun = false;           // the first step sets the references (rows far apart: all steps go the plain way)
    auto values = [&](int b, int half) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2 * DT; ++i) {
        const h8_t v = v_at(b, half, i);
        o[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[i / DT], o[i % DT], 0, 0, 0);
        if constexpr (FINE) o[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pr[i / DT], o[i % DT], 0, 0, 0);
      }
    };
    // Any half: keys that a row does not see hidden, the reference moved where it must be
    auto slow = [&](int b, int s, int half, bool made, f16_t& now, f16_t& next) __attribute__((always_inline)) {
      const int h = 2 * s + half;
      if (!made) {
        values(b, half);
        next = zero;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) next = __builtin_amdgcn_mfma_f32_32x32x16_f16(k_at(b, half, ks), q[ks], next, 0, 0, 0);
      }
      const int key0 = 32 * h + 4 * hi, m = lim - key0;
      uint32_t gone = 0;
      if (!there)
        gone = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(page_in(table[min((32 * h + l32) >> a.c.log2page, width - 1)]) < 0) >> (4 * hi));
      float y[16], top = -INFINITY;
      if (apart) now *= srow[wave * 32 + l32];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = 8 * (i >> 2) + (i & 3);
        y[i] = now[i] * sks[h & 7][4 * hi + key];
        y[i] = (key >= m) | ((gone >> key) & 1) ? -INFINITY : y[i];
        top = fmax_nc(top, y[i]);
      }
      top = across_max<false>(top);
      const float to = top - ref > REF_STALE ? reference_under(top) : ref;
      float f = __builtin_amdgcn_exp2f(ref - to);
      ref = to;
      sum *= f;
      // to weights; FINE or rows apart: times their values' scales (one that the row does not see may be anything)
      const float* scale = &svs[h & 7][4 * hi];
      if (apart) {
        float vtop = 0.0f, w = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) vtop = fmaxf(vtop, y[i] == -INFINITY ? 0.0f : scale[8 * (i >> 2) + (i & 3)]);
        const float base = pow2_over(across_max<false>(vtop)), ibase = pow2_inverse(__float_as_int(base));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = __builtin_amdgcn_exp2f(y[i] - to);
          sum += e;
          y[i] = e * ((y[i] == -INFINITY ? 0.0f : scale[8 * (i >> 2) + (i & 3)]) * ibase);
          w = fmaxf(w, y[i]);
        }
        float* unit = &sunit[wave * 32 + l32];
        const float now_in = weight_unit(*unit, f, across_max<false>(w), base), inv = pow2_inverse(__float_as_int(now_in));
        f *= *unit * inv;
        *unit = now_in;
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] *= base * inv;
      } else {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float e0 = __builtin_amdgcn_exp2f(y[i] - to), e1 = __builtin_amdgcn_exp2f(y[i + 1] - to);
          const float* v = scale + 8 * (i >> 2) + (i & 3);
          sum += e0 + e1;
          y[i] = FINE ? e0 * (y[i] == -INFINITY ? 0.0f : v[0]) : e0;
          y[i + 1] = FINE ? e1 * (y[i + 1] == -INFINITY ? 0.0f : v[1]) : e1;
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        uint32_t rest = 0;
        set2(p, i, weights(y[i], y[i + 1], rest));
        if constexpr (FINE) set2(pr, i, rest);
      }
    };

    auto take = [&](const h8_t (&n)[2], const h8_t (&nr)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        p[i] = n[i];
        if constexpr (FINE) pr[i] = nr[i];
      }
    };
    if (t0 < t1) {
      // stage t0 - 1 is only K of window t0
#pragma unroll
      for (int i = 0; i < 2 * NP; ++i) put_k(t0 - 1, i, apart);
      next_v(t0 - 1);
      next_k(t0 - 1);
      __syncthreads();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) sa = __builtin_amdgcn_mfma_f32_32x32x16_f16(k_at((t0 - 1) & 1, 1, ks), q[ks], sa, 0, 0, 0);
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
        h8_t f[AHEAD], n[2], nr[2];
        float4 k0[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) k0[c] = *reinterpret_cast<const float4*>(&sks[(2 * s) & 7][8 * c + 4 * hi]);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) f[i] = k_at(b, 0, i);
        __builtin_amdgcn_sched_barrier(0);
        float more = fast(std::integral_constant<int, 0>(), b, s, sa, sb, f, k0, n, nr, [&](int i) __attribute__((always_inline)) {
          if (i >= MM / 2 && i % EACH == 0) put_v(s + 1, (i - MM / 2) / EACH, false);
          if (i == MM - 1) next_v(s + 1);
        });
        staged_v = made = true;
        if (__builtin_amdgcn_ballot_w64(more > SUM_STALE)) break;   // a reference has to move
        sum += more;
        take(n, nr);
        odd = true;
        more = fast(std::integral_constant<int, 1>(), b, s, sb, sa, f, k0, n, nr, [&](int i) __attribute__((always_inline)) {
          if (i >= MM / 2 && i % EACH == 0) put_k(s + 1, (i - MM / 2) / EACH, false);
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
      }
      if (s >= t1) break;
      const int b = s & 1;
      if ((s - 1) * KT < top_key) {   // (a step past the last key that a row sees sums its last values)
        if (!odd) slow(b, s, 0, made, sa, sb);
        slow(b, s, 1, made && odd, sb, sa);
      }
      if (!staged_v) stage_v(s + 1);
      if (!staged_k) stage_k(s + 1);
      begun = !apart;
      __syncthreads();
      there = all_there(++s);
    }
    if (t0 < t1) {   // the last half's values
      values(t1 & 1, 0);
    }
    __syncthreads();   // the next item's tiles go where these are read

    // lane: query row l % 32, channels 32 d + 8 i + 4 (l / 32) + 0 .. 3
    const float total = across_sum<false>(sum);
    const float unit = apart ? sunit[wave * 32 + l32] : __int_as_float(vref);
    if (has) {
      if (whole && !a.keep) {
        const int tok = row / a.group, hd = kvh * a.group + row - tok * a.group;
        const float inv = total == 0.0f ? 0.0f : unit / total;
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
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(po + 32 * d + 8 * i) =
                make_float4(o[d][4 * i] * PART * unit, o[d][4 * i + 1] * PART * unit, o[d][4 * i + 2] * PART * unit,
                            o[d][4 * i + 3] * PART * unit);
        if (hi == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * R + rl) * 2) = make_float2(total == 0.0f ? -INFINITY : ref, total);
      }
    }
  }
}

}  // namespace

void launch_chunk(const AttnArgs& a, int fmt, int dim, int rows, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(a.wgs)), dim3(static_cast<uint32_t>(2 * rows)), 0, st, a); };
  auto by = [&](auto four, auto eight, auto four_fine, auto eight_fine) {
    if (rows == 128) a.fp16 ? go(four_fine) : go(four);
    else a.fp16 ? go(eight_fine) : go(eight);
  };
  if (fmt == INT8 && dim == 128)
    by(chunk_kernel<INT8, 128, 4, false>, chunk_kernel<INT8, 128, 8, false>, chunk_kernel<INT8, 128, 4, true>, chunk_kernel<INT8, 128, 8, true>);
  else if (fmt == INT8)
    by(chunk_kernel<INT8, 64, 4, false>, chunk_kernel<INT8, 64, 8, false>, chunk_kernel<INT8, 64, 4, true>, chunk_kernel<INT8, 64, 8, true>);
  else if (dim == 128)
    by(chunk_kernel<E4M3, 128, 4, false>, chunk_kernel<E4M3, 128, 8, false>, chunk_kernel<E4M3, 128, 4, true>, chunk_kernel<E4M3, 128, 8, true>);
  else
    by(chunk_kernel<E4M3, 64, 4, false>, chunk_kernel<E4M3, 64, 8, false>, chunk_kernel<E4M3, 64, 4, true>, chunk_kernel<E4M3, 64, 8, true>);
}

}  // namespace kv
}  // namespace rh3
