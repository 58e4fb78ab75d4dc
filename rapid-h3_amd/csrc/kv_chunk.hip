// Attention of many query rows over the paged cache: a chunk of a prompt, the tokens of a frame, a whole batch against a prefix
// that it shares.
//
// Bound by the matrix units and, close behind, by the vector instructions of the softmax: 4 dim flops per query row and key,
// while a key's 2 (dim + 4) bytes serve all rows of a tile. A workgroup of 4 or 8 waves holds 32 query rows of one K/V head on
// each and walks its keys 64 at a time. The tile's codes come to registers while the previous tile is computed, are converted to
// f16 once for all waves and written to LDS (two buffers, one barrier to a tile): K as it is, V channel-major with its keys in
// the order that the probabilities have. Per wave
//   S^T = K Q^T (32x32x16 f16): a lane has one query row (l % 32) and 16 of 32 keys, so a row's softmax is in-lane but for one
//   exchange, and only when its reference moves; the probabilities are the B operand of
//   O^T = V^T P^T as they stand: k-step t of 32 keys takes keys 16 t + 4 (l / 32) + 0 .. 3 and those + 8.
// Vector work per score: one fma (key scale, softmax scale and reference at once), half a max, the exponential, the sum and half a
// conversion. For that, the query rows of a workgroup share one power of
// two (an element 2^22 below the tile's largest loses low bits, 2^-33 of the largest at most, which is what an absolute error
// of a score can be); and a value's scale, relative to a power of two over the largest seen, is multiplied into V as it is
// converted (rounded to f16, 2^-11 at most, as the probabilities are).
#include "kv_attn.hpp"

namespace rh3 {
namespace kv {
namespace {

constexpr int KT = CHUNK_KEYS;
constexpr float NO_REF = -0x1p100f;   // reference of a row that has seen no key: any score moves it

// 16-byte pieces of the LDS rows. Each row has one piece more than it needs, so that 16 rows' pieces of one number lie in all 16
// parts of the banks, and every read of a tile is one lane address with an immediate offset.
template <int D>
constexpr int K_ROW = D / 8 + 1;                               // K: [64 keys][D] f16
constexpr int V_ROW = KT / 8 + 1;                              // V^T: [D][64 keys] f16, pieces of 8 keys

// What a wave has in flight of a tile: the codes that it will convert, and of key l of the 64 its scales and table entry. With 8
// waves a wave has keys or values, in the same registers.
template <int D, int WAVES>
struct Stage {
  static constexpr int KW = D / 16, VAT = WAVES == 4 ? KW : 0;
  uint32_t raw[VAT + 8];       // words of 16 keys (KW), of 8 keys x 4 channels (8 from VAT)
  float vs, ks;
  int entry;
};

template <int FMT, int D, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, 2) chunk_kernel(AttnArgs a) {
  constexpr int R = WAVES * 32, KS = D / 16, DT = D / 32;
  const Tiling TILING = tiling(true, R);
  __shared__ uint4 sk[2][KT * K_ROW<D>];
  __shared__ uint4 sv[2][D * V_ROW];
  __shared__ float sks[2][KT];
  __shared__ uint4 sf[WAVES][KT / 8];   // a wave's value scales as f16, in V's key order
  __shared__ float stop[WAVES];
  const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // of the 64 keys, a wave converts 16 keys and 16 values (4 waves), or 16 of either (8 waves: the first four keys)
  const int part = wave & 3;
  const bool does_k = WAVES == 4 || wave < 4, does_v = WAVES == 4 || wave >= 4;

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
      if (blk.at + 64 >= a.s.batch) return;
      next_block(a, TILING, blk);
    }
    const int in_block = __builtin_ctzll(__builtin_amdgcn_ballot_w64(blk.base + blk.units > u));
    const int seq = blk.at + in_block;
    const SeqItems sw = seq_in(a, blk, in_block);
    const Seq sq = sw.seq;
    const int64_t local = u - sw.before;
    const int item = scalar(static_cast<int>(quotient(local, sw.key_tiles)));
    const int t0 = static_cast<int>(local - static_cast<int64_t>(item) * sw.key_tiles);
    const int share_t1 = static_cast<int>(end - u < sw.key_tiles - t0 ? t0 + (end - u) : sw.key_tiles);
    const bool whole = t0 == 0 && share_t1 == sw.key_tiles;
    const int kvh = scalar(item / sw.row_tiles), at = item - kvh * sw.row_tiles;
    const int rt = a.causal ? tile_at_place(at, sw.row_tiles) : at;
    const int rows = sq.n * a.group;
    const int tok_last = scalar(min(rows - 1, rt * R + R - 1) / a.group);
    const int seen = a.causal ? min(sq.len, max(0, sq.len - sq.n + tok_last + 1)) : sq.len;   // keys that some row sees
    const int t1 = min(share_t1, (seen + KT - 1) / KT);

    const int row = rt * R + wave * 32 + l32;
    const bool has = row < rows;
    const int rr = has ? row : rows - 1;
    const int tok = rr / a.group, hd = kvh * a.group + rr - tok * a.group;
    h8_t q[KS];
    float qf;
    {
      const int64_t qat = (sq.first + tok) * a.q_st + hd * a.q_sh + 8 * hi;
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        float x[8];
        load_q8(a, qat + 16 * s, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.0f);
      }
      top = wave_max(top);
      if (lane == 0) stop[wave] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stop[w]);
      const int e = q_exponent(top);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        float x[8];
        load_q8(a, qat + 16 * s, x);
        q[s] = q_f16(x, e);
      }
      qf = __builtin_amdgcn_ldexpf(a.scale_log2, -e);
    }
    const int lim = a.causal ? min(sq.len, sq.len - sq.n + tok + 1) : sq.len;
    // of the wave's rows: keys that all see, keys that some see
    const int r0 = rt * R + wave * 32, r1 = min(rows - 1, r0 + 31);
    const int low = a.causal ? min(sq.len, sq.len - sq.n + scalar(r0 / a.group) + 1) : sq.len;
    const int top_key = r0 >= rows ? 0 : a.causal ? min(sq.len, sq.len - sq.n + scalar(r1 / a.group) + 1) : sq.len;

    f16_t o[DT];
    float ref = NO_REF, sum = 0.0f;
    int vref = -1;   // bits of the values' reference, the same in all lanes; no tile has that of -1: the first one is never fast
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

    const int32_t* table = a.s.table + seq * a.s.table_stride;
    const int mask = (1 << a.c.log2page) - 1;
    auto lookup = [&](int t) {   // table entry of key l of tile t
      return table[min((t * KT + lane) >> a.c.log2page, a.s.width - 1)];
    };
    // V: a thread takes 4 channels of the 8 keys of one piece; D 64: the first 16 lanes of each half
    const int vq = lane & (D / 4 - 1);
    const bool vmine = D == 128 || (lane & 16) == 0;
    using St = Stage<D, WAVES>;
    auto page_in = [&](int entry) { return entry >= 0 && entry < a.c.pages ? entry : -1; };
    auto load = [&](St& s, int t) {   // s.entry: of this tile
      const int page = page_in(s.entry);
      const int64_t pl = max(page, 0);
      const int64_t at = pl * a.c.spage_stride + kvh * a.c.shead_stride + ((t * KT + lane) & mask);
      s.vs = a.c.vs[at];
      s.ks = a.c.ks[at];
      const int64_t p = max(__builtin_amdgcn_readlane(page, 16 * part), 0);
      const int64_t code = p * a.c.page_stride + kvh * a.c.head_stride + ((t * KT + 16 * part) & mask) * D;
      if (does_k) {
        const uint8_t* kb = a.c.k + code;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const uint4 w = *reinterpret_cast<const uint4*>(kb + (64 * c + lane) * 16);
          s.raw[4 * c] = w.x; s.raw[4 * c + 1] = w.y; s.raw[4 * c + 2] = w.z; s.raw[4 * c + 3] = w.w;
        }
      }
      if (does_v) {
        const uint8_t* vb = a.c.v + code;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          s.raw[St::VAT + j] = *reinterpret_cast<const uint32_t*>(vb + (4 * hi + (j & 3) + 8 * (j >> 2)) * D + 4 * vq);
      }
    };
    int nvref = 0;   // that of the tile converted last
    bool absent = false;
    auto store = [&](St& s, int t, int buf) {
      const int page = page_in(s.entry);
      const bool here = t * KT + lane < sq.len && page >= 0;
      absent = __builtin_amdgcn_ballot_w64(page < 0) != 0;
      // a NaN value would reach rows that do not see its key (0 x NaN): its key is made NaN, its codes 0
      if (wave == 0) sks[buf][lane] = fmaf(s.vs, 0.0f, s.ks * qf);
      const float vs = here && s.vs < INFINITY ? s.vs : 0.0f;
      // The reference is such that the largest code times its scale comes to 2^14 to 2^15: f16's range down from there is the
      // smaller scales'. A float that is not negative is ordered like its bits.
      constexpr int HEAD = (FMT == INT8 ? 8 : 6) << 23;
      if (__builtin_amdgcn_ballot_w64(__float_as_int(vs) > (nvref ? nvref + HEAD : 0)))
        nvref = max(nvref, scalar(__float_as_int(pow2_over(wave_max(vs)))) - HEAD);
      if (does_k) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const int e = 64 * c + lane;                      // 16-byte piece of the 16 keys
          const int key = 16 * part + e / (D / 16), piece = 2 * (e % (D / 16));
          sk[buf][key * K_ROW<D> + piece] = __builtin_bit_cast(uint4, f16x8<FMT>(s.raw[4 * c], s.raw[4 * c + 1]));
          sk[buf][key * K_ROW<D> + piece + 1] = __builtin_bit_cast(uint4, f16x8<FMT>(s.raw[4 * c + 2], s.raw[4 * c + 3]));
        }
      }
      if (does_v) {
        // scales through LDS from a key to a lane to the 8 keys of a piece
        reinterpret_cast<_Float16*>(sf[wave])[(lane >> 4) * 16 + ((lane >> 2) & 1) * 8 + (lane & 3) + ((lane >> 3) & 1) * 4] =
            static_cast<_Float16>(nvref > 0 ? vs * pow2_inverse(nvref) : 0.0f);
        asm volatile("" ::: "memory");   // a wave's LDS accesses are in order; the compiler keeps this one
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = s.raw[St::VAT + j];
        if constexpr (FMT == E4M3) {   // behind the sequence there may be NaN codes
          if (t * KT + 16 * part + 16 > sq.len || __builtin_amdgcn_readlane(page, 16 * part) < 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (__builtin_amdgcn_readlane(page, 16 * part) < 0 || t * KT + 16 * part + 4 * hi + (j & 3) + 8 * (j >> 2) >= sq.len) w[j] = 0u;
          }
        }
        h8_t v[4];
        f16x8_across<FMT>(w, v);
        const h8_t f = __builtin_bit_cast(h8_t, sf[wave][2 * part + hi]);
        if (vmine) {
#pragma unroll
          for (int c = 0; c < 4; ++c) sv[buf][(4 * vq + c) * V_ROW + 2 * part + hi] = __builtin_bit_cast(uint4, v[c] * f);
        }
      }
    };

    St stage;
    int entry_next = 0;   // looked at a tile later, when the load has come
    if (t0 < t1) {
      stage.entry = lookup(t0);
      load(stage, t0);
      entry_next = lookup(t0 + 1);
      store(stage, t0, 0);
    }

    const f16_t zero = {};
    auto probabilities = [&](const float* y) __attribute__((always_inline)) {   // of 8 keys, added to the sum
      h2_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = __builtin_amdgcn_exp2f(y[2 * e]), p1 = __builtin_amdgcn_exp2f(y[2 * e + 1]);
        sum += p0 + p1;
        w[e] = __builtin_bit_cast(h2_t, pack_h2(p0, p1));
      }
      return join(w[0], w[1], w[2], w[3]);
    };
    // Any tile: keys that a row does not see (from `most` on, or absent: gone) hidden, the reference moved where it must be
    auto slow = [&](int buf, int most, unsigned long long gone) {
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        float y[16];
        const uint4* kp = &sk[buf][(32 * h + l32) * K_ROW<D> + hi];
        const uint4* vp = &sv[buf][l32 * V_ROW + 4 * h + hi];
        f16_t s = zero;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, kp[2 * ks]), q[ks], s, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = s[i] * sks[buf][32 * h + 8 * (i >> 2) + 4 * hi + (i & 3)];
        const int m = most - 32 * h - 4 * hi;
        const uint32_t g = static_cast<uint32_t>(gone >> (32 * h + 4 * hi));
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = 8 * (i >> 2) + (i & 3);
          y[i] = (key >= m) | ((g >> key) & 1) ? -INFINITY : y[i];
          top = fmax_nc(top, y[i]);
        }
        top = across_max<false>(top);
        const float now = top > ref + REF_STALE ? top - REF_UNDER : ref;
        const float f = __builtin_amdgcn_exp2f(ref - now);
        ref = now;
        sum *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= f;
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] -= now;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const h8_t p = probabilities(y + 8 * c);
#pragma unroll
          for (int d = 0; d < DT; ++d)
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, vp[32 * d * V_ROW + 2 * c]), p, o[d], 0, 0, 0);
        }
      }
    };
    // Each wave meets one barrier to a tile, whichever way it takes through it. The fast tiles are a loop of their own, which
    // keeps the accumulators in place.
    __syncthreads();
    int t = t0;
    while (t < t1) {
      bool loaded = false;
      auto ahead = [&]() __attribute__((always_inline)) {
        if (t + 1 < t1) {
          stage.entry = entry_next;
          entry_next = lookup(t + 2);
          load(stage, t + 1);
        }
      };
      // tiles whose every key every row sees
      while (t + 1 < t1 && t * KT + KT <= low && nvref == vref && !absent) {
        ahead();
        const int buf = (t - t0) & 1;
        const uint4* kp = &sk[buf][l32 * K_ROW<D> + hi];
        const uint4* vp = &sv[buf][l32 * V_ROW + hi];
        const float4* sp = reinterpret_cast<const float4*>(&sks[buf][4 * hi]);
        // Each MFMA's operand is read four MFMAs (128 cycles) before it; left alone, the compiler puts every read right before its
        // use. Only vector and scalar arithmetic moves past a step's end.
        constexpr int AHEAD = 4, ARITH = 0x2 | 0x4 | 0x400;
        float4 kv[8];
        h8_t f[AHEAD];
        f16_t s[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) kv[i] = sp[2 * i];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) f[i] = __builtin_bit_cast(h8_t, kp[2 * i]);
        __builtin_amdgcn_sched_barrier(ARITH);
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) {
          const int h = i / KS, ks = i % KS, n = i + AHEAD;
          s[h] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i % AHEAD], q[ks], ks ? s[h] : zero, 0, 0, 0);
          if (n < 2 * KS) f[i % AHEAD] = __builtin_bit_cast(h8_t, kp[32 * (n / KS) * K_ROW<D> + 2 * (n % KS)]);
          else kv[4 + n - 2 * KS] = sp[8 + 2 * (n - 2 * KS)];
          __builtin_amdgcn_sched_barrier(ARITH);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) f[i] = __builtin_bit_cast(h8_t, vp[32 * (i % DT) * V_ROW + 2 * (i / DT)]);
        float y[32], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[4 * i] = fmaf(s[i / 4][4 * (i % 4)], kv[i].x, -ref);
          y[4 * i + 1] = fmaf(s[i / 4][4 * (i % 4) + 1], kv[i].y, -ref);
          y[4 * i + 2] = fmaf(s[i / 4][4 * (i % 4) + 2], kv[i].z, -ref);
          y[4 * i + 3] = fmaf(s[i / 4][4 * (i % 4) + 3], kv[i].w, -ref);
          top = max3(max3(top, y[4 * i], y[4 * i + 1]), y[4 * i + 2], y[4 * i + 3]);
        }
        if (__builtin_amdgcn_ballot_w64(top > REF_STALE)) {   // a reference has to move: the slow way
          loaded = true;
          break;
        }
        h8_t p;
#pragma unroll
        for (int i = 0; i < 4 * DT; ++i) {
          const int c = i / DT, d = i % DT, n = i + AHEAD;
          if (d == 0) p = probabilities(y + 8 * c);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i % AHEAD], p, o[d], 0, 0, 0);
          if (n < 4 * DT) f[i % AHEAD] = __builtin_bit_cast(h8_t, vp[32 * (n % DT) * V_ROW + 2 * (n / DT)]);
          __builtin_amdgcn_sched_barrier(ARITH);
        }
        store(stage, t + 1, (t - t0 + 1) & 1);
        __syncthreads();
        ++t;
      }
      if (!loaded) ahead();
      if (t * KT < top_key) {
        if (nvref != vref) {
          const float f = vref > 0 ? __int_as_float(vref) * pow2_inverse(nvref) : 0.0f;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d] *= f;
          vref = nvref;
        }
        slow((t - t0) & 1, lim - t * KT, absent ? __builtin_amdgcn_ballot_w64(page_in(lookup(t)) < 0) : 0ull);
      }
      if (t + 1 < t1) store(stage, t + 1, (t - t0 + 1) & 1);
      __syncthreads();
      ++t;
    }

    // lane: query row l % 32, channels 32 d + 8 i + 4 (l / 32) + 0 .. 3
    const float total = across_sum<false>(sum);
    if (has) {
      if (whole && !a.keep) {
        const int tok = row / a.group, hd = kvh * a.group + row - tok * a.group;
        const float inv = total == 0.0f ? 0.0f : __int_as_float(max(vref, 0)) / total;
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
        const float vf = __int_as_float(max(vref, 0));
        float* po = a.part_o + (slot * R + rl) * D + 4 * hi;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(po + 32 * d + 8 * i) =
                make_float4(o[d][4 * i] * vf, o[d][4 * i + 1] * vf, o[d][4 * i + 2] * vf, o[d][4 * i + 3] * vf);
        if (hi == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * R + rl) * 2) = make_float2(total == 0.0f ? -INFINITY : ref, total);
      }
    }
    u += share_t1 - t0;
  }
}

}  // namespace

void launch_chunk(const AttnArgs& a, int fmt, int dim, int rows, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(a.wgs)), dim3(static_cast<uint32_t>(2 * rows)), 0, st, a); };
  if (fmt == INT8 && dim == 128) rows == 128 ? go(chunk_kernel<INT8, 128, 4>) : go(chunk_kernel<INT8, 128, 8>);
  else if (fmt == INT8) rows == 128 ? go(chunk_kernel<INT8, 64, 4>) : go(chunk_kernel<INT8, 64, 8>);
  else if (dim == 128) rows == 128 ? go(chunk_kernel<E4M3, 128, 4>) : go(chunk_kernel<E4M3, 128, 8>);
  else rows == 128 ? go(chunk_kernel<E4M3, 64, 4>) : go(chunk_kernel<E4M3, 64, 8>);
}

}  // namespace kv
}  // namespace rh3
