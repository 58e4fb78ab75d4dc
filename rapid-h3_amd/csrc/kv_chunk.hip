// Attention of many query rows over the paged cache: a chunk of a prompt, the tokens of a frame, a whole batch against a prefix
// that it shares.
//
// Bound by the matrix units: 4 dim flops per query row and key, while a key's 2 (dim + 4) bytes serve all rows of a tile. A
// workgroup of 4 waves holds 4 x 32 QT query rows of one K/V head and walks its keys 64 at a time. The tile's codes come to
// registers while the previous tile is computed, are converted to f16 once for the 4 waves and written to LDS (two buffers, one
// barrier to a tile): K as it is, V channel-major with its keys in the order that the probabilities have. Per wave
//   S^T = K Q^T (32x32x16 f16): a lane has one query row (l % 32) and 16 of 32 keys, so a row's softmax is in-lane but for one
//   exchange, and only when its reference moves; the probabilities are the B operand of
//   O^T = V^T P^T as they stand: k-step t of 32 keys takes keys 16 t + 4 (l / 32) + 0 .. 3 and those + 8.
// A value's scale, relative to a power of two over the largest seen, is multiplied into V as it is converted (rounded to f16,
// 2^-12, as the probabilities are), which leaves only the key's scale to be read per score.
#include "kv_attn.hpp"

namespace rh3 {
namespace kv {
namespace {

constexpr int NT = 256, WAVES = 4, KT = 64;

// 16-byte pieces of the LDS rows, spread so that the lanes of a read or write meet different banks
template <int D>
__device__ __forceinline__ int k_piece(int key, int piece) {   // K: [64 keys][D] f16
  constexpr int N = D / 8;
  return key * N + (piece ^ (D == 128 ? key & 15 : (key >> 1) & 7));
}
__device__ __forceinline__ int v_piece(int d, int piece) {     // V^T: [D][64 keys] f16, pieces of 8 keys
  return d * 8 + (piece ^ (((d >> 1) ^ (d >> 4)) & 7));
}

template <int D>
struct Stage {
  uint4 k[D / 64];     // the wave's 16 keys
  uint32_t v[8];       // 8 keys x 4 channels
  float4 vs0, vs1;     // their scales
  float vsl, ksl;      // scales of key l of the 64
  int page;            // page of key l, -1 where absent
};

template <int FMT, int D, int QT>
__global__ void __launch_bounds__(NT, QT == 1 ? 2 : 1) chunk_kernel(AttnArgs a) {
  constexpr int R = WAVES * 32 * QT, KS = D / 16, DT = D / 32;
  __shared__ uint4 sk[2][KT * D / 8];
  __shared__ uint4 sv[2][KT * D / 8];
  __shared__ float sks[2][KT];
  const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // the item: row tiles of all sequences in order, for each K/V head, each in `splits` key ranges. The last row tiles go first
  // (causal: they have the most keys). A K/V head's items are 8 apart in the grid where heads allow, so that one XCD's L2 holds it.
  const int idx = blockIdx.x;
  const int kvh = idx % a.c.heads;
  const int rest = idx / a.c.heads;
  const int split = rest % a.splits;
  const int tile = a.tiles - 1 - rest / a.splits;
  int b = -1, rt = 0;
  {
    int64_t base = 0;
    for (int at = 0; at < a.s.batch && b < 0; at += 64) {
      int64_t n = 0;
      if (at + lane < a.s.batch) n = (static_cast<int64_t>(seq_at(a.s, at + lane).n) * a.group + R - 1) / R;
      const int64_t s = wave_scan(n);
      const unsigned long long m = __builtin_amdgcn_ballot_w64(base + s > tile);
      if (m) {
        const int l = __builtin_ctzll(m);
        b = __builtin_amdgcn_readfirstlane(at + l);
        rt = __builtin_amdgcn_readfirstlane(static_cast<int>(tile - base - __shfl(s - n, l)));
      }
      base += __shfl(s, 63);
    }
  }
  if (b < 0) return;
  const Seq sq = seq_at(a.s, b);
  const int rows = sq.n * a.group;
  const int tok_last = min(rows - 1, rt * R + R - 1) / a.group;
  const int seen = a.causal ? min(sq.len, max(0, sq.len - sq.n + tok_last + 1)) : sq.len;   // keys that some row sees
  const int nkt = (seen + KT - 1) / KT;
  const int per = (nkt + a.splits - 1) / a.splits;
  const int t0 = min(nkt, split * per), t1 = min(nkt, t0 + per);

  h8_t q[QT][KS];
  float qf[QT];
  int lim[QT], row_of[QT];
#pragma unroll
  for (int m = 0; m < QT; ++m) {
    const int row = rt * R + wave * 32 * QT + 32 * m + l32;
    const bool has = row < rows;
    const int rr = has ? row : rows - 1;
    const int tok = rr / a.group, hd = kvh * a.group + rr - tok * a.group;
    const int64_t at = (sq.first + tok) * a.q_st + hd * a.q_sh + 8 * hi;
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8];
      load_q8(a, at + 16 * s, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
    }
    const int e = q_exponent(across_max<false>(top));
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8];
      load_q8(a, at + 16 * s, x);
      q[m][s] = q_f16(x, e);
    }
    qf[m] = __builtin_amdgcn_ldexpf(a.scale_log2, -e);
    lim[m] = a.causal ? min(sq.len, sq.len - sq.n + tok + 1) : sq.len;
    row_of[m] = has ? row : -1;
  }
  // of the wave's rows: keys that all see, keys that some see
  const int r0 = rt * R + wave * 32 * QT, r1 = min(rows - 1, r0 + 32 * QT - 1);
  const bool idle = r0 >= rows;
  const int low = a.causal ? min(sq.len, sq.len - sq.n + r0 / a.group + 1) : sq.len;
  const int top_key = idle ? 0 : a.causal ? min(sq.len, sq.len - sq.n + r1 / a.group + 1) : sq.len;

  f16_t o[QT][DT];
  float ref[QT], sum[QT], vref = 0.0f, ivref = 0.0f;
#pragma unroll
  for (int m = 0; m < QT; ++m) {
    ref[m] = -INFINITY;
    sum[m] = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[m][d][i] = 0.0f;
  }

  const int32_t* table = a.s.table + b * a.s.table_stride;
  const int mask = (1 << a.c.log2page) - 1;
  auto lookup = [&](int t) {   // page of key l of tile t
    const int p = table[min((t * KT + lane) >> a.c.log2page, a.s.width - 1)];
    return p >= 0 && p < a.c.pages ? p : -1;
  };
  // V: a thread takes 4 channels of the 8 keys of one piece; D 64: the first 16 lanes of each half
  const int vq = lane & (D / 4 - 1);
  const bool vmine = D == 128 || (lane & 16) == 0;
  auto load = [&](Stage<D>& s, int t, int page) {
    s.page = page;
    const int64_t pl = max(page, 0);
    const int offl = (t * KT + lane) & mask;
    const int64_t sl = pl * a.c.spage_stride + kvh * a.c.shead_stride + offl;
    s.vsl = a.c.vs[sl];
    s.ksl = a.c.ks[sl];
    const int64_t p = max(__builtin_amdgcn_readlane(page, 16 * wave), 0);
    const int off = (t * KT + 16 * wave) & mask;
    const int64_t code = p * a.c.page_stride + kvh * a.c.head_stride + off * D;
    const uint8_t* kb = a.c.k + code;
    const uint8_t* vb = a.c.v + code;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) s.k[c] = *reinterpret_cast<const uint4*>(kb + (64 * c + lane) * 16);
    const float* sb = a.c.vs + p * a.c.spage_stride + kvh * a.c.shead_stride + off + 4 * hi;
    s.vs0 = *reinterpret_cast<const float4*>(sb);
    s.vs1 = *reinterpret_cast<const float4*>(sb + 8);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      s.v[j] = *reinterpret_cast<const uint32_t*>(vb + (4 * hi + (j & 3) + 8 * (j >> 2)) * D + 4 * vq);
  };
  // codes to f16 in LDS; returns the values' reference of this tile and whether a page is absent
  float nvref = 0.0f;
  bool absent = false;
  auto store = [&](Stage<D>& s, int t, int buf) {
    const bool here = t * KT + lane < sq.len && s.page >= 0;
    absent = __builtin_amdgcn_ballot_w64(s.page < 0) != 0;
    const float vt = wave_max(here && s.vsl < INFINITY ? s.vsl : 0.0f);
    // so that the largest code times its scale comes to 2^14 to 2^15: f16's range down from there is the smaller scales'
    const float over = pow2_over(vt) * (FMT == INT8 ? 0x1p-8f : 0x1p-6f);
    nvref = vt > 0.0f && nvref < over ? over : nvref;
    const float iv = nvref > 0.0f ? 1.0f / nvref : 0.0f;
    // a NaN value would reach rows that do not see its key (0 x NaN): its key is made NaN, its codes 0
    if (wave == 0) sks[buf][lane] = fmaf(s.vsl, 0.0f, s.ksl);
    float vs[8] = {s.vs0.x, s.vs0.y, s.vs0.z, s.vs0.w, s.vs1.x, s.vs1.y, s.vs1.z, s.vs1.w};
    const int page = __builtin_amdgcn_readlane(s.page, 16 * wave);
    if (t * KT + 16 * wave + 16 > sq.len || page < 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (page < 0 || t * KT + 16 * wave + 4 * hi + (j & 3) + 8 * (j >> 2) >= sq.len) {
          vs[j] = 0.0f;
          s.v[j] = 0u;
        }
    }
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const int e = 64 * c + lane;                      // 16-byte piece of the wave's 16 keys
      const int key = 16 * wave + e / (D / 16), piece = 2 * (e % (D / 16));
      sk[buf][k_piece<D>(key, piece)] = __builtin_bit_cast(uint4, f16x8<FMT>(s.k[c].x, s.k[c].y));
      sk[buf][k_piece<D>(key, piece + 1)] = __builtin_bit_cast(uint4, f16x8<FMT>(s.k[c].z, s.k[c].w));
    }
    if (vmine) {
      h8_t v[4], f;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = static_cast<_Float16>(fmaxf(vs[j] * iv, 0.0f));
      f16x8_across<FMT>(s.v, v);
#pragma unroll
      for (int c = 0; c < 4; ++c) sv[buf][v_piece(4 * vq + c, 2 * wave + hi)] = __builtin_bit_cast(uint4, v[c] * f);
    }
  };

  Stage<D> stage;
  int page_next = 0;
  if (t0 < t1) {
    load(stage, t0, lookup(t0));
    page_next = lookup(t0 + 1);
    store(stage, t0, 0);
  }
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    const bool more = t + 1 < t1;
    const float tile_vref = nvref;
    const bool tile_absent = absent;
    const int pages_now = stage.page;
    if (more) {
      load(stage, t + 1, page_next);
      page_next = lookup(t + 2);
    }
    if (t * KT < top_key) {
      const bool edge = t * KT + KT > low || tile_absent;
      if (tile_vref != vref) {
        const float f = vref / tile_vref;
#pragma unroll
        for (int m = 0; m < QT; ++m)
#pragma unroll
          for (int d = 0; d < DT; ++d) o[m][d] *= f;
        vref = tile_vref;
      }
      unsigned long long gone = 0;
      if (edge) gone = __builtin_amdgcn_ballot_w64(pages_now < 0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f16_t s[QT];
#pragma unroll
        for (int m = 0; m < QT; ++m)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[m][i] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const h8_t k = __builtin_bit_cast(h8_t, sk[buf][k_piece<D>(32 * h + l32, 2 * ks + hi)]);
#pragma unroll
          for (int m = 0; m < QT; ++m) s[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[m][ks], s[m], 0, 0, 0);
        }
        float top[QT];
        bool move = false;
#pragma unroll
        for (int m = 0; m < QT; ++m) top[m] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 kv = *reinterpret_cast<const float4*>(&sks[buf][32 * h + 8 * i + 4 * hi]);
          const float ks4[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
          for (int m = 0; m < QT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float x = s[m][4 * i + j] * (ks4[j] * qf[m]);
              if (edge) {
                const int key = 32 * h + 8 * i + 4 * hi + j;
                if (t * KT + key >= lim[m] || ((gone >> key) & 1)) x = -INFINITY;
              }
              s[m][4 * i + j] = x;
              top[m] = fmaxf(top[m], x);
            }
        }
#pragma unroll
        for (int m = 0; m < QT; ++m) move |= top[m] > ref[m] + REF_STALE;
        if (__builtin_amdgcn_ballot_w64(move)) {
#pragma unroll
          for (int m = 0; m < QT; ++m) {
            const float n = across_max<false>(top[m]);
            if (n > ref[m] + REF_STALE) {
              const float f = __builtin_amdgcn_exp2f(ref[m] - (n - REF_UNDER));
              ref[m] = n - REF_UNDER;
              sum[m] *= f;
#pragma unroll
              for (int d = 0; d < DT; ++d) o[m][d] *= f;
            }
          }
        }
        h8_t p[QT][2];
#pragma unroll
        for (int m = 0; m < QT; ++m) {
          const float r = ref[m] == -INFINITY ? 0.0f : ref[m];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            s[m][i] = __builtin_amdgcn_exp2f(s[m][i] - r);
            sum[m] += s[m][i];
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = pack_h2(s[m][8 * c + 2 * e], s[m][8 * c + 2 * e + 1]);
            p[m][c] = join(__builtin_bit_cast(h2_t, w[0]), __builtin_bit_cast(h2_t, w[1]), __builtin_bit_cast(h2_t, w[2]),
                           __builtin_bit_cast(h2_t, w[3]));
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const h8_t v = __builtin_bit_cast(h8_t, sv[buf][v_piece(32 * d + l32, 4 * h + 2 * c + hi)]);
#pragma unroll
            for (int m = 0; m < QT; ++m) o[m][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[m][c], o[m][d], 0, 0, 0);
          }
      }
    }
    if (more) store(stage, t + 1, buf ^ 1);
    __syncthreads();
  }

  // lane: query row l % 32, channels 32 d + 8 i + 4 (l / 32) + 0 .. 3
#pragma unroll
  for (int m = 0; m < QT; ++m) {
    const float total = across_sum<false>(sum[m]);
    if (row_of[m] < 0) continue;
    if (a.splits == 1 && !a.keep) {
      const int tok = row_of[m] / a.group, hd = kvh * a.group + row_of[m] - tok * a.group;
      const float inv = total == 0.0f ? 0.0f : vref / total;
      uint16_t* dst = static_cast<uint16_t*>(a.out) + (sq.first + tok) * a.o_st + hd * a.o_sh + 4 * hi;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint2*>(dst + 32 * d + 8 * i) = make_uint2(pack_out(a, o[m][d][4 * i] * inv, o[m][d][4 * i + 1] * inv),
                                                                    pack_out(a, o[m][d][4 * i + 2] * inv, o[m][d][4 * i + 3] * inv));
      if (a.lse && hi == 0)
        a.lse[static_cast<int64_t>(sq.first + tok) * a.c.heads * a.group + hd] =
            total == 0.0f ? -INFINITY : (__builtin_amdgcn_logf(total) + ref[m]) * 0.6931471805599453f;
    } else {
      const int64_t slot = (static_cast<int64_t>(kvh) * a.tiles + tile) * a.splits + split;
      const int rl = row_of[m] - rt * R;
      float* po = a.part_o + (slot * R + rl) * D + 4 * hi;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(po + 32 * d + 8 * i) = make_float4(o[m][d][4 * i] * vref, o[m][d][4 * i + 1] * vref,
                                                                     o[m][d][4 * i + 2] * vref, o[m][d][4 * i + 3] * vref);
      if (hi == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * R + rl) * 2) = make_float2(ref[m], total);
    }
  }
}

}  // namespace

void launch_chunk(const AttnArgs& a, int fmt, int dim, int rows, int64_t grid, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(grid)), dim3(NT), 0, st, a); };
  if (fmt == INT8 && dim == 128) rows == 128 ? go(chunk_kernel<INT8, 128, 1>) : go(chunk_kernel<INT8, 128, 2>);
  else if (fmt == INT8) rows == 128 ? go(chunk_kernel<INT8, 64, 1>) : go(chunk_kernel<INT8, 64, 2>);
  else if (dim == 128) rows == 128 ? go(chunk_kernel<E4M3, 128, 1>) : go(chunk_kernel<E4M3, 128, 2>);
  else rows == 128 ? go(chunk_kernel<E4M3, 64, 1>) : go(chunk_kernel<E4M3, 64, 2>);
}

}  // namespace kv
}  // namespace rh3
