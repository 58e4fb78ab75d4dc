// The RMS norm of each query and key head with its position rotation, in one pass over the rows; and the same on the way into the
// paged cache, with the keys and values quantised where they lie: no key is written and read in between.
//
// A row x of a head (dim channels): y = (x * r) * w, r = 1 / sqrt(mean x^2 + eps); then pairs (a, b) of the first `rot` channels turn by
// the angle position * f_i: (a cos - b sin, b cos + a sin), the pairs being channels (i, i + rot / 2) or (2 i, 2 i + 1). One rounding to
// the rows' type at the end. What is quantised afterwards may lie next to a code's border, so every step is defined to the last
// bit or nearly so: the squares are summed and r is made in 64 bits and rounded to fp32 once, angles are 64-bit products (a far
// position times a frequency), their cosines and sines are made in 64 bits (good to some 2^-52) and rounded to fp32 once, the rest
// are single fp32 operations in the order written. The vector units do as many 64-bit fused multiply-adds as 32-bit ones, and an
// angle's are shared by all heads of a token.
//
// Bound by memory. A workgroup takes 4 tokens (few rows: 1), makes their cosines and sines in LDS, one angle to a thread, and walks
// the heads, 16 rows of 128 at a time (64: 32); a row is 8 channels in each of dim / 8 lanes, which keep their token and so the
// cosines and sines of their channels in registers. The 8 are 4 and the 4 that they turn with, so no lane needs another's (8
// neighbours, and their partners loaded and normed a second time: 305 us for the next line's 272, the vector units 71 % busy); keys
// on their way into a cache are 8 neighbours, as their codes lie. (Rows of more than the last cache holds streamed past it take the
// same time, 16 and 32 bits, alone, with a reader behind them and on their way into a cache.)
// Measured: 22,332 rows x 112 heads of 128, bf16, 96 channels turned, normed (1.28 GB) 272 us, 4.7 TB/s (a large copy moves 5.1), the
// vector units 64 % busy; 24,009 rows x 56 query heads and 8 K/V heads, fp16, 64 channels turned, into an int8 cache (0.84 GB) 190 us,
// 4.4 TB/s. 8 rows x 40 heads 4.4 us, 24 x 48 into a 4-bit cache 5.2: a few dependent loads, the cosines and a barrier.
#include "kv_rows.hpp"

namespace rh3 {
namespace kv {
namespace {

constexpr int NONE = -1;             // FMT of the rows that go to no cache
constexpr int MOST_PAIRS = 64;       // of a head

struct Turn {
  const double* freq;                // [rot / 2] radians to a position, or null
  double factor;                     // of the cosines and sines
  int rot, interleaved;
  int norm, wide;                    // wide: fp32 weights (else of the rows' type)
  double eps;
  const void *qw, *kw;               // [dim] or null
};
struct RopeArgs {
  Turn t;
  rh3_head_rows q, k, v;             // v: not of FMT NONE
  rh3_head_rows qo, ko;              // ko: of FMT NONE
  int q_heads, k_heads, rows, log2tt;
  int first;                         // added to the positions of the cache's rows
  const int32_t* positions;          // FMT NONE
  Cache c;
  Seqs s;
};

// cosine and sine of a (64 bits): a less the nearest multiple of pi / 2 (in two parts of 53 bits), then the Taylor series, whose next
// terms are under 2^-54 on +-pi / 4
__device__ __forceinline__ float2 cos_sin(double a, double factor) {
  const double n = __builtin_rint(a * 0.63661977236758134308);
  double r = __builtin_fma(n, -1.57079632679489655800, a);
  r = __builtin_fma(n, -6.12323399573676603587e-17, r);
  const double z = r * r;
  double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
  s = __builtin_fma(s, z, 1.0 / 6227020800.0);
  s = __builtin_fma(s, z, -1.0 / 39916800.0);
  s = __builtin_fma(s, z, 1.0 / 362880.0);
  s = __builtin_fma(s, z, -1.0 / 5040.0);
  s = __builtin_fma(s, z, 1.0 / 120.0);
  s = __builtin_fma(s, z, -1.0 / 6.0);
  s = __builtin_fma(s * z, r, r);
  c = __builtin_fma(c, z, -1.0 / 87178291200.0);
  c = __builtin_fma(c, z, 1.0 / 479001600.0);
  c = __builtin_fma(c, z, -1.0 / 3628800.0);
  c = __builtin_fma(c, z, 1.0 / 40320.0);
  c = __builtin_fma(c, z, -1.0 / 720.0);
  c = __builtin_fma(c, z, 1.0 / 24.0);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int quarter = static_cast<int>(n - 4.0 * __builtin_floor(n * 0.25));   // 0 .. 3 quarters of a turn
  const double x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
  return make_float2(static_cast<float>((quarter == 1 || quarter == 2 ? -x : x) * factor), static_cast<float>((quarter >= 2 ? -y : y) * factor));
}

// a lane's 64-bit value from lane l ^ 8, 4, 2 or 1 of its 16
template <int CTRL>
__device__ __forceinline__ double moved(double v) {
  const int64_t b = __builtin_bit_cast(int64_t, v);
  const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, 0xf, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (static_cast<int64_t>(hi) << 32) | static_cast<uint32_t>(lo));
}
__device__ __forceinline__ double squares8(const float* x) {
  double s = 0.0;
#pragma unroll
  for (int e = 0; e < 8; ++e) s = __builtin_fma(static_cast<double>(x[e]), static_cast<double>(x[e]), s);
  return s;
}
// 1 / sqrt(mean x^2 + eps) of a row in dim / 8 lanes by their sums of squares
template <int D>
__device__ __forceinline__ float inverse_rms(double s, double eps) {
  s += moved<0xB1>(s);                      // quad_perm [1,0,3,2]
  s += moved<0x4E>(s);                      // quad_perm [2,3,0,1]
  s += moved<0x1B>(moved<0x141>(s));        // row_half_mirror, quad_perm [3,2,1,0]: lane ^ 4
  if constexpr (D == 128) s += moved<0x128>(s);   // row_ror:8
  const double m = __builtin_fma(s, 1.0 / D, eps);
  double y = __builtin_amdgcn_rsq(m);
  if (m > 0.0 && m < static_cast<double>(INFINITY)) {   // two steps of Newton's method on the hardware's first 2^-24 or so
    const double h = 0.5 * m;
    y = __builtin_fma(y, __builtin_fma(-h * y, y, 0.5), y);
    y = __builtin_fma(y, __builtin_fma(-h * y, y, 0.5), y);
  }
  return static_cast<float>(y);
}

// 4 channels of a row as they lie
template <int DT>
struct Raw4 {
  uint32_t w[DT == RH3_DTYPE_F32 ? 4 : 2];
};
template <int DT>
__device__ __forceinline__ Raw4<DT> load_raw4(const void* p, int64_t at) {
  Raw4<DT> r;
  if constexpr (DT == RH3_DTYPE_F32) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(static_cast<const float*>(p) + at);
    r.w[0] = x[0]; r.w[1] = x[1]; r.w[2] = x[2]; r.w[3] = x[3];
  } else {
    const u32x2_t x = *reinterpret_cast<const u32x2_t*>(static_cast<const uint16_t*>(p) + at);
    r.w[0] = x[0]; r.w[1] = x[1];
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void values_of(const Raw4<DT>& r, float* x) {
  if constexpr (DT == RH3_DTYPE_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(r.w[e]);
  } else if constexpr (DT == RH3_DTYPE_BF16) {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      x[e] = __uint_as_float(r.w[e / 2] << 16);
      x[e + 1] = __uint_as_float(r.w[e / 2] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const h2_t h = __builtin_bit_cast(h2_t, r.w[e / 2]);
      x[e] = static_cast<float>(h[0]);
      x[e + 1] = static_cast<float>(h[1]);
    }
  }
}
template <int DT>
__device__ __forceinline__ void store4(void* p, int64_t at, const float* x) {
  if constexpr (DT == RH3_DTYPE_F32) {
    const u32x4_t r = {__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    *reinterpret_cast<u32x4_t*>(static_cast<float*>(p) + at) = r;
  } else {
    const u32x2_t r = DT == RH3_DTYPE_BF16 ? u32x2_t{pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3])} : u32x2_t{pack_h2(x[0], x[1]), pack_h2(x[2], x[3])};
    *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(p) + at) = r;
  }
}
template <int DT, int N>
__device__ __forceinline__ void weights_of(const Turn& t, const void* w, int at, float* x) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    if (!w) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i + e] = 1.0f;
    } else if (t.wide) {
      values_of<RH3_DTYPE_F32>(load_raw4<RH3_DTYPE_F32>(w, at + i), x + i);
    } else {
      values_of<DT>(load_raw4<DT>(w, at + i), x + i);
    }
  }
}
// rounded to the rows' type
template <int DT>
__device__ __forceinline__ void rounded8(float* x) {
  if constexpr (DT == RH3_DTYPE_BF16) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = round_bf(x[e]);
  } else if constexpr (DT == RH3_DTYPE_F16) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(static_cast<_Float16>(x[e]));
  }
}

// 5 waves to a SIMD for 16-bit rows into a cache (24,009 bf16 rows, 56 / 8 heads of 128, normed, int8: 212 us for 235 with 4)
template <int FMT, int D, int DT>
__global__ void __launch_bounds__(NT, FMT == NONE || DT == RH3_DTYPE_F32 ? 4 : 5) rope_kernel(RopeArgs a) {
  constexpr int LPR = D / 8, SLOTS = NT / LPR;
  __shared__ float2 turns[4][MOST_PAIRS];
  const int l = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  const int tt = 1 << a.log2tt, heads_at_once = SLOTS >> a.log2tt;
  const int tok = slot & (tt - 1), row = (blockIdx.x << a.log2tt) + tok, hs = slot >> a.log2tt;
  const Turn& t = a.t;
  const int half = t.rot >> 1;
  // two pieces of 4 channels that hold whole pairs: 4 l and its partners, or 8 neighbours
  const bool split = !t.interleaved && l < half / 4;
  const int c0 = split ? 4 * l : 8 * l, c1 = split ? half + 4 * l : c0 + 4;
  const bool turned = split || (t.interleaved && c0 < t.rot);

  Place place{0, 0, 0, true, false};
  if constexpr (FMT != NONE) place = place_of<FMT, D>(a.s, a.c, row);
  const bool mine = row < a.rows && place.mine;
  // groups of heads that go at once: the queries', then the keys'
  const int q_groups = (a.q_heads + heads_at_once - 1) / heads_at_once, k_groups = (a.k_heads + heads_at_once - 1) / heads_at_once;
  const int plain = FMT == NONE ? q_groups + k_groups : q_groups;   // those whose rows go out as rows
  int g = blockIdx.y;
  auto load = [&](int g, Raw4<DT>& r0, Raw4<DT>& r1) __attribute__((always_inline)) {
    const bool key = g >= q_groups;
    const int h = (key ? g - q_groups : g) * heads_at_once + hs;
    if (mine && g < plain && h < (key ? a.k_heads : a.q_heads)) {
      const rh3_head_rows& r = key ? a.k : a.q;
      const int64_t at = row * r.st + h * r.sh;
      r0 = load_raw4<DT>(r.x, at + c0);
      r1 = load_raw4<DT>(r.x, at + c1);
    }
  };
  Raw4<DT> raw0{}, raw1{};
  load(g, raw0, raw1);

  if (half) {
    if constexpr (FMT == NONE) {
      for (int i = threadIdx.x; i < half << a.log2tt; i += NT) {
        const int r = i / half, f = i - r * half, at = (blockIdx.x << a.log2tt) + r;
        turns[r][f] = cos_sin(static_cast<double>(at < a.rows ? a.positions[at] : 0) * t.freq[f], t.factor);
      }
    } else {
      // a token's position is known to its own lanes, those of all its heads
      const double pos = static_cast<double>(place.pos + a.first);
      for (int f = hs * LPR + l; f < half; f += heads_at_once * LPR) turns[tok][f] = cos_sin(pos * t.freq[f], t.factor);
    }
    __syncthreads();
  }
  {
    float cs[4], sn[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 v = turned ? turns[tok][4 * l + e] : make_float2(1.0f, 0.0f);
      cs[e] = v.x;
      sn[e] = v.y;
    }
    float w0[4], w1[4];
    bool loaded_q = false, loaded_k = false;
    for (; g < plain; g += gridDim.y) {
      const bool key = g >= q_groups;
      const int h = (key ? g - q_groups : g) * heads_at_once + hs;
      const bool here = mine && h < (key ? a.k_heads : a.q_heads);
      Raw4<DT> next0{}, next1{};
      load(g + gridDim.y, next0, next1);
      if (t.norm && !(key ? loaded_k : loaded_q)) {
        weights_of<DT, 4>(t, key ? t.kw : t.qw, c0, w0);
        weights_of<DT, 4>(t, key ? t.kw : t.qw, c1, w1);
        loaded_q = !key;
        loaded_k = key;
      }
      if (here) {   // whole rows of lanes
        float x[8];
        values_of<DT>(raw0, x);
        values_of<DT>(raw1, x + 4);
        if (t.norm) {
          const float r = inverse_rms<D>(squares8(x), t.eps);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = (x[e] * r) * w0[e];
            x[4 + e] = (x[4 + e] * r) * w1[e];
          }
        }
        if (turned) {
          float y[8];
          if (t.interleaved) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[2 * e] = x[2 * e] * cs[e] - x[2 * e + 1] * sn[e];
              y[2 * e + 1] = x[2 * e + 1] * cs[e] + x[2 * e] * sn[e];
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[e] = x[e] * cs[e] - x[4 + e] * sn[e];
              y[4 + e] = x[4 + e] * cs[e] + x[e] * sn[e];
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = y[e];
        }
        const rh3_head_rows& o = key ? a.ko : a.qo;
        const int64_t at = row * o.st + h * o.sh;
        store4<DT>(o.x, at + c0, x);
        store4<DT>(o.x, at + c1, x + 4);
      }
      raw0 = next0;
      raw1 = next1;
    }
  }
  if constexpr (FMT != NONE) {
    // Keys and values on their way into the cache: a lane has 8 neighbours, as the codes are kept. The other channels of its pairs,
    // where they lie rot / 2 apart, are loaded a second time (from L1) and normed again.
    const int own = 8 * l;
    const bool turned = own < t.rot;
    const int other = t.interleaved || !turned ? own : own < half ? own + half : own - half;
    auto load_kv = [&](int g, Raw<DT>& k, Raw<DT>& p, Raw<DT>& v) __attribute__((always_inline)) {
      const int h = (g - q_groups) * heads_at_once + hs;
      if (place.there && h < a.k_heads) {
        const int64_t at = row * a.k.st + h * a.k.sh;
        k = load_raw<DT>(a.k.x, at + own);
        p = load_raw<DT>(a.k.x, at + other);
        v = load_raw<DT>(a.v.x, row * a.v.st + h * a.v.sh + own);
      }
    };
    // The lane's squares in the order of rows that go out as rows (whose norm may be rounded otherwise if they are summed otherwise):
    // lane m of pairs rot / 2 apart has channels 4 m + 0 .. 3 and their partners, which the first of the two lanes that hold 8 of them
    // and their partners sums for even m, the second for odd m.
    auto squares = [&](const float* x, const float* o) __attribute__((always_inline)) {
      if (t.interleaved || !half) return squares8(x);
      const bool first = own < half;
      float u[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u[e] = !turned || first ? x[e] : o[4 + e];
        u[4 + e] = turned && first ? o[e] : x[4 + e];
      }
      const double mine = squares8(u), theirs = __shfl(mine, (l >> 1) + (l & 1) * (half >> 3), LPR);
      return turned ? theirs : mine;
    };
    Raw<DT> rk{}, rp{}, rv{};
    if (g < q_groups + k_groups) load_kv(g, rk, rp, rv);
    float cs[8], sn[8], w[8], wo[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 v = turned ? turns[tok][t.interleaved ? (own + e) >> 1 : (own < half ? own : own - half) + e] : make_float2(1.0f, 0.0f);
      cs[e] = v.x;
      sn[e] = (t.interleaved ? (e & 1) == 0 : own < half) ? -v.y : v.y;
    }
    if (t.norm && g < q_groups + k_groups) {
      weights_of<DT, 8>(t, t.kw, own, w);
      weights_of<DT, 8>(t, t.kw, other, wo);
    }
    for (; g < q_groups + k_groups; g += gridDim.y) {
      const int h = (g - q_groups) * heads_at_once + hs;
      Raw<DT> nk{}, np{}, nv{};
      load_kv(g + gridDim.y, nk, np, nv);
      if (place.there && h < a.k_heads) {   // whole rows of lanes
        float x[8], o[8], y[8];
        values_of<DT>(rk, x);
        values_of<DT>(rp, o);
        values_of<DT>(rv, y);
        if (t.norm) {
          const float r = inverse_rms<D>(squares(x, o), t.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = (x[e] * r) * w[e];
            o[e] = (o[e] * r) * wo[e];
          }
        }
        if (turned) {
          if (t.interleaved) {
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = x[e ^ 1];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = x[e] * cs[e] + o[e] * sn[e];
        }
        rounded8<DT>(x);
        put<FMT, D>(a.c, place, h, l, x, y);
      }
      rk = nk;
      rp = np;
      rv = nv;
    }
  }
}

int check_turn(const char* name, const rh3_turn& x, int64_t dim, Turn& t) {
  RH3_REQUIRE(dim == 64 || dim == 128, "%s: head dim %lld (64 or 128)", name, static_cast<long long>(dim));
  RH3_REQUIRE(x.rot >= 0 && x.rot <= dim && x.rot % 16 == 0, "%s: %lld rotated channels of %lld (a multiple of 16)", name,
              static_cast<long long>(x.rot), static_cast<long long>(dim));
  RH3_REQUIRE(x.rot == 0 || x.freq, "%s: no frequencies for %lld rotated channels", name, static_cast<long long>(x.rot));
  RH3_REQUIRE(x.rot || x.norm, "%s: neither a norm nor a rotation", name);
  RH3_REQUIRE(aligned16(x.qw) && aligned16(x.kw) && (reinterpret_cast<uintptr_t>(x.freq) & 7) == 0,
              "%s: weights must be 16-byte aligned, frequencies 8-byte", name);
  t = Turn{x.freq, x.factor, static_cast<int>(x.rot), x.interleaved != 0, x.norm != 0, x.wide_weights != 0, x.eps, x.qw, x.kw};
  return RH3_OK;
}
int check_type(const char* name, int64_t dtype) {
  RH3_REQUIRE(dtype == RH3_DTYPE_BF16 || dtype == RH3_DTYPE_F16 || dtype == RH3_DTYPE_F32, "%s: row type %lld (bf16, fp16 or fp32)", name,
              static_cast<long long>(dtype));
  return RH3_OK;
}
int check_rows(const char* name, const char* what, const rh3_head_rows& r) {
  RH3_REQUIRE(r.x, "%s: null %s", name, what);
  RH3_REQUIRE(aligned16(r.x) && r.st % 8 == 0 && r.sh % 8 == 0, "%s: %s must be 16-byte aligned with strides that are multiples of 8", name, what);
  return RH3_OK;
}
int check_out(const char* name, const char* what, const rh3_head_rows& r, int64_t rows, int64_t heads) {
  if (const int e = check_rows(name, what, r)) return e;
  RH3_REQUIRE((rows == 1 || r.st != 0) && (heads == 1 || r.sh != 0), "%s: rows or heads of %s share memory", name, what);
  return RH3_OK;
}

// Few tokens go one to a workgroup, whose heads then take fewer turns; heads are spread over workgroups until there are 8 to a CU.
template <int FMT, int D>
int launch_rope(const char* name, RopeArgs& a, int64_t dtype, hipStream_t st) {
  const int64_t cus = device_cus() > 0 ? device_cus() : 256;
  a.log2tt = a.rows < 4 * cus ? 0 : 2;
  const int at_once = NT / (D / 8) >> a.log2tt;
  const int64_t gx = (static_cast<int64_t>(a.rows) + (1 << a.log2tt) - 1) >> a.log2tt;
  const int64_t groups = (a.q_heads + at_once - 1) / at_once + (a.k_heads + at_once - 1) / at_once;
  int64_t gy = (8 * cus + gx - 1) / gx;
  gy = gy < 1 ? 1 : gy > groups ? groups : gy;
  RH3_REQUIRE(gx <= MAX_GRID_256, "%s: %d rows in one call", name, a.rows);
  const dim3 grid(static_cast<uint32_t>(gx), static_cast<uint32_t>(gy));
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(NT), 0, st, a); };
  if (dtype == RH3_DTYPE_BF16) go(rope_kernel<FMT, D, RH3_DTYPE_BF16>);
  else if (dtype == RH3_DTYPE_F16) go(rope_kernel<FMT, D, RH3_DTYPE_F16>);
  else go(rope_kernel<FMT, D, RH3_DTYPE_F32>);
  return launch_status(name);
}

}  // namespace
}  // namespace kv
}  // namespace rh3

using namespace rh3;
using namespace rh3::kv;

extern "C" int rh3_qk_norm_rope(const rh3_rope_args* x, hipStream_t stream) {
  const char* name = "qk_norm_rope";
  clear_error();
  RH3_REQUIRE(x, "%s: null arguments", name);
  RopeArgs a{};
  if (const int e = check_turn(name, x->turn, x->dim, a.t)) return e;
  RH3_REQUIRE(x->rows >= 0 && x->rows <= MAX_ROWS, "%s: %lld rows", name, static_cast<long long>(x->rows));
  RH3_REQUIRE(x->q_heads >= 0 && x->q_heads <= 65535 && x->k_heads >= 0 && x->k_heads <= 65535, "%s: %lld and %lld heads", name,
              static_cast<long long>(x->q_heads), static_cast<long long>(x->k_heads));
  if (const int e = check_type(name, x->dtype)) return e;
  if (x->rows == 0 || x->q_heads + x->k_heads == 0) return RH3_OK;
  RH3_REQUIRE(x->turn.rot == 0 || x->positions, "%s: no positions", name);
  if (x->q_heads) {
    if (const int e = check_rows(name, "q", x->q)) return e;
    if (const int e = check_out(name, "q's result", x->q_out, x->rows, x->q_heads)) return e;
  }
  if (x->k_heads) {
    if (const int e = check_rows(name, "k", x->k)) return e;
    if (const int e = check_out(name, "k's result", x->k_out, x->rows, x->k_heads)) return e;
  }
  a.q = x->q;
  a.k = x->k;
  a.qo = x->q_out;
  a.ko = x->k_out;
  a.q_heads = static_cast<int>(x->q_heads);
  a.k_heads = static_cast<int>(x->k_heads);
  a.rows = static_cast<int>(x->rows);
  a.positions = x->positions;
  return x->dim == 128 ? launch_rope<NONE, 128>(name, a, x->dtype, stream) : launch_rope<NONE, 64>(name, a, x->dtype, stream);
}

extern "C" int rh3_kv_write_rope(const rh3_kv_cache* cache, const rh3_kv_rope_args* x, hipStream_t stream) {
  const char* name = "kv_write_rope";
  clear_error();
  RH3_REQUIRE(x, "%s: null arguments", name);
  RopeArgs a{};
  if (const int e = check_cache(name, cache, a.c)) return e;
  if (const int e = check_seqs(name, a.c, x->table, x->table_stride, x->width, x->lens, x->cu, x->batch, x->rows, a.s)) return e;
  if (const int e = check_turn(name, x->turn, cache->dim, a.t)) return e;
  RH3_REQUIRE(x->q_heads >= 1 && x->q_heads <= 65535, "%s: %lld query heads", name, static_cast<long long>(x->q_heads));
  RH3_REQUIRE(x->first >= -MAX_ROWS && x->first <= MAX_ROWS, "%s: first position %lld", name, static_cast<long long>(x->first));
  if (const int e = check_type(name, x->dtype)) return e;
  if (x->rows == 0) return RH3_OK;
  if (const int e = check_rows(name, "q", x->q)) return e;
  if (const int e = check_rows(name, "k", x->k)) return e;
  if (const int e = check_rows(name, "v", x->v)) return e;
  if (const int e = check_out(name, "q's result", x->q_out, x->rows, x->q_heads)) return e;
  a.q = x->q;
  a.k = x->k;
  a.v = x->v;
  a.qo = x->q_out;
  a.q_heads = static_cast<int>(x->q_heads);
  a.k_heads = a.c.heads;
  a.rows = static_cast<int>(x->rows);
  a.first = static_cast<int>(x->first);
  const int64_t fmt = cache->format;
  if (cache->dim == 128)
    return fmt == INT8 ? launch_rope<INT8, 128>(name, a, x->dtype, stream)
                       : fmt == E4M3 ? launch_rope<E4M3, 128>(name, a, x->dtype, stream) : launch_rope<FP4, 128>(name, a, x->dtype, stream);
  return fmt == INT8 ? launch_rope<INT8, 64>(name, a, x->dtype, stream)
                     : fmt == E4M3 ? launch_rope<E4M3, 64>(name, a, x->dtype, stream) : launch_rope<FP4, 64>(name, a, x->dtype, stream);
}
