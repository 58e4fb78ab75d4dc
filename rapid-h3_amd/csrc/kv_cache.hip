// Writing rows of keys and values into a paged cache as INT8 or e4m3 codes with one fp32 scale per row and head, and reading
// them back.
//
// s = max(amax / QMAX, 1e-12) (QMAX 127 or 448), code = round to nearest even of the fp32 quotient x / s: the rule of the row
// quantizers, over the 64 or 128 values of one head. A row that holds an infinity or a NaN gets s = NaN and codes 0: it reads
// back as NaN and every attention row that sees it is NaN, while no code of the cache is ever a NaN.
//
// Both are bound by memory. A row of a head is 8 values in each of dim / 8 lanes (16-byte loads of 16-bit rows, 8 bytes of codes);
// a workgroup takes 256 / (dim / 8) consecutive rows of one head after another, so that the codes it writes (a page holds a
// head's positions back to back) and its scales are whole lines, while each read of a row is dim consecutive values.
// Measured, K and V of 22,332 rows x 56 heads of 128, bf16 and e4m3 (0.97 GB each way; a large copy moves 4.8 TB/s): written in
// 237 us (4.1 TB/s, the vector units 55 % busy), read back in 184 us (5.3 TB/s); 8 x 7,919 rows x 16 heads int8 (0.79 GB)
// read back in 160 to 187 us. 16 rows of 8 heads: 3.9 and 2.8 us, the length of a few dependent loads.
#include "kv_common.hpp"

namespace rh3 {
namespace kv {
namespace {

constexpr int NT = 256;

// where a row of the call lies in the cache: offsets of its codes and scale without the head's part; false if it lies nowhere
// (no sequence has the row, its position is before the first or past the table, its page is absent). `mine`: a sequence has the row.
struct Place {
  int64_t code, scale;
  bool mine, there;
};
template <int D>
__device__ __forceinline__ Place place_of(const Seqs& s, const Cache& c, int row) {
  Place p{0, 0, false, false};
  Seq q;
  const int b = seq_of_row<D / 8 == 16 ? 16 : 8>(s, min(row, s.rows - 1), q);
  if (b < 0 || row >= s.rows) return p;
  p.mine = true;
  const int pos = q.pos + (row - q.first);
  if (pos < 0 || pos >= s.cap) return p;
  const int pg = page_of(s, c, b, pos);
  if (pg < 0) return p;
  const int off = pos & ((1 << c.log2page) - 1);
  p.code = pg * c.page_stride + off * D;
  p.scale = pg * c.spage_stride + off;
  p.there = true;
  return p;
}

// max over the D / 8 lanes of a row
template <int D>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 1)));
  v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 2)));
  v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 4)));
  if constexpr (D == 128) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 8)));
  return v;
}

template <int FMT, int D>
__device__ __forceinline__ void put(const float* x, uint8_t* codes, float* scale, bool first) {
  uint32_t m = 0;   // magnitudes order like their bits, infinities and NaN last
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
  m = row_max<D>(m);
  uint2 q = make_uint2(0u, 0u);
  float s = __uint_as_float(0x7fc00000u);
  if (m < 0x7f800000u) {
    s = fmaxf(__uint_as_float(m) / (FMT == INT8 ? 127.0f : 448.0f), 1e-12f);
    const float inv = 1.0f / s;
    if constexpr (FMT == INT8)
      q = quant8_i8(x, s, inv);
    else
      q = quant8_fp8(x, s, inv, fp8_odd(__uint_as_float(m), 0.0f, s));
  }
  *reinterpret_cast<uint2*>(codes) = q;
  if (first) *scale = s;
}

template <int FMT, int D, int DT>
__global__ void __launch_bounds__(NT) write_kernel(Cache c, Seqs s, const void* __restrict__ k, int64_t k_st, int64_t k_sh,
                                                   const void* __restrict__ v, int64_t v_st, int64_t v_sh) {
  constexpr int LPR = D / 8;
  const int l = threadIdx.x % LPR;
  const int row = blockIdx.x * (NT / LPR) + threadIdx.x / LPR;
  const Place p = place_of<D>(s, c, row);
  if (!p.there) return;   // whole rows of lanes leave together
  for (int h = blockIdx.y; h < c.heads; h += gridDim.y) {
    float x[8], y[8];
    load_row8<DT>(k, row * k_st + h * k_sh + 8 * l, x);
    load_row8<DT>(v, row * v_st + h * v_sh + 8 * l, y);
    const int64_t code = p.code + h * c.head_stride + 8 * l, scale = p.scale + h * c.shead_stride;
    put<FMT, D>(x, c.k + code, c.ks + scale, l == 0);
    put<FMT, D>(y, c.v + code, c.vs + scale, l == 0);
  }
}

template <int FMT>
__device__ __forceinline__ void values(uint2 w, float s, float* x) {
  if constexpr (FMT == INT8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = static_cast<float>(static_cast<int8_t>(w.x >> (8 * e))) * s;
      x[4 + e] = static_cast<float>(static_cast<int8_t>(w.y >> (8 * e))) * s;
    }
  } else {
    const f2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, true);
    const f2_t d = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, true);
    x[0] = a[0] * s; x[1] = a[1] * s; x[2] = b[0] * s; x[3] = b[1] * s;
    x[4] = d[0] * s; x[5] = d[1] * s; x[6] = e[0] * s; x[7] = e[1] * s;
  }
}

template <int FMT, int D, int DT>
__global__ void __launch_bounds__(NT) read_kernel(Cache c, Seqs s, void* __restrict__ k, int64_t k_st, int64_t k_sh,
                                                  void* __restrict__ v, int64_t v_st, int64_t v_sh) {
  constexpr int LPR = D / 8;
  const int l = threadIdx.x % LPR;
  const int row = blockIdx.x * (NT / LPR) + threadIdx.x / LPR;
  const Place p = place_of<D>(s, c, row);
  if (!p.mine) return;
  for (int h = blockIdx.y; h < c.heads; h += gridDim.y) {
    float x[8] = {}, y[8] = {};
    if (p.there) {
      const int64_t code = p.code + h * c.head_stride + 8 * l, scale = p.scale + h * c.shead_stride;
      values<FMT>(*reinterpret_cast<const uint2*>(c.k + code), c.ks[scale], x);
      values<FMT>(*reinterpret_cast<const uint2*>(c.v + code), c.vs[scale], y);
    }
    store_row8<DT>(k, row * k_st + h * k_sh + 8 * l, x);
    store_row8<DT>(v, row * v_st + h * v_sh + 8 * l, y);
  }
}

// Workgroups for `rows` rows: along x the rows, along y as many heads side by side as it takes for 8 workgroups to a CU; the
// other heads are the workgroup's loop, which resolves a row's page once for all of them.
dim3 grid_of(int64_t rows, int heads, int dim) {
  const int64_t gx = (rows + NT / (dim / 8) - 1) / (NT / (dim / 8));
  const int64_t want = 8 * static_cast<int64_t>(device_cus() > 0 ? device_cus() : 256);
  int64_t gy = (want + gx - 1) / gx;
  gy = gy < 1 ? 1 : gy > heads ? heads : gy;
  return dim3(static_cast<uint32_t>(gx), static_cast<uint32_t>(gy));
}

template <bool WRITE, int FMT, int D>
void launch_rows(int dtype, dim3 g, hipStream_t st, const Cache& c, const Seqs& s, void* k, int64_t k_st, int64_t k_sh, void* v,
                 int64_t v_st, int64_t v_sh) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, dim3(NT), 0, st, c, s, k, k_st, k_sh, v, v_st, v_sh); };
  if constexpr (WRITE) {
    if (dtype == RH3_DTYPE_BF16) go(write_kernel<FMT, D, RH3_DTYPE_BF16>);
    else if (dtype == RH3_DTYPE_F16) go(write_kernel<FMT, D, RH3_DTYPE_F16>);
    else go(write_kernel<FMT, D, RH3_DTYPE_F32>);
  } else {
    if (dtype == RH3_DTYPE_BF16) go(read_kernel<FMT, D, RH3_DTYPE_BF16>);
    else if (dtype == RH3_DTYPE_F16) go(read_kernel<FMT, D, RH3_DTYPE_F16>);
    else go(read_kernel<FMT, D, RH3_DTYPE_F32>);
  }
}

template <bool WRITE>
int rows_call(const char* name, const rh3_kv_cache* cache, void* k, int64_t k_st, int64_t k_sh, void* v, int64_t v_st, int64_t v_sh,
              int dtype, int64_t rows, const int32_t* table, int64_t table_stride, int64_t width, const int32_t* lens,
              const int32_t* cu, int64_t batch, hipStream_t st) {
  clear_error();
  Cache c;
  if (const int e = check_cache(name, cache, c)) return e;
  Seqs s;
  if (const int e = check_seqs(name, c, table, table_stride, width, lens, cu, batch, rows, s)) return e;
  if (rows == 0) return RH3_OK;
  RH3_REQUIRE(dtype == RH3_DTYPE_BF16 || dtype == RH3_DTYPE_F16 || dtype == RH3_DTYPE_F32, "%s: row type %d (bf16, fp16 or fp32)", name, dtype);
  RH3_REQUIRE(k && v, "%s: null rows", name);
  RH3_REQUIRE(aligned16(k) && aligned16(v) && k_st % 8 == 0 && k_sh % 8 == 0 && v_st % 8 == 0 && v_sh % 8 == 0,
              "%s: rows must be 16-byte aligned with strides that are multiples of 8", name);
  if constexpr (!WRITE)
    RH3_REQUIRE((rows == 1 || (k_st != 0 && v_st != 0)) && (c.heads == 1 || (k_sh != 0 && v_sh != 0)),
                "%s: rows or heads of the result share memory", name);
  const int dim = static_cast<int>(cache->dim), fmt = static_cast<int>(cache->format);
  const dim3 g = grid_of(rows, c.heads, dim);
  RH3_REQUIRE(g.x <= MAX_GRID_256, "%s: %lld rows in one call", name, static_cast<long long>(rows));
  if (fmt == INT8 && dim == 128) launch_rows<WRITE, INT8, 128>(dtype, g, st, c, s, k, k_st, k_sh, v, v_st, v_sh);
  else if (fmt == INT8) launch_rows<WRITE, INT8, 64>(dtype, g, st, c, s, k, k_st, k_sh, v, v_st, v_sh);
  else if (dim == 128) launch_rows<WRITE, E4M3, 128>(dtype, g, st, c, s, k, k_st, k_sh, v, v_st, v_sh);
  else launch_rows<WRITE, E4M3, 64>(dtype, g, st, c, s, k, k_st, k_sh, v, v_st, v_sh);
  return launch_status(name);
}

}  // namespace

int check_cache(const char* name, const rh3_kv_cache* x, Cache& c) {
  RH3_REQUIRE(x, "%s: null cache", name);
  RH3_REQUIRE(x->k && x->v && x->k_scale && x->v_scale, "%s: null cache array", name);
  RH3_REQUIRE(x->format == RH3_KV_INT8 || x->format == RH3_KV_E4M3, "%s: cache format %lld", name, static_cast<long long>(x->format));
  RH3_REQUIRE(x->dim == 64 || x->dim == 128, "%s: head dim %lld (64 or 128)", name, static_cast<long long>(x->dim));
  RH3_REQUIRE(x->page >= 16 && x->page <= 256 && (x->page & (x->page - 1)) == 0, "%s: page of %lld positions (16, 32, 64, 128 or 256)",
              name, static_cast<long long>(x->page));
  RH3_REQUIRE(x->pages >= 1 && x->pages <= INT32_MAX, "%s: %lld pages", name, static_cast<long long>(x->pages));
  RH3_REQUIRE(x->heads >= 1 && x->heads <= 65535, "%s: %lld heads", name, static_cast<long long>(x->heads));
  RH3_REQUIRE(aligned16(x->k) && aligned16(x->v) && aligned16(x->k_scale) && aligned16(x->v_scale) && x->page_stride % 16 == 0 &&
                  x->head_stride % 16 == 0 && x->scale_page_stride % 4 == 0 && x->scale_head_stride % 4 == 0,
              "%s: pages and heads of the cache must be 16-byte aligned", name);
  RH3_REQUIRE(x->page_stride >= 0 && x->head_stride >= 0 && x->scale_page_stride >= 0 && x->scale_head_stride >= 0,
              "%s: negative stride in the cache", name);
  c.k = static_cast<uint8_t*>(x->k);
  c.v = static_cast<uint8_t*>(x->v);
  c.ks = x->k_scale;
  c.vs = x->v_scale;
  c.page_stride = x->page_stride;
  c.head_stride = x->head_stride;
  c.spage_stride = x->scale_page_stride;
  c.shead_stride = x->scale_head_stride;
  c.pages = static_cast<int>(x->pages);
  c.heads = static_cast<int>(x->heads);
  c.log2page = __builtin_ctzll(static_cast<unsigned long long>(x->page));
  return RH3_OK;
}

int check_seqs(const char* name, const Cache& c, const int32_t* table, int64_t table_stride, int64_t width, const int32_t* lens,
               const int32_t* cu, int64_t batch, int64_t rows, Seqs& s) {
  RH3_REQUIRE(rows >= 0 && rows <= MAX_ROWS, "%s: %lld rows", name, static_cast<long long>(rows));
  if (rows == 0 && batch == 0) return RH3_OK;   // the callers have nothing to do
  RH3_REQUIRE(batch >= 1 && batch <= 65536, "%s: %lld sequences (1 to 65536)", name, static_cast<long long>(batch));
  RH3_REQUIRE(table && lens, "%s: null page table or lengths", name);
  RH3_REQUIRE(width >= 1 && table_stride >= (batch > 1 ? width : 0) && width <= (MAX_ROWS >> c.log2page),
              "%s: page table of %lld entries per sequence, stride %lld", name, static_cast<long long>(width), static_cast<long long>(table_stride));
  RH3_REQUIRE(cu || rows % batch == 0, "%s: %lld rows do not divide over %lld sequences (give their offsets)", name,
              static_cast<long long>(rows), static_cast<long long>(batch));
  s.table = table;
  s.table_stride = table_stride;
  s.lens = lens;
  s.cu = cu;
  s.width = static_cast<int>(width);
  s.batch = static_cast<int>(batch);
  s.rows = static_cast<int>(rows);
  s.per = cu ? 0 : static_cast<int>(rows / batch);
  s.cap = static_cast<int>(width << c.log2page);
  return RH3_OK;
}

}  // namespace kv
}  // namespace rh3

extern "C" int rh3_kv_write(const rh3_kv_cache* cache, const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st,
                            int64_t v_sh, int dtype, int64_t rows, const int32_t* table, int64_t table_stride, int64_t width,
                            const int32_t* lens, const int32_t* cu, int64_t batch, hipStream_t stream) {
  return rh3::kv::rows_call<true>("kv_write", cache, const_cast<void*>(k), k_st, k_sh, const_cast<void*>(v), v_st, v_sh, dtype, rows,
                                  table, table_stride, width, lens, cu, batch, stream);
}

extern "C" int rh3_kv_read(const rh3_kv_cache* cache, void* k, int64_t k_st, int64_t k_sh, void* v, int64_t v_st, int64_t v_sh,
                           int dtype, int64_t rows, const int32_t* table, int64_t table_stride, int64_t width, const int32_t* lens,
                           const int32_t* cu, int64_t batch, hipStream_t stream) {
  return rh3::kv::rows_call<false>("kv_read", cache, k, k_st, k_sh, v, v_st, v_sh, dtype, rows, table, table_stride, width, lens,
                                   cu, batch, stream);
}
