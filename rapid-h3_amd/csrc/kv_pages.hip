// The page tables of a batch from one step to the next, kept on the GPU: sequences that have ended give their pages back, those that
// take rows back (drafts that were not accepted, a step for which there were too few pages) the pages behind them, every sequence
// takes the pages that its new rows need, and of each new row the position and the slot in the cache are written down.
//
// A pool is a list of free pages, taken and given back at its end, and how many there are. In the order of the sequences, and of each
// one's table: the pages that come back go on the list, then those that are needed come off it. With start = 0 for a sequence that has
// ended, its length less the rows it takes back else, end = start + its new rows, P positions to a page: the entries
// [ceil(start / P), ceil(length / P)) of its row of the table come back, the entries [ceil(start / P), ceil(end / P)) are then the next
// pages off the list, as far as the row and the list reach.
// All of it is prefix sums over the sequences and searches in them, so the result is the same in every run.
//
// Bound by latency: a step moves 9 bytes a sequence, 12 a row and 8 a page. The sums need one workgroup: it makes them, walks the
// pages that come back (8 entries to a thread at a time, in order) and, of small calls, does the rest too; of large ones a second
// launch spreads the pages taken and the rows over the chip. A page that is taken is looked up in the list, not in the table, which
// the same launch is writing. Measured: 16 sequences, a row each, 5.6 us; 700 sequences, 7,698 pages back, 10,112 taken, 161,371
// rows 10.8 + 5.3 us (with each entry's search on its own 15.4 + 5.3), of which the pages that come back are 6.5.
#include "kv_common.hpp"

namespace rh3 {
namespace kv {
namespace {

constexpr int ROW_NT = 256;
constexpr int NEAR = 2048;             // sequences whose sums are kept in LDS
constexpr int MOST = 1 << 30;          // positions of a sequence

struct PagesArgs {
  int32_t* free;
  int32_t* state;                      // pages in the list; what the last call lacked
  int32_t* table;
  int64_t table_stride;
  int32_t* lens;
  const int32_t* more;                 // new rows
  const uint8_t* done;
  int32_t* cu;
  int32_t* positions;
  int64_t* slots;
  int32_t *back, *taken, *start;       // workspace: pages given back and taken before each sequence [batch + 1], starts [batch + 1]
  int pages, width, batch, rows, log2page, alone;
};

// the last i in [0, n) with at[i] <= v, where at[0] <= v < at[n]
template <typename Array>
__device__ __forceinline__ int search(const Array at, int n, int v) {
  int lo = 0;
  while (n > 1) {
    const int half = n >> 1;
    if (at[lo + half] <= v) {
      lo += half;
      n -= half;
    } else {
      n = half;
    }
  }
  return lo;
}

// the same for N values side by side, whose loads do not wait for each other
template <int N, typename Array>
__device__ __forceinline__ void search(const Array at, int n, const int (&v)[N], int (&lo)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) lo[i] = 0;
  while (n > 1) {   // halves of one size for all: the second may begin inside the first
    const int half = n >> 1;
#pragma unroll
    for (int i = 0; i < N; ++i) lo[i] = at[lo[i] + half] <= v[i] ? lo[i] + half : lo[i];
    n -= half;
  }
}

__device__ __forceinline__ int pages_for(const PagesArgs& a, int positions) {
  return min((positions + (1 << a.log2page) - 1) >> a.log2page, a.width);
}

// sums over the threads before this one, in place, and over all; one barrier before the next call's may begin
struct Counts {
  int back, taken;
  int64_t rows;
};
template <int WAVES>
__device__ __forceinline__ Counts scan(Counts& v, Counts (&waves)[WAVES]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Counts s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const Counts up{__shfl_up(s.back, d), __shfl_up(s.taken, d), __shfl_up(s.rows, d)};
    if (lane >= d) {
      s.back += up.back;
      s.taken += up.taken;
      s.rows += up.rows;
    }
  }
  if (lane == 63) waves[wave] = s;
  __syncthreads();
  // the waves' sums, one to a lane, and theirs up to each
  Counts w = lane < WAVES ? waves[lane] : Counts{0, 0, 0};
  const Counts own = waves[wave];
#pragma unroll
  for (int d = 1; d < WAVES; d <<= 1) {
    const Counts up{__shfl_up(w.back, d), __shfl_up(w.taken, d), __shfl_up(w.rows, d)};
    if (lane >= d) w = Counts{w.back + up.back, w.taken + up.taken, w.rows + up.rows};
  }
  auto at = [&](int l) { return Counts{__shfl(w.back, l), __shfl(w.taken, l), __shfl(w.rows, l)}; };
  const Counts to = at(wave);
  v = Counts{to.back - own.back + s.back - v.back, to.taken - own.taken + s.taken - v.taken, to.rows - own.rows + s.rows - v.rows};
  return at(WAVES - 1);
}

// page i of those taken, off the end of a list of `held`; -1 where it is empty
__device__ __forceinline__ int taken_page(const PagesArgs& a, int held, int i) { return i < held ? a.free[held - 1 - i] : -1; }

// ... into its place in the table
template <typename Array>
__device__ __forceinline__ void take(const PagesArgs& a, const Array taken, int held, int i) {
  const int s = search(taken, a.batch, i);
  const int p0 = pages_for(a, a.start[s]);
  a.table[s * a.table_stride + p0 + i - taken[s]] = taken_page(a, held, i);
}

// position and slot of row r
template <typename Cu, typename Array>
__device__ __forceinline__ void row(const PagesArgs& a, const Cu cu, const Array taken, int held, int r, int& pos, int64_t& slot) {
  pos = -1;
  slot = -1;
  if (r >= cu[a.batch]) return;
  const int s = search(cu, a.batch, r);
  const int start = a.start[s];
  pos = static_cast<int>(min(static_cast<int64_t>(start) + (r - cu[s]), static_cast<int64_t>(MOST)));
  const int p = pos >> a.log2page, p0 = pages_for(a, start);
  if (p >= a.width) return;
  const int page = p < p0 ? a.table[s * a.table_stride + p] : taken_page(a, held, taken[s] + p - p0);
  if (page >= 0 && page < a.pages) slot = (static_cast<int64_t>(page) << a.log2page) + (pos & ((1 << a.log2page) - 1));
}

template <int NT>
__global__ void __launch_bounds__(NT) plan_kernel(PagesArgs a) {
  constexpr int WAVES = NT / 64;
  constexpr bool FEW = NT == 256;      // calls that are near and alone
  __shared__ int near_back[NEAR + 1], near_taken[NEAR + 1], near_cu[NEAR + 1];
  __shared__ int near_entry[NEAR];      // the first entry that comes back, less those of the sequences before
  __shared__ Counts counts[2][WAVES];   // two in turn, so that one barrier to a turn is enough
  constexpr int EACH = 8;
  __shared__ int valid[2][EACH * WAVES];
  const int tid = threadIdx.x;
  const bool near = FEW || a.batch <= NEAR, alone = FEW || a.alone;
  const int held0 = min(max(a.state[0], 0), a.pages);
  Counts sum{0, 0, 0};
  for (int at = 0, turn = 0; at < a.batch; at += NT, turn ^= 1) {
    const int b = at + tid;
    int start = 0, end = 0;
    Counts mine{0, 0, 0};
    if (b < a.batch) {
      const int len = min(max(a.lens[b], 0), MOST), more = min(max(a.more[b], -MOST), MOST);
      const bool over = a.done && a.done[b];
      start = over ? 0 : max(len + min(more, 0), 0);
      end = min(start + max(more, 0), MOST);
      mine = Counts{pages_for(a, len) - pages_for(a, start), pages_for(a, end) - pages_for(a, start), max(more, 0)};
    }
    const Counts all = scan(mine, counts[turn]);
    if (b < a.batch) {
      const int back = sum.back + mine.back, taken = sum.taken + mine.taken;
      const int cu = static_cast<int>(min(sum.rows + mine.rows, static_cast<int64_t>(INT32_MAX)));
      a.lens[b] = end;
      a.cu[b] = cu;
      a.start[b] = start;
      if (near) {
        near_back[b] = back;
        near_entry[b] = pages_for(a, start) - back;
        near_taken[b] = taken;
        near_cu[b] = cu;
      } else {
        a.back[b] = back;
      }
      if (!alone) a.taken[b] = taken;
    }
    sum = Counts{sum.back + all.back, sum.taken + all.taken, sum.rows + all.rows};
  }
  const int back = sum.back, taken = sum.taken;
  if (tid == 0) {
    const int cu = static_cast<int>(min(sum.rows, static_cast<int64_t>(INT32_MAX)));
    a.cu[a.batch] = cu;
    a.taken[a.batch] = taken;
    if (near) {
      near_back[a.batch] = back;
      near_taken[a.batch] = taken;
      near_cu[a.batch] = cu;
    } else {
      a.back[a.batch] = back;
    }
  }
  __syncthreads();

  // what comes back: EACH entries to a thread, NT apart, so that neighbours' lie side by side. An entry's place on the list is counted
  // over those before it: of earlier EACH, of earlier waves, of earlier lanes.
  int held = held0;
  const int lane = tid & 63, wave = tid >> 6;
  for (int at = 0, turn = 0; at < back; at += NT * EACH, turn ^= 1) {
    int f[EACH], s[EACH], entry[EACH];
    uint64_t there[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) f[i] = min(at + NT * i + tid, back - 1);
    near ? search(near_back, a.batch, f, s) : search(a.back, a.batch, f, s);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      int32_t* e = a.table + s[i] * a.table_stride + (f[i] + (near ? near_entry[s[i]] : pages_for(a, a.start[s[i]]) - a.back[s[i]]));
      entry[i] = -1;
      if (at + NT * i + tid < back) {
        entry[i] = *e;
        *e = -1;
      }
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      there[i] = __builtin_amdgcn_ballot_w64(entry[i] >= 0 && entry[i] < a.pages);
      if (lane == 0) valid[turn][i * WAVES + wave] = __popcll(there[i]);
    }
    __syncthreads();
    // counts in order, PER to a lane, and their sums up to each
    constexpr int PER = (EACH * WAVES + 63) / 64;
    int n[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      n[i] = PER * lane + i < EACH * WAVES ? valid[turn][PER * lane + i] : 0;
      sum += n[i];
    }
    int upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(upto, d);
      if (lane >= d) upto += up;
    }
    const int all = __shfl(upto, 63);
    int before[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int at = i * WAVES + wave, l = at / PER;
      before[i] = __shfl(upto - sum, l);
#pragma unroll
      for (int j = 0; j + 1 < PER; ++j) before[i] += j < at % PER ? __shfl(n[j], l) : 0;
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int to = held + before[i] + static_cast<int>(__popcll(there[i] & ((uint64_t{1} << lane) - 1)));
      if ((there[i] >> lane & 1) && to < a.pages) a.free[to] = entry[i];
    }
    held = min(held + all, a.pages);
  }
  if (tid == 0) {
    a.state[0] = max(held - taken, 0);
    a.state[1] = max(taken - held, 0);
    a.start[a.batch] = held;           // for the second launch
  }
  if (!alone) return;                  // (alone: few sequences, whose sums are near)
  __syncthreads();
  for (int i = tid; i < taken; i += NT) take(a, near_taken, held, i);
  for (int r = tid; r < a.rows; r += NT) {
    int pos;
    int64_t slot;
    row(a, near_cu, near_taken, held, r, pos, slot);
    a.positions[r] = pos;
    a.slots[r] = slot;
  }
}

__global__ void __launch_bounds__(ROW_NT) rows_kernel(PagesArgs a) {
  __shared__ int near_taken[NEAR + 1], near_cu[NEAR + 1];
  const bool near = a.batch <= NEAR;
  if (near) {
    for (int i = threadIdx.x; i <= a.batch; i += ROW_NT) {
      near_taken[i] = a.taken[i];
      near_cu[i] = a.cu[i];
    }
    __syncthreads();
  }
  const int held = a.start[a.batch], taken = near ? near_taken[a.batch] : a.taken[a.batch];
  const int first = blockIdx.x * ROW_NT + threadIdx.x, step = gridDim.x * ROW_NT;
  for (int i = first; i < taken; i += step) near ? take(a, near_taken, held, i) : take(a, a.taken, held, i);
  for (int64_t r = first; r < a.rows; r += step) {
    int pos;
    int64_t slot;
    if (near) row(a, near_cu, near_taken, held, static_cast<int>(r), pos, slot);
    else row(a, a.cu, a.taken, held, static_cast<int>(r), pos, slot);
    a.positions[r] = pos;
    a.slots[r] = slot;
  }
}

}  // namespace
}  // namespace kv
}  // namespace rh3

using namespace rh3;
using namespace rh3::kv;

extern "C" int64_t rh3_kv_extend_workspace_bytes(int64_t batch) { return batch < 1 || batch > 65536 ? 0 : 3 * (batch + 1) * 4; }

extern "C" int rh3_kv_extend(const rh3_kv_extend_args* x, hipStream_t stream) {
  const char* name = "kv_extend";
  clear_error();
  RH3_REQUIRE(x, "%s: null arguments", name);
  const int64_t page = x->page, width = x->width, batch = x->batch, rows = x->rows;
  RH3_REQUIRE(x->pages >= 1 && x->pages <= INT32_MAX, "%s: %lld pages", name, static_cast<long long>(x->pages));
  RH3_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "%s: page of %lld positions (16, 32, 64, 128 or 256)", name,
              static_cast<long long>(page));
  RH3_REQUIRE(rows >= 0 && rows <= MAX_ROWS, "%s: %lld rows", name, static_cast<long long>(rows));
  if (rows == 0 && batch == 0) return RH3_OK;
  RH3_REQUIRE(batch >= 1 && batch <= 65536, "%s: %lld sequences (1 to 65536)", name, static_cast<long long>(batch));
  PagesArgs a{};
  a.log2page = __builtin_ctzll(static_cast<unsigned long long>(page));
  RH3_REQUIRE(width >= 1 && width <= (MAX_ROWS >> a.log2page) && x->table_stride >= (batch > 1 ? width : 0) && batch * width <= MAX_ROWS,
              "%s: page table of %lld entries per sequence, stride %lld", name, static_cast<long long>(width),
              static_cast<long long>(x->table_stride));
  RH3_REQUIRE(x->free_pages && x->state && x->table && x->lens && x->more && x->cu, "%s: null pool, page table, lengths, new rows or offsets", name);
  RH3_REQUIRE(rows == 0 || (x->positions && x->slots), "%s: null positions or slots", name);
  RH3_REQUIRE(x->workspace && aligned16(x->workspace) && x->workspace_bytes >= rh3_kv_extend_workspace_bytes(batch),
              "%s: workspace of %lld bytes needed, %lld given", name, static_cast<long long>(rh3_kv_extend_workspace_bytes(batch)),
              static_cast<long long>(x->workspace_bytes));
  a.free = x->free_pages;
  a.state = x->state;
  a.table = x->table;
  a.table_stride = x->table_stride;
  a.lens = x->lens;
  a.more = x->more;
  a.done = x->done;
  a.cu = x->cu;
  a.positions = x->positions;
  a.slots = x->slots;
  a.back = static_cast<int32_t*>(x->workspace);
  a.taken = a.back + batch + 1;
  a.start = a.taken + batch + 1;
  a.pages = static_cast<int>(x->pages);
  a.width = static_cast<int>(width);
  a.batch = static_cast<int>(batch);
  a.rows = static_cast<int>(rows);
  // 1,024 threads for as long as one workgroup is enough for all, 256 where they would idle (each barrier is for all of them)
  a.alone = rows <= 4096 && batch <= NEAR;
  if (rows <= 1024 && batch <= 256) hipLaunchKernelGGL(plan_kernel<256>, dim3(1), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(plan_kernel<1024>, dim3(1), dim3(1024), 0, stream, a);
  if (const int e = launch_status(name)) return e;
  if (a.alone) return RH3_OK;
  const int64_t all = rows + rows / page + batch, most = 8 * static_cast<int64_t>(device_cus() > 0 ? device_cus() : 256);
  const int64_t grid = (all + ROW_NT - 1) / ROW_NT;
  hipLaunchKernelGGL(rows_kernel, dim3(static_cast<uint32_t>(grid < most ? grid : most)), dim3(ROW_NT), 0, stream, a);
  return launch_status("kv_extend (rows)");
}
