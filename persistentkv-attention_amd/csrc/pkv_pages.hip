// pkv_pages.hip — pages of the cache between steps: rows that continue another row's tokens, rows
// that end, and pages moved to the front of the pool, all from tables and lists on the GPU, and
// the copies of one layer's pages that go with them.  The reference has none of this (its pools
// and tables are filled once, tests/benchmark_serving_trace.py:285-298, 668-780).
//
// A page may be held by several rows: page_shares[p] is the number of holders beyond the first, so
// that a page fresh off the list has 0 and the operators that know nothing of sharing need not
// change.  Only full pages are shared; the page that a row still writes to is its own.
//
// Results do not depend on the order of the GPU's work: counts are integers, and lists are
// filled in the order of page ids or of the call's own lists.
//
// What bounds them is latency, a launch and a few dependent reads each, but for the copies, which are
// bound by memory.  8 forks: 3.7 us and 2.8 for a layer's copies; 64 of 700 pages each 6.8 (45,000
// counts raised, 16 on each) and 4.5; 3 rows of a pool of 61,000 pages freed: 3.2, 2.6 and 3.5 us; 90
// rows of 196,000 pages: 10.8, 2.6 and 4.1.  A pool of 31,000 pages compacted: 13 us, and 198 for the
// copies of a layer (1.0 GB, 5.0 TB/s).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pkv.h"
#include "pkv_device.h"

namespace pkv {
int fail(int status, const char* fmt, ...);  // pkv_decode.hip: sets pkv_last_error()
int ok();
}  // namespace pkv

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kChunk = 1024;     // pages that a workgroup counts and ranks
constexpr int kMaxPairs = 8000;  // rows that one call forks or frees
constexpr int kMaxColumns = 1 << 30;  // of a table: column numbers plus a workgroup's stay in 32 bits

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The sums of x over the threads before this one, and over all of them.
template <int WAVES = kWaves>
__device__ inline void block_scan(int x, int* lds, int& before, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int sum = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(sum, d);
    if (lane >= d) sum += y;
  }
  __syncthreads();  // the scan before is done with `lds`
  if (lane == 63) lds[wave] = sum;
  __syncthreads();
  before = sum - x, total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += lds[w];
    total += lds[w];
  }
}
__device__ inline int block_sum(int x, int* lds) {
  int before, total;
  block_scan(x, lds, before, total);
  return total;
}

// ---------------------------------------------------------------------------------
// Forks.
// ---------------------------------------------------------------------------------
struct ForkArgs {
  const int32_t* parents;   // [n]
  const int32_t* children;  // [n]
  const int32_t* lens;      // [batch]
  int32_t* block_table;     // [batch, max_pages]
  int32_t* page_shares;     // [num_pages]
  const int32_t* free_pages;
  const int32_t* num_free;
  int32_t* num_free_out;
  int32_t* copy_src;  // [n]
  int32_t* copy_dst;
  int32_t n, batch, max_pages, num_pages, free_capacity, page_size, columns;  // columns of a workgroup
};

// The parent's tokens, or 0 where the pair is none.
__device__ inline int fork_tokens(const ForkArgs& a, int i, int& parent, int& child) {
  parent = a.parents[i], child = a.children[i];
  if ((unsigned)parent >= (unsigned)a.batch || (unsigned)child >= (unsigned)a.batch || parent == child) return 0;
  return (int)min((long)max(a.lens[parent], 0), (long)a.max_pages * a.page_size);
}

// A workgroup a (pair, range of columns).  Each counts for itself the pairs before its own that
// need a page, and those in all: one load after another, like the launch itself, and no second
// launch to wait for.
__global__ __launch_bounds__(kThreads) void fork_kernel(ForkArgs a) {
  __shared__ int lds[kWaves];
  const int mine = blockIdx.y, tid = threadIdx.x;
  int earlier = 0, all = 0, parent, child;
  for (int i = tid; i < a.n; i += kThreads) {
    const int need = fork_tokens(a, i, parent, child) % a.page_size > 0;
    all += need;
    if (i < mine) earlier += need;
  }
  all = block_sum(all, lds);
  earlier = block_sum(earlier, lds);
  const int avail = min(max(*a.num_free, 0), a.free_capacity);
  const bool fits = all <= avail;
  const bool first = blockIdx.x == 0 && tid == 0;
  if (first && mine == 0) *a.num_free_out = avail - all;
  if (mine >= a.n) return;  // a call without pairs
  const int tokens = fork_tokens(a, mine, parent, child);
  const int full = tokens / a.page_size;
  const bool tail = tokens - full * a.page_size > 0;
  int32_t* const to = a.block_table + (long)child * a.max_pages;
  const int32_t* const from = a.block_table + (long)parent * a.max_pages;
  if (first) {
    int src = -1, dst = -1;
    if (fits && tail) {
      src = from[full], dst = a.free_pages[avail - 1 - earlier];
      to[full] = dst;
    }
    a.copy_src[mine] = src, a.copy_dst[mine] = dst;
  }
  if (!fits) return;
  const int end = min(full, (int)(blockIdx.x + 1) * a.columns);
  for (int c = blockIdx.x * a.columns + tid; c < end; c += kThreads) {
    const int page = from[c];
    to[c] = page;
    if ((unsigned)page < (unsigned)a.num_pages) atomicAdd(a.page_shares + page, 1);
  }
}

// ---------------------------------------------------------------------------------
// Pages in ascending order: counts of the chunks of kChunk pages, then places from them.
// ---------------------------------------------------------------------------------
constexpr int kEach = kChunk / kThreads;

// A thread's kEach consecutive entries of its workgroup's chunk; `other` past the end.
__device__ inline void chunk_entries(const int32_t* x, int n, int other, int (&v)[kEach]) {
  const long first = (long)blockIdx.x * kChunk + threadIdx.x * kEach;
#pragma unroll
  for (int i = 0; i < kEach; ++i) v[i] = first + i < n ? x[first + i] : other;
}

// How many entries of each chunk are negative (NEGATIVE), or not.
template <bool NEGATIVE>
__global__ __launch_bounds__(kThreads) void count_kernel(const int32_t* x, int n, int32_t* counts) {
  __shared__ int lds[kWaves];
  int v[kEach], sum = 0;
  chunk_entries(x, n, NEGATIVE ? 0 : -1, v);
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += (v[i] < 0) == NEGATIVE;
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) counts[blockIdx.x] = sum;
}

// The counts before the workgroup's chunk, and of all chunks.
__device__ inline void before_chunk(const int32_t* counts, int chunks, int* lds, int& before, int& total) {
  int b = 0, t = 0;
  for (int i = threadIdx.x; i < chunks; i += kThreads) {
    const int x = counts[i];
    t += x;
    if (i < (int)blockIdx.x) b += x;
  }
  total = block_sum(t, lds);
  before = block_sum(b, lds);
}

// ---------------------------------------------------------------------------------
// Rows that end.
// ---------------------------------------------------------------------------------
struct FreeArgs {
  const int32_t* rows;  // [n]
  const int32_t* lens;  // [batch]
  const int32_t* block_table;
  int32_t* page_shares;
  int32_t* free_pages;
  const int32_t* num_free;
  int32_t* num_free_out;
  int32_t* counts;
  int32_t n, batch, max_pages, num_pages, free_capacity, page_size, columns;
};

// One holder less for every page of the rows: a workgroup a (listed row, range of columns).  A row
// counts where it is listed first.
__global__ __launch_bounds__(kThreads) void release_kernel(FreeArgs a) {
  const int mine = blockIdx.y, tid = threadIdx.x, row = a.rows[mine];
  if ((unsigned)row >= (unsigned)a.batch) return;
  bool again = false;
  for (int i = tid; i < mine; i += kThreads) again |= a.rows[i] == row;
  if (__syncthreads_or(again)) return;
  const int len = max(a.lens[row], 0), whole = len / a.page_size;
  const int held = min(whole + (whole * a.page_size < len), a.max_pages);
  const int end = min((long)held, (long)(blockIdx.x + 1) * a.columns);
  for (int c = blockIdx.x * a.columns + tid; c < end; c += kThreads) {
    const int page = a.block_table[(long)row * a.max_pages + c];
    if ((unsigned)page < (unsigned)a.num_pages) atomicSub(a.page_shares + page, 1);
  }
}

// Pages without a holder to the end of the list, in ascending order.
__global__ __launch_bounds__(kThreads) void reclaim_kernel(FreeArgs a, int chunks) {
  __shared__ int lds[kWaves];
  int v[kEach], n = 0, before, total, earlier, unused;
  chunk_entries(a.page_shares, a.num_pages, 0, v);
#pragma unroll
  for (int i = 0; i < kEach; ++i) n += v[i] < 0;
  before_chunk(a.counts, chunks, lds, before, total);
  block_scan(n, lds, earlier, unused);
  const int avail = min(max(*a.num_free, 0), a.free_capacity);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.num_free_out = (int32_t)min((long)avail + total, (long)a.free_capacity);
  long at = (long)avail + before + earlier;
  const int first = blockIdx.x * kChunk + threadIdx.x * kEach;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (v[i] >= 0) continue;
    if (at < a.free_capacity) a.free_pages[at] = first + i;
    ++at;
    a.page_shares[first + i] = 0;
  }
}

// ---------------------------------------------------------------------------------
// Pages moved to the front.
// ---------------------------------------------------------------------------------
struct CompactArgs {
  const int32_t* block_table;  // [entries]
  const int32_t* page_shares;
  const int32_t* free_pages;
  const int32_t* num_free;
  int32_t* page_map;  // [num_pages]
  int32_t* block_table_out;
  int32_t* page_shares_out;
  int32_t* free_pages_out;
  int32_t* num_free_out;
  int32_t* copy_src;  // [copies]
  int32_t* copy_dst;
  int32_t* counts;    // [chunks], then the number of pages that move
  int64_t entries;
  int32_t num_pages, free_capacity, copies, chunks;
};

// Pools of up to kBitPages pages: one launch.  Every workgroup keeps a bit for every page in LDS, and
// the number of used pages before every 32, reads the whole list for it, and then places its
// share of the table's entries and of the pages without a word from the others.
constexpr int kBitPages = 1 << 19;  // 16384 words, twice: 128 of the 160 KB
constexpr int kBitThreads = 1024;
// The kernel's LDS, all of it in the launch's size, by which the host asks for more than 64 KB.
constexpr size_t bit_bytes(int words) { return (2 * (size_t)words + kBitThreads / 64) * sizeof(int); }
struct PageBits {
  const uint32_t* used;
  const int* before;
  int words, total;  // total: of used pages
  __device__ inline bool is_used(int p) const { return used[p >> 5] >> (p & 31) & 1; }
  __device__ inline int rank(int p) const { return before[p >> 5] + __popc(used[p >> 5] & ((1u << (p & 31)) - 1)); }
  // The free page with h free ones before it (there is one).
  __device__ inline int hole(int h) const {
    int w = 0;  // the last word with at most h free pages before it
    for (int step = 1 << (31 - __builtin_clz(words)); step; step >>= 1)
      if (w + step < words && 32 * (w + step) - before[w + step] <= h) w += step;
    uint32_t free = ~used[w];
    for (int skip = h - (32 * w - before[w]); skip > 0; --skip) free &= free - 1;
    return 32 * w + __builtin_ctz(free);
  }
  __device__ inline int place(int p) const {
    if (!is_used(p)) return -1;
    return p < total ? p : hole(total - 1 - rank(p));
  }
};
__global__ __launch_bounds__(kBitThreads) void compact_kernel(CompactArgs a) {
  extern __shared__ uint32_t bits[];  // [words], then the counts [words], then the scan's [waves]
  const int tid = threadIdx.x, words = (a.num_pages + 31) / 32;
  int* const counts = (int*)bits + words;
  int* const lds = counts + words;
  for (int w = tid; w < words; w += kBitThreads) bits[w] = 0xffffffffu;
  __syncthreads();
  if (tid == 0 && (a.num_pages & 31)) bits[words - 1] = (1u << (a.num_pages & 31)) - 1;
  __syncthreads();
  const int avail = min(max(*a.num_free, 0), a.free_capacity);
  for (int i = tid; i < avail; i += 4 * kBitThreads) {
    int page[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) page[k] = i + k * kBitThreads < avail ? a.free_pages[i + k * kBitThreads] : -1;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if ((unsigned)page[k] < (unsigned)a.num_pages) atomicAnd(&bits[page[k] >> 5], ~(1u << (page[k] & 31)));
  }
  __syncthreads();
  int before = 0, total = 0;
  for (int base = 0; base < words; base += kBitThreads) {
    const int w = base + tid;
    int earlier, sum;
    block_scan<kBitThreads / 64>(w < words ? __popc(bits[w]) : 0, lds, earlier, sum);
    if (w < words) counts[w] = before + earlier;
    before += sum;
  }
  total = before;
  __syncthreads();
  const PageBits b{bits, counts, words, total};
  const int moved = total < a.num_pages ? total - b.rank(total) : 0, left = a.num_pages - total;
  const long id = (long)blockIdx.x * kBitThreads + tid, threads = (long)gridDim.x * kBitThreads;
  if (id == 0) *a.num_free_out = left;
  for (long i = id; i < a.entries; i += threads) {
    const int page = a.block_table[i];
    a.block_table_out[i] = (unsigned)page < (unsigned)a.num_pages ? b.place(page) : page;
  }
  for (long p = id; p < a.num_pages; p += threads) {
    const int to = b.place((int)p);
    a.page_map[p] = to;
    if (to >= 0) a.page_shares_out[to] = a.page_shares[p];
    if (p >= total) {
      a.page_shares_out[p] = 0;
      if (to >= 0) {
        const int h = total - 1 - b.rank((int)p);
        a.copy_src[h] = (int)p, a.copy_dst[h] = to;
      }
    }
    if (p < left) a.free_pages_out[p] = a.num_pages - 1 - (int)p;
  }
  for (long k = moved + id; k < a.copies; k += threads) a.copy_src[k] = a.copy_dst[k] = -1;
}

// Larger pools, pass by pass.
__global__ __launch_bounds__(kThreads) void all_used_kernel(CompactArgs a) {
  const long p = (long)blockIdx.x * kThreads + threadIdx.x;
  if (p < a.num_pages) a.page_map[p] = 0;
}
__global__ __launch_bounds__(kThreads) void unused_kernel(CompactArgs a) {
  const long i = (long)blockIdx.x * kThreads + threadIdx.x;
  if (i >= min(max(*a.num_free, 0), a.free_capacity)) return;
  const int page = a.free_pages[i];
  if ((unsigned)page < (unsigned)a.num_pages) a.page_map[page] = -1;
}

// page_map holds 0 for pages in use and -1 for the others.  With U pages in use, the free page of
// rank h below U (h = its id less the used pages before it) takes the used page of rank U - 1 - h:
// the highest goes to the lowest place.  The pages that stay get their own id, those that move
// -2 - h, and the copies' lists are filled by either side for itself.
__global__ __launch_bounds__(kThreads) void place_kernel(CompactArgs a) {
  __shared__ int lds[kWaves];
  int v[kEach], n = 0, before, total, earlier, unused;
  chunk_entries(a.page_map, a.num_pages, -1, v);
#pragma unroll
  for (int i = 0; i < kEach; ++i) n += v[i] >= 0;
  before_chunk(a.counts, a.chunks, lds, before, total);
  block_scan(n, lds, earlier, unused);
  int rank = before + earlier;  // used pages before the entry
  const int first = blockIdx.x * kChunk + threadIdx.x * kEach;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int p = first + i;
    if (p >= a.num_pages) break;
    if (p == total) a.counts[a.chunks] = total - rank;  // the holes below, and what moves there
    if (v[i] >= 0) {
      const int h = total - 1 - rank;
      if (p >= total) a.copy_src[h] = p;
      a.page_map[p] = p >= total ? -2 - h : p;
      ++rank;
    } else if (p < total) {
      a.copy_dst[p - rank] = p;
    }
  }
  if (total == a.num_pages && blockIdx.x == 0 && threadIdx.x == 0) a.counts[a.chunks] = 0;
}

// Where page p has gone.  Another thread may be putting the final id in the place of -2 - h.
__device__ inline int place_of(const CompactArgs& a, int p) {
  const int m = __hip_atomic_load(a.page_map + p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return m < -1 ? a.copy_dst[-2 - m] : m;
}

__global__ __launch_bounds__(kThreads) void remap_kernel(CompactArgs a) {
  __shared__ int lds[kWaves];
  int used = 0;
  for (int i = threadIdx.x; i < a.chunks; i += kThreads) used += a.counts[i];
  used = block_sum(used, lds);
  const int moved = a.counts[a.chunks], left = a.num_pages - used;
  const long id = (long)blockIdx.x * kThreads + threadIdx.x, threads = (long)gridDim.x * kThreads;
  if (id == 0) *a.num_free_out = left;
  for (long i = id; i < a.entries; i += threads) {
    const int page = a.block_table[i];
    a.block_table_out[i] = (unsigned)page < (unsigned)a.num_pages ? place_of(a, page) : page;
  }
  for (long p = id; p < a.num_pages; p += threads) {
    const int to = place_of(a, (int)p);
    if (to >= 0) a.page_shares_out[to] = a.page_shares[p];
    if (p >= used) a.page_shares_out[p] = 0;
    if (to >= 0 && p >= used) __hip_atomic_store(a.page_map + p, to, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (p < left && p < a.free_capacity) a.free_pages_out[p] = a.num_pages - 1 - (int)p;
    if (p < a.copies && p >= moved) a.copy_src[p] = a.copy_dst[p] = -1;
  }
  for (long p = a.num_pages + id; p < a.copies; p += threads) a.copy_src[p] = a.copy_dst[p] = -1;
}

// ---------------------------------------------------------------------------------
// Copies.
// ---------------------------------------------------------------------------------
struct CopyArgs {
  const int32_t* src;  // [n]
  const int32_t* dst;
  uint8_t* pages[2];   // K, V
  float* scales;       // [num_pages, hkv, 2], or null
  long page_bytes;     // of K, and of V
  int32_t n, num_pages, hkv, slices;
};

// A workgroup a (pair, K or V, slice of LOADS * 4 KB), in turn.
template <int LOADS>
__global__ __launch_bounds__(kThreads) void copy_kernel(CopyArgs a) {
  const long units = (long)a.n * 2 * a.slices;
  for (long u = blockIdx.x; u < units; u += gridDim.x) {
    const int i = (int)(u / (2 * a.slices)), part = (int)(u - (long)i * 2 * a.slices);
    const int src = a.src[i], dst = a.dst[i];
    if ((unsigned)src >= (unsigned)a.num_pages || (unsigned)dst >= (unsigned)a.num_pages || src == dst) continue;
    uint8_t* const pool = a.pages[part & 1];
    const long at = (long)(part >> 1) * LOADS * kThreads * 16 + threadIdx.x * 16;
    u32x4 x[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      if (at + j * kThreads * 16 < a.page_bytes)
        x[j] = *(const u32x4*)(pool + src * a.page_bytes + at + j * kThreads * 16);
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      if (at + j * kThreads * 16 < a.page_bytes)
        *(u32x4*)(pool + dst * a.page_bytes + at + j * kThreads * 16) = x[j];
    if (a.scales && part == 0)
      for (int j = threadIdx.x; j < 2 * a.hkv; j += kThreads)
        a.scales[(long)dst * 2 * a.hkv + j] = a.scales[(long)src * 2 * a.hkv + j];
  }
}

int launched(const char* op) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? pkv::ok() : pkv::fail(PKV_ERR_LAUNCH, "%s launch: %s", op, hipGetErrorString(e));
}

// A call's tensors: those that it writes first, then those that it only reads.  One that is written must
// have no byte in common with another, which would be read or written while it changes.
struct Span {
  const char* name;
  const void* at;
  int64_t bytes;
};
template <int N>
int refuse_overlaps(const char* op, const Span (&spans)[N], int written) {
  for (int i = 0; i < written; ++i)
    for (int j = i + 1; j < N; ++j)
      if (spans[i].bytes > 0 && spans[j].bytes > 0 && (uintptr_t)spans[i].at < (uintptr_t)spans[j].at + spans[j].bytes &&
          (uintptr_t)spans[j].at < (uintptr_t)spans[i].at + spans[i].bytes)
        return pkv::fail(PKV_ERR_INVALID_ARGUMENT, "%s: %s must not overlap %s", op, spans[i].name, spans[j].name);
  return PKV_OK;
}
int64_t ints(int64_t n) { return n * (int64_t)sizeof(int32_t); }

// Columns that one workgroup takes, so that about four workgroups a CU share `n` rows of them out.
int columns_of(int n, int max_pages) {
  const long groups = 4L * pkv::compute_units() / n;
  const long columns = groups > 1 ? (max_pages + groups - 1) / groups : max_pages;
  return (int)((columns + kThreads - 1) / kThreads * kThreads);
}

int chunks_of(int num_pages) { return (int)(((long)num_pages + kChunk - 1) / kChunk); }

}  // namespace

extern "C" {

size_t pkv_page_workspace_bytes(int32_t num_pages) {
  return num_pages > 0 ? sizeof(int32_t) * ((size_t)chunks_of(num_pages) + 1) : 0;
}

int pkv_fork_rows(const int32_t* parents, const int32_t* children, const int32_t* lens,
                  int32_t* block_table, int32_t* page_shares, const int32_t* free_pages,
                  const int32_t* num_free, int32_t* num_free_out, int32_t* copy_src, int32_t* copy_dst,
                  int32_t num_forks, int32_t batch, int32_t max_pages, int32_t num_pages,
                  int32_t free_capacity, int32_t page_size, void* stream) {
  using pkv::fail;
  if (num_forks < 0 || batch < 0 || max_pages <= 0 || num_pages <= 0 || free_capacity < 0 || page_size <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT,
                "fork_rows: num_forks %d, batch %d, max_pages %d, num_pages %d, free_capacity %d, page_size %d",
                num_forks, batch, max_pages, num_pages, free_capacity, page_size);
  if (num_forks > kMaxPairs) return fail(PKV_ERR_UNSUPPORTED, "fork_rows: %d forks (at most %d)", num_forks, kMaxPairs);
  if ((int64_t)max_pages * page_size > INT32_MAX || max_pages > kMaxColumns)
    return fail(PKV_ERR_UNSUPPORTED, "fork_rows: max_pages * page_size does not fit in int32, or max_pages %d past %d",
                max_pages, kMaxColumns);
  if (!num_free || !num_free_out || (free_capacity > 0 && !free_pages) ||
      (num_forks > 0 && (!parents || !children || !lens || !block_table || !page_shares || !copy_src || !copy_dst)))
    return fail(PKV_ERR_INVALID_ARGUMENT, "fork_rows: null pointer");
  if (num_free == num_free_out)
    return fail(PKV_ERR_INVALID_ARGUMENT, "fork_rows: num_free_out must not be num_free");
  const int64_t listed = ints(num_forks), one = ints(1);
  const Span spans[] = {{"num_free_out", num_free_out, one}, {"copy_src", copy_src, listed}, {"copy_dst", copy_dst, listed},
                        {"block_table", block_table, listed ? ints((int64_t)batch * max_pages) : 0},
                        {"page_shares", page_shares, listed ? ints(num_pages) : 0}, {"parents", parents, listed},
                        {"children", children, listed}, {"lens", lens, listed ? ints(batch) : 0},
                        {"free_pages", free_pages, ints(free_capacity)}, {"num_free", num_free, one}};
  if (const int status = refuse_overlaps("fork_rows", spans, 5)) return status;
  const int n = num_forks > 0 ? num_forks : 1, columns = columns_of(n, max_pages);
  const ForkArgs a{parents, children, lens, block_table, page_shares, free_pages, num_free, num_free_out,
                   copy_src, copy_dst, num_forks, batch, max_pages, num_pages, free_capacity, page_size, columns};
  fork_kernel<<<dim3((unsigned)((max_pages - 1) / columns + 1), (unsigned)n), dim3(kThreads), 0, (hipStream_t)stream>>>(a);
  return launched("fork_rows");
}

int pkv_free_rows(const int32_t* rows, const int32_t* lens, const int32_t* block_table,
                  int32_t* page_shares, int32_t* free_pages, const int32_t* num_free,
                  int32_t* num_free_out, void* workspace, size_t workspace_size, int32_t num_rows,
                  int32_t batch, int32_t max_pages, int32_t num_pages, int32_t free_capacity,
                  int32_t page_size, void* stream) {
  using pkv::fail;
  if (num_rows < 0 || batch < 0 || max_pages <= 0 || num_pages <= 0 || free_capacity < 0 || page_size <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT,
                "free_rows: num_rows %d, batch %d, max_pages %d, num_pages %d, free_capacity %d, page_size %d",
                num_rows, batch, max_pages, num_pages, free_capacity, page_size);
  if (num_rows > kMaxPairs) return fail(PKV_ERR_UNSUPPORTED, "free_rows: %d rows (at most %d)", num_rows, kMaxPairs);
  if (max_pages > kMaxColumns)
    return fail(PKV_ERR_UNSUPPORTED, "free_rows: max_pages %d (at most %d)", max_pages, kMaxColumns);
  if (free_capacity < num_pages)
    return fail(PKV_ERR_INVALID_ARGUMENT, "free_rows: a list of %d places for %d pages", free_capacity, num_pages);
  if (!page_shares || !free_pages || !num_free || !num_free_out ||
      (num_rows > 0 && (!rows || !lens || !block_table)))
    return fail(PKV_ERR_INVALID_ARGUMENT, "free_rows: null pointer");
  if (num_free == num_free_out)
    return fail(PKV_ERR_INVALID_ARGUMENT, "free_rows: num_free_out must not be num_free");
  if (!workspace || workspace_size < pkv_page_workspace_bytes(num_pages) || ((uintptr_t)workspace & 3))
    return fail(PKV_ERR_WORKSPACE_TOO_SMALL, "free_rows: workspace of %zu bytes is smaller than %zu, or misaligned",
                workspace_size, pkv_page_workspace_bytes(num_pages));
  const int64_t listed = ints(num_rows), one = ints(1);
  const Span spans[] = {{"workspace", workspace, (int64_t)pkv_page_workspace_bytes(num_pages)}, {"num_free_out", num_free_out, one},
                        {"page_shares", page_shares, ints(num_pages)}, {"free_pages", free_pages, ints(free_capacity)},
                        {"rows", rows, listed}, {"lens", lens, listed ? ints(batch) : 0},
                        {"block_table", block_table, listed ? ints((int64_t)batch * max_pages) : 0}, {"num_free", num_free, one}};
  if (const int status = refuse_overlaps("free_rows", spans, 4)) return status;
  const int chunks = chunks_of(num_pages), columns = num_rows > 0 ? columns_of(num_rows, max_pages) : max_pages;
  const FreeArgs a{rows, lens, block_table, page_shares, free_pages, num_free, num_free_out, (int32_t*)workspace,
                   num_rows, batch, max_pages, num_pages, free_capacity, page_size, columns};
  if (num_rows > 0)
    release_kernel<<<dim3((unsigned)((max_pages - 1) / columns + 1), (unsigned)num_rows), dim3(kThreads), 0,
                     (hipStream_t)stream>>>(a);
  count_kernel<true><<<dim3((unsigned)chunks), dim3(kThreads), 0, (hipStream_t)stream>>>(page_shares, num_pages, a.counts);
  reclaim_kernel<<<dim3((unsigned)chunks), dim3(kThreads), 0, (hipStream_t)stream>>>(a, chunks);
  return launched("free_rows");
}

int pkv_compact_pages(const int32_t* block_table, const int32_t* page_shares, const int32_t* free_pages,
                      const int32_t* num_free, int32_t* page_map, int32_t* block_table_out,
                      int32_t* page_shares_out, int32_t* free_pages_out, int32_t* num_free_out,
                      int32_t* copy_src, int32_t* copy_dst, void* workspace, size_t workspace_size,
                      int32_t batch, int32_t max_pages, int32_t num_pages, int32_t free_capacity,
                      int32_t num_copies, void* stream) {
  using pkv::fail;
  if (batch < 0 || max_pages < 0 || num_pages <= 0 || free_capacity < 0 || num_copies < 0)
    return fail(PKV_ERR_INVALID_ARGUMENT,
                "compact_pages: batch %d, max_pages %d, num_pages %d, free_capacity %d, num_copies %d", batch,
                max_pages, num_pages, free_capacity, num_copies);
  if (free_capacity < num_pages)
    return fail(PKV_ERR_INVALID_ARGUMENT, "compact_pages: a list of %d places for %d pages", free_capacity, num_pages);
  if (num_copies < num_pages / 2)
    return fail(PKV_ERR_INVALID_ARGUMENT, "compact_pages: copy_src and copy_dst of %d places (num_pages / 2 = %d)",
                num_copies, num_pages / 2);
  const int64_t entries = (int64_t)batch * max_pages;
  if (!page_shares || !free_pages || !num_free || !page_map || !page_shares_out || !free_pages_out || !num_free_out ||
      (num_copies > 0 && (!copy_src || !copy_dst)) || (entries > 0 && (!block_table || !block_table_out)))
    return fail(PKV_ERR_INVALID_ARGUMENT, "compact_pages: null pointer");
  const char* const same = num_free == num_free_out         ? "num_free"
                           : page_shares == page_shares_out ? "page_shares"
                           : free_pages == free_pages_out   ? "free_pages"
                                                            : nullptr;
  if (same) return fail(PKV_ERR_INVALID_ARGUMENT, "compact_pages: %s_out must not be %s", same, same);
  if (!workspace || workspace_size < pkv_page_workspace_bytes(num_pages) || ((uintptr_t)workspace & 3))
    return fail(PKV_ERR_WORKSPACE_TOO_SMALL, "compact_pages: workspace of %zu bytes is smaller than %zu, or misaligned",
                workspace_size, pkv_page_workspace_bytes(num_pages));
  const int64_t table = ints(entries), pages = ints(num_pages), list = ints(free_capacity), moves = ints(num_copies), one = ints(1);
  const Span spans[] = {{"workspace", workspace, (int64_t)pkv_page_workspace_bytes(num_pages)}, {"page_map", page_map, pages},
                        {"page_shares_out", page_shares_out, pages}, {"free_pages_out", free_pages_out, list},
                        {"num_free_out", num_free_out, one}, {"copy_src", copy_src, moves}, {"copy_dst", copy_dst, moves},
                        {"block_table_out", block_table_out, table}, {"page_shares", page_shares, pages},
                        {"free_pages", free_pages, list}, {"num_free", num_free, one},
                        {"block_table", block_table, block_table_out == block_table ? 0 : table}};
  if (const int status = refuse_overlaps("compact_pages", spans, 8)) return status;
  const int chunks = chunks_of(num_pages);
  const CompactArgs a{block_table, page_shares, free_pages, num_free, page_map, block_table_out, page_shares_out,
                      free_pages_out, num_free_out, copy_src, copy_dst, (int32_t*)workspace, entries, num_pages,
                      free_capacity, num_copies, chunks};
  const hipStream_t st = (hipStream_t)stream;
  auto groups = [](int64_t n) { return dim3((unsigned)((n + kThreads - 1) / kThreads)); };
  if (num_pages <= kBitPages) {
    const int64_t share = 2L * kBitThreads, wanted = (entries + num_pages + share - 1) / share, units = pkv::compute_units();
    const size_t lds = bit_bytes((num_pages + 31) / 32);
    if (lds > 64 * 1024) {
      const hipError_t e = hipFuncSetAttribute((const void*)compact_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e != hipSuccess) return fail(PKV_ERR_LAUNCH, "compact_pages: %s", hipGetErrorString(e));
    }
    compact_kernel<<<dim3((unsigned)(wanted < units ? wanted : units)), dim3(kBitThreads), lds, st>>>(a);
    return launched("compact_pages");
  }
  all_used_kernel<<<groups(num_pages), dim3(kThreads), 0, st>>>(a);
  unused_kernel<<<groups(free_capacity), dim3(kThreads), 0, st>>>(a);
  count_kernel<false><<<dim3((unsigned)chunks), dim3(kThreads), 0, st>>>(page_map, num_pages, a.counts);
  place_kernel<<<dim3((unsigned)chunks), dim3(kThreads), 0, st>>>(a);
  const int64_t work = entries > num_pages ? entries : num_pages, most = 8L * pkv::compute_units() * kThreads;
  remap_kernel<<<groups(work < most ? work : most), dim3(kThreads), 0, st>>>(a);
  return launched("compact_pages");
}

int pkv_copy_pages(const int32_t* copy_src, const int32_t* copy_dst, void* k_pages, void* v_pages,
                   float* kv_scales, int32_t num_copies, int32_t num_pages, int32_t num_kv_heads,
                   int32_t page_size, int32_t head_dim, int32_t element_bytes, void* stream) {
  using pkv::fail;
  if (num_copies < 0 || num_pages <= 0 || num_kv_heads <= 0 || page_size <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "copy_pages: num_copies %d, num_pages %d, num_kv_heads %d, page_size %d",
                num_copies, num_pages, num_kv_heads, page_size);
  if (head_dim != PKV_HEAD_DIM) return fail(PKV_ERR_UNSUPPORTED, "copy_pages: head_dim %d (only 128)", head_dim);
  if (element_bytes != 1 && element_bytes != 2)
    return fail(PKV_ERR_INVALID_ARGUMENT, "copy_pages: elements of %d bytes (1 or 2)", element_bytes);
  const int64_t page_bytes = (int64_t)num_kv_heads * page_size * PKV_HEAD_DIM * element_bytes;
  if (page_bytes > INT32_MAX) return fail(PKV_ERR_UNSUPPORTED, "copy_pages: a page of 2 GiB or more");
  if (num_copies == 0) return pkv::ok();
  if (!copy_src || !copy_dst || !k_pages || !v_pages) return fail(PKV_ERR_INVALID_ARGUMENT, "copy_pages: null pointer");
  if ((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) || ((uintptr_t)kv_scales & 3))
    return fail(PKV_ERR_INVALID_ARGUMENT, "copy_pages: K and V must be 16-byte aligned");
  // 16 KB a workgroup, or 4 KB where that leaves CUs without one.
  constexpr int kLine = kThreads * 16;
  const bool few = 2L * num_copies * ((page_bytes + 4 * kLine - 1) / (4 * kLine)) < 2L * pkv::compute_units();
  const int64_t slice = few ? kLine : 4 * kLine, slices = (page_bytes + slice - 1) / slice;
  const CopyArgs a{copy_src, copy_dst, {(uint8_t*)k_pages, (uint8_t*)v_pages}, kv_scales, page_bytes, num_copies,
                   num_pages, num_kv_heads, (int32_t)slices};
  const int64_t units = 2L * num_copies * slices, most = 16L * pkv::compute_units();
  auto* const kernel = few ? copy_kernel<1> : copy_kernel<4>;
  kernel<<<dim3((unsigned)(units < most ? units : most)), dim3(kThreads), 0, (hipStream_t)stream>>>(a);
  return launched("copy_pages");
}

}  // extern "C"
