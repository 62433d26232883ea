// pkv_tables.hip — block tables, token offsets and slot map of a step, built on the GPU.
//
// The reference builds its metadata on the host (tests/benchmark_serving_trace.py:668-780),
// from lengths it holds there.  A serving loop whose lengths live on the GPU needs the pages
// of the new tokens and their slots without a copy to the host:
//   new_b  = max(0, seq_lens[b] - cached_lens[b])          tokens of row b in this step
//   held_b = min(ceil(cached_b / ps), max_pages)           pages its table row has already
//   need_b = min(ceil(seq_b / ps), max_pages) - held_b     pages it takes from the list
// Row b's j-th new page is free_pages[num_free - 1 - sum_{c<b} need_c - j], its tokens start at
// sum_{c<b} new_c in packed order.
//
// One launch, no atomics.  Every workgroup scans all rows' (new, need) into LDS by itself (two
// coalesced loads a row, from L2 for all workgroups but the first), then takes its share of
// the packed tokens and of the new pages, finding a token's row by bisection in LDS.  That
// repeats the scan, at most 8000 rows, and saves the second launch and the wait on a global
// prefix that a shared scan would need.  What bounds it is latency: lengths, a page id and
// the store follow one another.  64 rows of one new token: 4.9 us (launch to end); 48 rows
// of 331,000 new tokens, 1.5 MB: 7.3 us.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pkv.h"

namespace pkv {
int fail(int status, const char* fmt, ...);  // pkv_decode.hip: sets pkv_last_error()
int ok();
}  // namespace pkv

namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxRows = 8000;         // two LDS prefixes of 4 bytes a row: just under 64 KiB
constexpr int kTokensPerThread = 4;
constexpr uint32_t kTop = 0x7fffffffu;

struct TableArgs {
  const int32_t* cached_lens;  // [B]
  const int32_t* seq_lens;     // [B]
  const int32_t* free_pages;   // [free_capacity]
  const int32_t* num_free;     // [1]
  int32_t* block_table;        // [B, max_pages]
  int32_t* token_offsets;      // [B + 1]
  int32_t* slot_mapping;       // [slots]
  int32_t* num_free_out;       // [1]
  int32_t batch, free_capacity, max_pages, slots, page_size;
  int32_t page_shift;  // log2(page_size), or -1
};

// Sums that stop at 2^31 - 1 (addends of at most that much each; associative).
__device__ inline uint32_t add_sat(uint32_t a, uint32_t b) { return min(a + b, kTop); }

__device__ inline int page_index(const TableArgs& a, int token) {
  return a.page_shift >= 0 ? token >> a.page_shift : token / a.page_size;
}
__device__ inline int pages_of(const TableArgs& a, int tokens) {
  const int p = page_index(a, tokens);
  return min(p + (p * a.page_size < tokens), a.max_pages);
}

// Inclusive saturating sum over the wave by DPP: within rows of 16 lanes, then across them.
template <int CTRL, int ROW_MASK>
__device__ inline uint32_t dpp_add_sat(uint32_t x) {
  return add_sat(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROW_MASK, 0xf, false));
}
__device__ inline uint32_t wave_scan(uint32_t x) {
  x = dpp_add_sat<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x = dpp_add_sat<0x112, 0xf>(x);
  x = dpp_add_sat<0x114, 0xf>(x);
  x = dpp_add_sat<0x118, 0xf>(x);
  x = dpp_add_sat<0x142, 0xa>(x);  // row_bcast 15, 31
  return dpp_add_sat<0x143, 0xc>(x);
}

__device__ inline void row_counts(const TableArgs& a, int row, uint32_t& tokens, uint32_t& pages) {
  const int cached = max(a.cached_lens[row], 0), len = max(a.seq_lens[row], cached);
  tokens = (uint32_t)(len - cached);
  pages = (uint32_t)(pages_of(a, len) - pages_of(a, cached));
}

// For N values x at once: the last row whose prefix is at most x (rows without elements share
// their successor's prefix and are passed over).  `top`: the largest power of two below n,
// or 0; the steps of the N bisections are independent LDS reads.
template <int N>
__device__ inline void rows_of(const uint32_t* prefix, int n, int top, const uint32_t (&x)[N], int (&row)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) row[i] = 0;
  for (int step = top; step; step >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = row[i] + step;
      if (at < n && prefix[at] <= x[i]) row[i] = at;
    }
  }
}

__global__ __launch_bounds__(kThreads) void tables_kernel(TableArgs a) {
  extern __shared__ uint32_t lds[];
  uint32_t* const tok = lds;                    // [B + 1] exclusive prefix of new tokens
  uint32_t* const pag = lds + a.batch + 1;      // [B + 1] exclusive prefix of new pages
  uint32_t* const sums = pag + a.batch + 1;     // [2 * kWaves]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int avail = min(max(*a.num_free, 0), a.free_capacity);

  uint32_t tok0 = 0, pag0 = 0;
  for (int base = 0; base < a.batch; base += kThreads) {
    const int row = base + tid;
    uint32_t t = 0, p = 0;
    if (row < a.batch) row_counts(a, row, t, p);
    const uint32_t ti = wave_scan(t), pi = wave_scan(p);
    if (lane == 63) sums[wave] = ti, sums[kWaves + wave] = pi;
    __syncthreads();
    uint32_t tw = tok0, pw = pag0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) tw = add_sat(tw, sums[w]), pw = add_sat(pw, sums[kWaves + w]);
      tok0 = add_sat(tok0, sums[w]), pag0 = add_sat(pag0, sums[kWaves + w]);
    }
    if (row < a.batch) {
      tok[row + 1] = add_sat(tw, ti);
      pag[row + 1] = add_sat(pw, pi);
    }
    __syncthreads();
  }
  if (tid == 0) tok[0] = 0, pag[0] = 0;
  __syncthreads();

  const uint32_t total_tok = tok[a.batch], total_pag = pag[a.batch];
  const uint32_t gid = blockIdx.x * kThreads + tid, threads = gridDim.x * kThreads;

  for (uint32_t i = gid; i <= (uint32_t)a.batch; i += threads) a.token_offsets[i] = (int32_t)tok[i];
  if (gid == 0) {
    *a.num_free_out = avail - (int32_t)total_pag;  // at least -(2^31 - 1)
  }
  const int top = a.batch > 1 ? 1 << (31 - __builtin_clz(a.batch - 1)) : 0;
  // The new pages of the table rows.
  for (uint32_t r = gid; r < total_pag; r += threads) {
    int row[1];
    rows_of<1>(pag, a.batch, top, {r}, row);
    const int held = pages_of(a, max(a.cached_lens[row[0]], 0));
    const long at = (long)avail - 1 - (long)r;
    a.block_table[(long)row[0] * a.max_pages + held + (int)(r - pag[row[0]])] = at >= 0 ? a.free_pages[at] : -1;
  }
  // The slots.  A new page's id comes from the list, not from the table, whose new entries
  // another workgroup may not have written yet.
  for (uint32_t base = blockIdx.x * kThreads * kTokensPerThread; base < (uint32_t)a.slots;
       base += threads * kTokensPerThread) {
    uint32_t t[kTokensPerThread];
    int row[kTokensPerThread], slot[kTokensPerThread];
#pragma unroll
    for (int i = 0; i < kTokensPerThread; ++i) t[i] = base + i * kThreads + tid;
    rows_of<kTokensPerThread>(tok, a.batch, top, t, row);
#pragma unroll
    for (int i = 0; i < kTokensPerThread; ++i) {
      slot[i] = -1;
      if (t[i] < min(total_tok, (uint32_t)a.slots)) {
        const int cached = max(a.cached_lens[row[i]], 0);
        const int pos = cached + (int)(t[i] - tok[row[i]]);
        const int logical = page_index(a, pos), held = pages_of(a, cached);
        if (logical < a.max_pages) {
          const long at = (long)avail - 1 - (long)pag[row[i]] - (logical - held);
          const int32_t* p = logical < held ? a.block_table + (long)row[i] * a.max_pages + logical
                                            : a.free_pages + at;
          const int page = logical < held || at >= 0 ? *p : -1;
          const long s = (long)page * a.page_size + (pos - logical * a.page_size);
          if (page >= 0 && s <= INT32_MAX) slot[i] = (int32_t)s;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kTokensPerThread; ++i)
      if (t[i] < (uint32_t)a.slots) a.slot_mapping[t[i]] = slot[i];
  }
}

}  // namespace

extern "C" int pkv_build_block_tables(
    const int32_t* cached_lens, const int32_t* seq_lens, const int32_t* free_pages,
    const int32_t* num_free, int32_t* block_table, int32_t* token_offsets, int32_t* slot_mapping,
    int32_t* num_free_out, int32_t batch, int32_t free_capacity, int32_t max_pages, int32_t slots,
    int32_t page_size, void* stream) {
  using pkv::fail;
  if (batch < 0 || free_capacity < 0 || max_pages <= 0 || slots < 0 || page_size <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT,
                "build_block_tables: batch %d, free_capacity %d, max_pages %d, slots %d, page_size %d",
                batch, free_capacity, max_pages, slots, page_size);
  if (batch > kMaxRows)
    return fail(PKV_ERR_UNSUPPORTED, "build_block_tables: batch %d (at most %d)", batch, kMaxRows);
  if (!num_free || !num_free_out || !token_offsets || (slots > 0 && !slot_mapping) ||
      (free_capacity > 0 && !free_pages) ||
      (batch > 0 && (!cached_lens || !seq_lens || !block_table)))
    return fail(PKV_ERR_INVALID_ARGUMENT, "build_block_tables: null pointer");
  if (num_free == num_free_out)
    return fail(PKV_ERR_INVALID_ARGUMENT, "build_block_tables: num_free_out must not be num_free");
  const TableArgs a{cached_lens, seq_lens, free_pages, num_free, block_table, token_offsets,
                    slot_mapping, num_free_out, batch, free_capacity, max_pages, slots, page_size,
                    (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1};
  const long work = (long)(slots > batch ? slots : batch);
  long groups = (work + kThreads * kTokensPerThread - 1) / (kThreads * kTokensPerThread);
  groups = groups < 1 ? 1 : groups > 1024 ? 1024 : groups;
  const size_t bytes = (size_t)(2 * (batch + 1) + 2 * kWaves) * sizeof(uint32_t);
  tables_kernel<<<dim3((unsigned)groups), dim3(kThreads), bytes, (hipStream_t)stream>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? pkv::ok()
                         : fail(PKV_ERR_LAUNCH, "build_block_tables launch: %s", hipGetErrorString(e));
}
