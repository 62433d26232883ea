// pkv_chunk.hip — attention of the newest tokens of every row over the row's pages, which hold
// them already: a second turn over a cached prefix, a piece of a long prompt, guessed tokens that
// are checked at once, single tokens among them (the reference has one token a row only,
// cuh:294-459).
//
//   o[i] = sum_{j <= p_i, j < L} softmax_j(q[i] k[j] / sqrt(128)) v[j],  p_i = L - n + i
//
// for the n newest of a row's L tokens; a token that sees no key gives 0.
//
// The products are those of the prompt attention (pkv_prefill.hip): rows of work are the (token,
// head of the group) pairs of a KV head, S^T = K Q^T and O^T += V^T P^T on 32x32x16 tiles, K/V
// tiles of 32 keys straight to LDS in a ring of three.  What is new:
//
// Pages.  A tile's keys lie in any pages, whose ids are in LDS (a window of the row's table, renewed
// every 512 pages).  A wave moves eight keys at a time: in pages of a multiple of 8 they lie in one
// page, whose place is scalar arithmetic; else, and at the row's end, every lane computes its key's
// (that for all tiles: 2048 tokens over 32768 in 1174 us instead of 1012).  Keys past the row's end
// read its last key again; their weights are 0.
//
// Splits.  Rows differ in length by orders of magnitude and a call may have very few rows, so work
// is cut by keys as well: with W tiles in all blocks of the call (as if every block saw all keys)
// and P parts wanted, two for every compute unit (more where parts are long, see kLongPart), a
// workgroup takes at most C = W / P tiles of a small row and, since large rows are cut into the
// nearest number of parts, less than 1.5 C of a large one.  All workgroups compute C and their own
// part from the lengths on the GPU.  The parts of a block leave their sums in the workspace in 32 bits,
// and a second kernel joins them.  Parts cost: the states of 128 rows are 66 KB each way, as much
// as a workgroup's 30 tiles, so more parts than the compute units ask for are slower (512 tokens
// over 8192: 512 parts 84 us, 768 88, 256 117), but rows of one wave at most (decoding rows,
// guessed tokens) cost little and are counted apart.  Large and small rows take turns, two to one,
// so that the ones' products run next to the others' reads (28 single tokens and 4 pieces of 512
// over up to 8192, weights in one term: 238 us; one after the other 280, in equal turns 270).
//
// P enters the product with V in the activation type.  Large rows, which wait for products, round it
// once, as the prompt attention does: bf16 outputs are 2.3e-3 from the exact ones (relative 2-norm;
// 1.7e-3 is the output's own rounding), fp16 2.7e-4 (2.1e-4).  Rows of one wave, which wait for memory,
// give bf16 P in two terms, as the decode kernels do, and are as exact as the output's rounding (1.66e-3
// of 1.66e-3) for 3 % (64 single tokens of 128-65536 keys, 32 / 4 heads: 331 us, 323 with one term; the
// 28 single tokens next to four pieces of 512: 249 for 239).
//
// Measured (bf16, 32 / 8 heads, pages of 16): 2048 tokens over 32768 1.00 ms, 1.06 PFLOP/s, the matrix
// units busy 57 % of the cycles; a CU's step takes 0.5 us with two workgroups and with three.  64 single
// tokens of 128-65536 keys (32 / 4 heads) 4.8 TB/s, where a copy reaches 5.1.  5 tokens over 2011: 11.3
// us, 7.7 of it the first kernel (four dependent reads before the first product), 3.6 the join.

#include <hip/hip_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>
#include <type_traits>

#include "pkv.h"
#include "pkv_attention_tile.h"
#include "pkv_device.h"

namespace pkv {
int fail(int status, const char* fmt, ...);  // pkv_decode.hip: sets pkv_last_error()
int ok();
}  // namespace pkv

namespace {

constexpr int kRows = kWaves * kWaveRows;  // of a block
constexpr int kIds = 512;                  // page ids in LDS
constexpr int kMinTiles = 2;               // of a part: 5 tokens over 2011 11.5 us, with 4 12.0, with 8 14.7
constexpr int kSmallBatch = 64;            // rows of a table whose plan every wave makes for itself
constexpr int kStateFloats = kD + 2;       // of one row: its sums, maximum and sum of weights

typedef float f32x4 __attribute__((ext_vector_type(4)));

// x / d for 0 <= x < 2^31 as mulhi(2 x, magic) >> shift: with 2^shift the power of two at or above d and
// magic = ceil(2^(31 + shift) / d), which is below 2^32, the error x (magic d - 2^(31 + shift)) is below
// 2^(31 + shift).
struct Divisor {
  uint32_t magic, shift;
};
__device__ inline int quotient(int x, Divisor d) { return (int)(__umulhi(2 * (uint32_t)x, d.magic) >> d.shift); }

struct ChunkArgs {
  const uint8_t* q;  // token t, head h at q + t * q_stride + h * 256 (bytes)
  const uint8_t* k_pages;  // [num_pages, Hkv, ps, 128]
  const uint8_t* v_pages;
  const int32_t* block_table;    // [B, max_pages]
  const int32_t* seq_lens;       // [B]
  const int32_t* token_offsets;  // [B + 1]
  uint8_t* output;               // [T, Hq, 128]
  int32_t* plan;                 // of more than kSmallBatch rows
  float* sums;                   // [state rows, Hkv, 128]
  float* tops;                   // [state rows, Hkv, 2]: maximum, sum of weights
  long q_stride;
  int32_t batch, tokens, hq, hkv, group, num_pages, max_pages, page_size;
  uint32_t page_bytes;
  Divisor by_page, by_group, by_heads;  // page_size, group, hkv
  float inv_group;
  float heads_per_part;  // Hkv / P, and a little more
};

// A row of the table: its n tokens of the call from `start` on, the first at position `before`
// (negative where more tokens are called new than the row has), and the keys that it has.
struct Seq {
  int start, n, before, len;
};
__device__ inline int offset_of(const ChunkArgs& a, int b) { return min(max(a.token_offsets[b], 0), a.tokens); }
__device__ inline Seq seq_of(const ChunkArgs& a, int b) {
  const int start = offset_of(a, b), n = max(offset_of(a, b + 1) - start, 0), total = max(a.seq_lens[b], 0);
  return {start, n, total - n, min(total, a.max_pages * a.page_size)};
}
__device__ inline int tiles_of(int len) { return (int)(((uint32_t)len + kKeys - 1) / kKeys); }
__device__ inline int blocks_of(const ChunkArgs& a, int n) { return (int)(((uint32_t)(n * a.group) + kRows - 1) / kRows); }

template <int CTRL, int ROW_MASK>
__device__ inline float add_lane(float x) {  // 0 where the lane has no source
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, ROW_MASK, 0xf, false));
}
__device__ inline float wave_sum(float x) {
  x = add_lane<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8; row_bcast 15, 31
  x = add_lane<0x112, 0xf>(x);
  x = add_lane<0x114, 0xf>(x);
  x = add_lane<0x118, 0xf>(x);
  x = add_lane<0x142, 0xa>(x);
  x = add_lane<0x143, 0xc>(x);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
// x / d for 0 <= x < 2^31, d > 0: the product with 1 / d is off by at most 2^-22 of the result, a
// second one for what is left over by one.
__device__ inline int divide(int x, int d) {
  const float inv = __builtin_amdgcn_rcpf((float)d);
  int y = (int)((float)x * inv), r = x - y * d;
  const int more = (int)floorf((float)r * inv);
  y += more, r -= more * d;
  return y + (r >= d) - (r < 0);
}

// Rows whose tokens are one wave's ("small": decoding rows, guessed tokens) and others have budgets of
// their own: a small row's parts cost little memory, and cut finer than long pieces of prompts they
// fill the compute units that those leave.
__device__ inline bool is_small(const ChunkArgs& a, const Seq& s) { return s.n * a.group <= kWaveRows; }
__device__ inline float tiles_in(const ChunkArgs& a, const Seq& s) { return (float)blocks_of(a, s.n) * (float)tiles_of(s.len); }
struct Cut {
  int large, small;  // the most tiles of a part
};
// C for the sum of blocks times tiles of a class and one KV head: a little more than W / P, so that the
// roundings of the sum (less than 2^-17 of it) never make more parts than the grid and the workspace hold.
// Large rows whose parts would be longer than kLongPart tiles have up to kFiner times as many: the GPU
// deals them out as it goes, and rows end together (12 rows of 1073 tokens over up to 22304, 6 / 2 heads:
// 518 us, 624 with P parts; 8 of 1024 over 4096-32768 2.31 ms and 2.41; of equal lengths 4 of 1024 over
// 16384 1.03 and 1.09, 2048 over 32768 1.005 and 1.014, its 136 MB of states among them).
constexpr int kLongPart = 192, kFiner = 4;
__device__ inline int part_tiles(float c) { return max(kMinTiles, (int)fminf(ceilf(c), 1e9f)); }
__device__ inline Cut cut_of(const ChunkArgs& a, float large, float small) {
  const float c = large * a.heads_per_part;
  return {part_tiles(fmaxf(c * (1.0f / kFiner), fminf(c, (float)kLongPart))), part_tiles(small * a.heads_per_part)};
}
__device__ inline int ratio_up(int x, int d) { return divide(x + d - 1, d); }
// A row's parts, as even as whole tiles are: as many as keep them to C for small rows, and the nearest
// number for large ones, whose parts cost more (4 x 64 tokens over 8192-16384: 76 us, 86 with as many
// as keep them to C; 8 x 5 tokens over up to 32768: 63 and 53).
struct Parts {
  int count, tiles;
};
__device__ inline Parts parts_of(const ChunkArgs& a, const Seq& s, const Cut& cut) {
  const int tiles = tiles_of(s.len), most = is_small(a, s) ? cut.small : cut.large;
  const int count = max(divide(tiles + (is_small(a, s) ? most - 1 : most >> 1), most), 1);
  return {count, max(ratio_up(tiles, count), 1)};
}

// What a row adds to the plan's running sums: units of work (blocks by parts), rows of states in the
// workspace, and rows to join.
struct Share {
  int units, states, joins;
};
__device__ inline Share share_of(const ChunkArgs& a, const Seq& s, const Cut& cut) {
  const int parts = parts_of(a, s, cut).count, rows = parts > 1 ? s.n * a.group : 0;
  return {blocks_of(a, s.n) * parts, rows * parts, rows};
}

// The plan in memory: the cut; the units before every row of the table, the large rows' first, then
// the small ones' (2 batch + 1 numbers); the states and the joins before every row (batch + 1 each).
__device__ inline int32_t* units_before(const ChunkArgs& a) { return a.plan + 2; }
__device__ inline int32_t* states_before(const ChunkArgs& a) { return a.plan + 3 + 2 * a.batch; }
__device__ inline int32_t* joins_before(const ChunkArgs& a) { return a.plan + 4 + 3 * a.batch; }

constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(ChunkArgs a) {
  constexpr int kPlanWaves = kPlanThreads / 64;
  __shared__ float total[2][kPlanWaves];
  __shared__ int sums[3][kPlanWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  double many[2] = {0., 0.};
  for (int b = tid; b < a.batch; b += kPlanThreads) {
    const Seq s = seq_of(a, b);
    many[is_small(a, s)] += (double)tiles_in(a, s);
  }
  float tiles[2] = {(float)many[0], (float)many[1]};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    tiles[i] = wave_sum(tiles[i]);
    if (lane == 0) total[i][wave] = tiles[i];
  }
  __syncthreads();
  tiles[0] = tiles[1] = 0.f;
  for (int w = 0; w < kPlanWaves; ++w) tiles[0] += total[0][w], tiles[1] += total[1][w];
  const Cut cut = cut_of(a, tiles[0], tiles[1]);
  int before[3] = {0, 0, 0};
  int32_t* const to[3] = {units_before(a), states_before(a), joins_before(a)};
  for (int base = 0; base <= 2 * a.batch; base += kPlanThreads) {
    const int e = base + tid, b = e < a.batch ? e : e - a.batch;
    int mine[3] = {0, 0, 0}, sum[3];
    if (e < 2 * a.batch) {
      const Seq s = seq_of(a, b);
      const Share x = share_of(a, s, cut);
      if (is_small(a, s) == (e >= a.batch)) mine[0] = x.units;
      if (e < a.batch) mine[1] = x.states, mine[2] = x.joins;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      sum[i] = wave_scan(mine[i]);
      if (lane == 63) sums[i][wave] = sum[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      int at = before[i] + sum[i] - mine[i];
      for (int w = 0; w < kPlanWaves; ++w) {
        if (w < wave) at += sums[i][w];
        before[i] += sums[i][w];
      }
      if (e <= (i == 0 ? 2 : 1) * a.batch) to[i][e] = at;
    }
    __syncthreads();
  }
  if (tid == 0) a.plan[0] = cut.large, a.plan[1] = cut.small;
}

// The plan of up to kSmallBatch rows, lane b's row, made by every wave for itself.
struct LanePlan {
  Seq seq;
  Cut cut;
  Share share;
  bool small;
};
__device__ inline LanePlan lane_plan(const ChunkArgs& a, int lane) {
  LanePlan p{};
  if (lane < a.batch) p.seq = seq_of(a, lane);
  p.small = is_small(a, p.seq);
  const float tiles = tiles_in(a, p.seq);
  p.cut = cut_of(a, wave_sum(p.small ? 0.f : tiles), wave_sum(p.small ? tiles : 0.f));
  p.share = share_of(a, p.seq, p.cut);
  return p;
}

// A unit of work: part `part`, of `tiles` tiles, of block `block` of a row of the table.  block < 0: none.
struct Unit {
  Seq seq;
  int row, block, part, tiles, states;
};

__device__ inline Seq seq_from(const Seq& s, int lane) {
  return {__builtin_amdgcn_readlane(s.start, lane), __builtin_amdgcn_readlane(s.n, lane),
          __builtin_amdgcn_readlane(s.before, lane), __builtin_amdgcn_readlane(s.len, lane)};
}

// Which unit of its class the `slot`-th is: two of large rows, which wait for products, then one of
// small ones, which wait for memory, as long as there are both.
struct Turn {
  bool small;
  int unit;  // negative: none
};
__device__ inline Turn turn_of(int slot, int large, int small) {
  const int thirds = min(large >> 1, small), third = (int)(__umulhi((uint32_t)slot, 0xaaaaaaabu) >> 1);
  if (third < thirds) {
    const int r = slot - 3 * third;
    return r < 2 ? Turn{false, 2 * third + r} : Turn{true, third};
  }
  slot -= thirds;  // less the small ones
  if (slot < large) return {false, slot};
  slot -= large - thirds;  // the small ones again, less the large
  return {true, slot < small ? slot : -1};
}

// Units go through the rows of their class; a row's part by part, a part's last block first: the
// blocks at work at one time share their keys in L2.
__device__ inline Unit unit_of(const ChunkArgs& a, int slot, int lane) {
  Unit u;
  u.block = -1;
  Cut cut;
  if (a.batch <= kSmallBatch) {
    const LanePlan p = lane_plan(a, lane);
    const int large = wave_scan(p.small ? 0 : p.share.units), small = wave_scan(p.small ? p.share.units : 0);
    const Turn t = turn_of(slot, __builtin_amdgcn_readlane(large, 63), __builtin_amdgcn_readlane(small, 63));
    if (t.unit < 0) return u;
    const int units = t.small ? small : large, own = t.small == p.small ? p.share.units : 0;
    slot = t.unit;
    const int states = wave_scan(p.share.states);
    u.row = __builtin_ctzll(__builtin_amdgcn_ballot_w64(units > slot));
    u.seq = seq_from(p.seq, u.row);
    u.states = __builtin_amdgcn_readlane(states - p.share.states, u.row);
    slot -= __builtin_amdgcn_readlane(units - own, u.row);
    cut = p.cut;
  } else {
    // The last row whose first unit is at most `slot` (rows without units share the next one's),
    // found among 64 candidates at a time.
    const int32_t* const first = units_before(a);
    const int large = uniform(first[a.batch]);
    const Turn t = turn_of(slot, large, uniform(first[2 * a.batch]) - large);
    if (t.unit < 0) return u;
    slot = t.unit + (t.small ? large : 0);
    int b = 0, n = 2 * a.batch;
    while (n > 1) {
      const int stride = (n + 63) / 64, at = b + lane * stride;
      const uint64_t fits = __builtin_amdgcn_ballot_w64(lane * stride < n && first[min(at, 2 * a.batch)] <= slot);
      const int found = 63 - __builtin_clzll(fits);  // the first candidate always fits
      n = min(stride, n - found * stride);
      b += found * stride;
    }
    b = uniform(b);
    slot -= uniform(first[b]);
    u.row = b < a.batch ? b : b - a.batch;
    u.seq = seq_of(a, u.row);
    u.states = uniform(states_before(a)[u.row]);
    cut = {uniform(a.plan[0]), uniform(a.plan[1])};
  }
  u.tiles = parts_of(a, u.seq, cut).tiles;
  const int blocks = blocks_of(a, u.seq.n);
  u.part = divide(slot, blocks);
  u.block = blocks - 1 - (slot - u.part * blocks);
  return u;
}

// The last key that token i of a row sees; -1: none.
__device__ inline int last_key(const Seq& s, int i) { return max(min(s.before + i, s.len - 1), -1); }

// 64 x 16 bytes straight to LDS, lane l's to `lds` + 16 l.  In assembly because the compiler lets
// every LDS read wait for every such load in flight; landed() is the wait.  m0, which nothing else in
// these kernels uses, must be one wait state old, and a scalar register that a vector instruction has
// written (a descriptor's or base's, by readfirstlane or as a spilled one brought back) five: the
// compiler keeps no distances to instructions in assembly, so this text carries them.
__device__ inline void load_to_lds(uint32_t lds, const uint8_t* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(lds), "v"(from) : "memory");
}
__device__ inline void load_to_lds(uint32_t lds, const uint8_t* base, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds), "v"(offset), "s"(base) : "memory");
}

// The lane's number, made anew where it is asked for: what follows from it is then neither kept
// in registers from tile to tile nor computed before the first one and spilled.
__device__ inline int fresh_lane() {
  int x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
  return x;
}

// x with the bit BIT the other way, likewise not kept: it seems to depend on the step.
template <int BIT>
__device__ inline uint32_t flipped(uint32_t x, int step) {
  uint32_t y;
  asm("v_xor_b32 %0, %2, %1" : "=v"(y) : "v"(x), "n"(BIT), "s"(step));
  return y;
}

template <class Elem>
__global__ __launch_bounds__(kWaves * 64, 3) void chunk_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kBuffers * 2 * kTileBytes];  // K and V of a tile
  __shared__ int ids[kIds];
  __shared__ int failed[kWaves];
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int slot = quotient((int)blockIdx.x, a.by_heads), kvh = (int)blockIdx.x - slot * a.hkv;
  const Unit u = unit_of(a, slot, lane);
  if (u.block < 0) return;
  const int start = uniform(u.seq.start), n = uniform(u.seq.n), len = uniform(u.seq.len);
  const Seq seq{start, n, uniform(u.seq.before), len};
  const int block = uniform(u.block), rows = n * a.group;
  // bf16 weights of rows that are one wave's: rounded, and the rest rounded again.
  const bool two_terms = std::is_same_v<Elem, BFloat> && rows <= kWaveRows;

  // Row row0 + r of the wave is token tok0 + (rem + r) / G: a quotient of numbers below 64, which
  // the product with 1 / G in 32 bits gives exactly (it is off by less than 1 / (2 G)).
  const int row0 = uniform(min(block * kRows + wave * kWaveRows, rows));
  const int tok0 = quotient(row0, a.by_group), rem = row0 - tok0 * a.group, live = rows - row0;  // may be 0
  auto token_of = [&](int r) { return (int)(((float)(rem + r) + 0.5f) * a.inv_group); };
  const int last_row = max(min(kWaveRows, live) - 1, 0);
  const int r = min(col, last_row), dt = token_of(r);
  const int tok = min(tok0 + dt, n - 1);  // a wave past the last row takes the last token's
  const int see = last_key(seq, tok);
  const int wave_first = last_key(seq, min(tok0, n - 1));
  const int wave_last = live > 0 ? last_key(seq, tok0 + uniform(token_of(last_row))) : -1;
  const int block_tiles = tiles_of(last_key(seq, quotient(min((block + 1) * kRows, rows) - 1, a.by_group)) + 1);
  const int part = uniform(u.part), most = uniform(u.tiles), tile0 = part * most;
  if (part > 0 && tile0 >= block_tiles) return;
  const int end = min(block_tiles, tile0 + most);
  const bool whole = block_tiles <= most;
  const int tiles = end - tile0;

  // A wave moves rows kMoved wave + 4 i + lane / 16 of a tile, 256 bytes a row.  16-byte chunk p of
  // row r in LDS is chunk p ^ r of K's row (p ^ 4 r of V's), so that reads of one chunk column
  // (K) or of 64 bytes of four rows (V) spread over all banks.
  constexpr int kMoved = kKeys / kWaves;
  constexpr int kLoads = kMoved / 4;  // per wave and tile of K, and of V
  const uint32_t lds0 = (uint32_t)uniform((int)((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds +
                                                (uint32_t)(wave * kMoved * kRowBytes)));
  const uint32_t head = (uint32_t)(kvh * a.page_size) * kRowBytes;
  const int32_t* const table = a.block_table + (long)u.row * a.max_pages;
  // ids[] holds the pages from `first_id` on, of the tiles before `id_end`.
  const int window = (int)min((long)(kIds - 1) * a.page_size / kKeys, 1L << 26);
  int first_id = 0, id_end = 0;
  auto renew_ids = [&](int tile) __attribute__((always_inline)) {
    first_id = uniform(quotient(tile * kKeys, a.by_page));
    id_end = tile + window;
    const int last = quotient(len - 1, a.by_page);
    for (int i = wave * 64 + fresh_lane(); i < kIds && first_id + i <= last; i += kWaves * 64)
      ids[i] = min(max(table[first_id + i], 0), a.num_pages - 1);
    __syncthreads();
  };
  // A wave's rows of a tile are eight keys in a row.  In pages of a multiple of 8 they lie in one page,
  // whose place is found once for all lanes; else, and at the row's end, every lane finds its own.
  static_assert(kMoved == 8 && kLoads == 2);
  const uint32_t row_in = (uint32_t)lane >> 4, swizzle = (8 * (wave & 1) + row_in) ^ ((uint32_t)lane & 15);
  const uint32_t koff = row_in * kRowBytes + (swizzle << 4);
  const uint32_t voff = row_in * kRowBytes + ((((uint32_t)lane & 15) ^ (row_in << 2)) << 4);
  const bool eights = a.page_size % 8 == 0;
  auto fetch = [&](int i, int buf) __attribute__((always_inline)) {  // the i-th tile
    const uint32_t to = lds0 + buf * 2 * kTileBytes;
    const int key0 = (tile0 + i) * kKeys + wave * kMoved;
    if (eights && key0 + kMoved <= len) {
      const int page = quotient(key0, a.by_page);
      const uint64_t at = (uint64_t)(uint32_t)uniform(ids[page - first_id]) * a.page_bytes +
                          (head + (uint32_t)(key0 - page * a.page_size) * kRowBytes);
      const uint8_t* const k = a.k_pages + at;
      const uint8_t* const v = a.v_pages + at;
      load_to_lds(to, k, koff);
      load_to_lds(to + 4 * kRowBytes, k + 4 * kRowBytes, koff ^ 64);
      load_to_lds(to + kTileBytes, v, voff);
      load_to_lds(to + kTileBytes + 4 * kRowBytes, v + 4 * kRowBytes, voff);
    } else {
      const int l = fresh_lane(), chunk = l & 15;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int srow = wave * kMoved + 4 * j + (l >> 4);
        const int key = min((tile0 + i) * kKeys + srow, len - 1), page = quotient(key, a.by_page);
        const uint64_t at = (uint64_t)(uint32_t)ids[page - first_id] * a.page_bytes +
                            (head + (uint32_t)(key - page * a.page_size) * kRowBytes);
        load_to_lds(to + j * 4 * kRowBytes, a.k_pages + at + ((chunk ^ (srow & 15)) << 4));
        load_to_lds(to + kTileBytes + j * 4 * kRowBytes, a.v_pages + at + ((chunk ^ ((srow & 3) << 2)) << 4));
      }
    }
  };

  u32x4 q[8];
  const uint8_t* qp = a.q + (start + (long)tok) * a.q_stride +
                      (long)(kvh * a.group + rem + r - dt * a.group) * kRowBytes + half * 16;
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) q[kk] = *(const u32x4*)(qp + kk * 32);

  // Reads: lane's K row (key col), chunk 2 kk + half; V rows 4 half + (lane % 16) / 4, four
  // dims from 32 db + 16 (lane / 16 % 2) + 4 (lane % 4) on.
  const uint32_t ksrc = col * kRowBytes + ((half ^ (col & 15)) << 4);
  const int vr = (lane >> 2) & 3;
  const uint32_t vsrc = (4 * half + vr) * kRowBytes + (vr << 6) + ((lane & 16) << 1) + ((lane & 3) << 3);

  f32x16 o[4];
  float m, l;
  bool large = false;  // a row of the wave has a large maximum
  // Half of the addresses; the others differ in one bit, and are made where they are used.
  uint32_t kat[4], vat[2];
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) kat[kk] = lds_at + (ksrc ^ (kk << 5));
#pragma unroll
  for (int db = 0; db < 2; ++db) vat[db] = lds_at + kTileBytes + (vsrc ^ (db << 6));

  // A masked weight is 0, and 0 times an infinity or NaN in V is NaN.  So where a row comes out
  // not finite, its workgroup computes once more, `careful`: such values are taken out of the tiles
  // that a row of it masks in part, those of the steps from `masked` on (the keys read twice past
  // the end among them), and put back at the end for the rows that see their token.  A second term,
  // which may be 0 or negative, never meets them.
  bool careful = false;
  const int masked = max((last_key(seq, quotient(block * kRows, a.by_group)) + 1) / kKeys - tile0, 0);
  auto clean = [&](int buf) {
    u32x4* const v = (u32x4*)(lds + buf * 2 * kTileBytes + kTileBytes) + wave * 64 + fresh_lane();
    for (int i = 0; i < kTileBytes / 16; i += kWaves * 64) {
      u32x4 x = v[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = drop_nonfinite<Elem>(x[j]);
      v[i] = x;
    }
    __syncthreads();
  };

  // The i-th tile, which lies in buffer `buf`, with the weights in `two` terms or in one.  The sum of the
  // weights is that of the rounded ones, or, for two terms, of the weights themselves.  Each has a loop
  // of its own: a branch between the exponentials and the products costs the large rows 3-9 %.
  auto step = [&](auto two, int i, int buf) __attribute__((always_inline)) {
    const int at = buf * 2 * kTileBytes;
    if (careful && i >= masked) clean(buf);
    if (i + 2 < tiles && tile0 + i + 2 >= id_end) {
      __syncthreads();  // the old ids have been read
      renew_ids(tile0 + i + 2);
    }
    if (i + 2 < tiles) fetch(i + 2, buf >= 1 ? buf - 1 : buf + 2);
    const int k0 = (tile0 + i) * kKeys;
    if (k0 <= wave_last) {
      f32x16 s = {};
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const uint32_t k = kk < 4 ? kat[kk] : flipped<128>(kat[kk - 4], i);
        s = Elem::mma(*(const __attribute__((address_space(3))) u32x4*)(k + at), q[kk], s);
      }
      auto value = [&](int c, int db) __attribute__((always_inline)) {  // keys 16 c ..., dims 32 db + lane % 32
        typedef __attribute__((address_space(3))) s16x4* Lds;
        const uint32_t v = (db < 2 ? vat[db] : flipped<128>(vat[db - 2], i)) + at + c * 16 * kRowBytes;
        const u32x2 v0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)v));
        const u32x2 v1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(v + 8 * kRowBytes)));
        return u32x4{v0[0], v0[1], v1[0], v1[1]};
      };
      u32x4 v0[4];
#pragma unroll
      for (int db = 0; db < 4; ++db) v0[db] = value(0, db);
      if (k0 + kKeys - 1 > wave_first) {
        const int visible = see - k0 - 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i >> 2) + (i & 3) > visible) s[i] = -INFINITY;
      }
      float mx = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
      if (__builtin_amdgcn_ballot_w64(mx > m + kSlack) != 0) {
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mn = fmaxf(m, mx);
        const float c = __builtin_amdgcn_exp2f((m - mn) * kScaleLog2);
        m = mn;
        large = __builtin_amdgcn_ballot_w64(fabsf(m) >= kLargeScore) != 0;
        l *= c;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[db][i] *= c;
      }
      float ms = m * kScaleLog2;
      if (large) {
        ms = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] -= m;
      }
      u32x4 p[2];
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], kScaleLog2, -ms));
        s[i + 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + 1], kScaleLog2, -ms));
        const uint32_t x = Elem::pack2(s[i], s[i + 1]);
        p[i >> 3][(i & 7) >> 1] = x;
        l = two.value ? l + (s[i] + s[i + 1]) : Elem::sum2(x, l);
      }
      if constexpr (two.value) {
        u32x4 rest[2];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const uint32_t x = p[i >> 3][(i & 7) >> 1];
          rest[i >> 3][(i & 7) >> 1] = Elem::pack2(s[i] - Elem::widen(x, false), s[i + 1] - Elem::widen(x, true));
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (c > 0)
#pragma unroll
            for (int db = 0; db < 4; ++db) v0[db] = value(c, db);
#pragma unroll
          for (int db = 0; db < 4; ++db) o[db] = Elem::mma(v0[db], p[c], o[db]);
          if (careful)
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
              for (int j = 0; j < 4; ++j) v0[db][j] = drop_nonfinite<Elem>(v0[db][j]);
#pragma unroll
          for (int db = 0; db < 4; ++db) o[db] = Elem::mma(v0[db], rest[c], o[db]);
        }
      } else {
        u32x4 v1[4];
#pragma unroll
        for (int db = 0; db < 4; ++db) {
          v1[db] = value(1, db);
          o[db] = Elem::mma(v0[db], p[0], o[db]);
        }
#pragma unroll
        for (int db = 0; db < 4; ++db) o[db] = Elem::mma(v1[db], p[1], o[db]);
      }
    }
    // The next tile has landed, and behind the barrier this one's place is free.
    if (i + 2 < tiles) landed<2 * kLoads>();
    else landed<0>();
    __syncthreads();
  };
  for (;;) {
    if (tiles > 0) renew_ids(tile0);
#pragma unroll 1
    for (int i = 0; i < min(tiles, 2); ++i) fetch(i, i);
    landed<0>();
    __syncthreads();
    m = -FLT_MAX, l = 0.f;  // finite where a row sees no key, or none but of score -inf
    large = true;
#pragma unroll
    for (int db = 0; db < 4; ++db) o[db] = f32x16{};
    auto steps = [&](auto two) __attribute__((always_inline)) {
      for (int i = 0; i < tiles; i += kBuffers) {  // LDS places known at compile time
        step(two, i, 0);
        if (i + 1 >= tiles) break;
        step(two, i + 1, 1);
        if (i + 2 >= tiles) break;
        step(two, i + 2, 2);
      }
    };
    if constexpr (std::is_same_v<Elem, BFloat>) {
      if (two_terms) steps(std::true_type{});
      else steps(std::false_type{});
    } else {
      steps(std::false_type{});
    }
    if (careful) {
      const int half = fresh_lane() >> 5;
      const int stop = min(see, end * kKeys - 1);
      for (int key = (tile0 + masked) * kKeys; key <= stop; ++key) {
        const int page = quotient(key, a.by_page), id = min(max(table[page], 0), a.num_pages - 1);
        const u32x2* const x = (const u32x2*)(a.v_pages + (uint64_t)(uint32_t)id * a.page_bytes +
                                              (head + (uint32_t)(key - page * a.page_size) * kRowBytes)) + half;
#pragma unroll
        for (int c = 0; c < 16; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float y = Elem::widen(x[2 * c][i >> 1], i & 1);
            o[c >> 2][4 * (c & 3) + i] += __builtin_isfinite(y) ? 0.f : y;
          }
      }
    }
    // The rows go out; where one is not finite (`zero` is NaN), once more after the second pass.
    const float sum = l + __shfl_xor(l, 32);
    float zero = 0.f;
    const int here = fresh_lane(), col = here & 31, half = here >> 5;
    // The wave's 32 rows pass through LDS, so that 16 lanes write 256 bytes of one; 16-byte chunks lie
    // under an exclusive or with the row.
    uint8_t* const mine = lds + wave * kWaveRows * kRowBytes;
    if (!whole) {  // sums in 32 bits, half of a row's dims at a time
      const long state = ((long)u.states + (long)part * rows + row0) * a.hkv + kvh;
      float* const to = a.sums + (state + (long)(here >> 4) * a.hkv) * kD + 4 * (here & 15);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const f32x16& y = o[2 * h + (c >> 2)];
          const f32x4 x{y[4 * (c & 3)], y[4 * (c & 3) + 1], y[4 * (c & 3) + 2], y[4 * (c & 3) + 3]};
          *(f32x4*)(mine + col * kRowBytes + (((2 * c + half) ^ (col & 15)) << 4)) = x;
#pragma unroll
          for (int i = 0; i < 4; ++i) zero = __builtin_fmaf(x[i], 0.f, zero);
        }
#pragma unroll
        for (int i = 0; i < kWaveRows / 4; ++i) {
          const int j = 4 * i + (here >> 4);
          const f32x4 x = *(const f32x4*)(mine + j * kRowBytes + (((here & 15) ^ (j & 15)) << 4));
          if (j < live) *(f32x4*)(to + (long)i * 4 * a.hkv * kD + 64 * h) = x;
        }
      }
      if (half == 0 && col < live) *(f32x2*)(a.tops + 2 * (state + (long)col * a.hkv)) = f32x2{m, sum};
    } else {
      // In the output's type, 0 for a token that sees no key.
      const float inv = see < 0 ? 0.f : 1.0f / sum;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float* const x = (const float*)&o[c >> 2] + 4 * (c & 3);
        const u32x2 y{Elem::pack2(x[0] * inv, x[1] * inv), Elem::pack2(x[2] * inv, x[3] * inv)};
        zero = Elem::times0(y[1], Elem::times0(y[0], zero));
        *(u32x2*)(mine + col * kRowBytes + ((c ^ (col & 15)) << 4) + 8 * half) = y;
      }
      // Row R of the (sequence, KV head), a row of its token t, is row R + t (Hq - G) of the output.
      uint8_t* const to = a.output + ((long)start * a.hq + kvh * a.group + row0 + (long)tok0 * (a.hq - a.group)) * kRowBytes +
                          (here & 15) * 16;
#pragma unroll
      for (int i = 0; i < kWaveRows / 4; ++i) {
        const int j = 4 * i + (here >> 4);
        if (j < live)
          *(u32x4*)(to + (long)(j + token_of(j) * (a.hq - a.group)) * kRowBytes) =
              *(const u32x4*)(mine + j * kRowBytes + (((here & 15) ^ (j & 15)) << 4));
      }
    }
    if (careful) return;
    const int bad = __builtin_amdgcn_ballot_w64(live > 0 && zero != 0.f) != 0;
    if (fresh_lane() == 0) failed[wave] = bad;
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) any |= failed[w];
    if (!uniform(any)) return;
    careful = true;
  }
}

// Joins the parts of the rows that were cut.  32 lanes hold a row, four dims each.  With fewer rows
// than such groups of lanes, the kJoin groups of a workgroup share one row's parts out.
constexpr int kJoin = 8;
template <class Elem>
__global__ __launch_bounds__(32 * kJoin) void join_kernel(ChunkArgs a) {
  __shared__ f32x4 part_sums[kJoin][32];
  __shared__ float part_m[kJoin], part_l[kJoin];
  __shared__ int small_states[kSmallBatch + 1], small_joins[kSmallBatch + 1];
  const int tid = threadIdx.x, lane = tid & 63, sub = tid >> 5, quad = tid & 31;
  Cut cut;
  if (a.batch <= kSmallBatch) {
    const LanePlan p = lane_plan(a, lane);
    const int states = wave_scan(p.share.states), joins = wave_scan(p.share.joins);
    if (tid < 64) {
      small_states[lane] = states - p.share.states, small_joins[lane] = joins - p.share.joins;
      if (lane == 63) small_joins[64] = joins;
    }
    cut = p.cut;
    __syncthreads();
  } else {
    cut = {a.plan[0], a.plan[1]};
  }
  const bool small = a.batch <= kSmallBatch;
  auto joins_at = [&](int b) { return small ? small_joins[b] : joins_before(a)[b]; };
  const long total = (long)joins_at(a.batch) * a.hkv;
  const bool shared = total <= 2L * gridDim.x;  // one row a workgroup at a time
  const int first = shared ? sub : 0, stride = shared ? kJoin : 1;
  for (long i = shared ? blockIdx.x : (long)blockIdx.x * kJoin + sub; i < total; i += (long)gridDim.x * (shared ? 1 : kJoin)) {
    const int join = (int)(i / a.hkv), kvh = (int)(i - (long)join * a.hkv);
    int b = 0;  // the last row of the table whose first join is at most `join`
    for (int step = 1 << (31 - __builtin_clz(a.batch)); step; step >>= 1)
      if (b + step < a.batch && joins_at(b + step) <= join) b += step;
    const Seq s = seq_of(a, b);
    const int row = join - joins_at(b), rows = s.n * a.group;
    const int tok = row / a.group, head = kvh * a.group + row - tok * a.group;
    const int last = min((row / kRows + 1) * kRows, rows) - 1;
    const int parts = ratio_up(tiles_of(last_key(s, last / a.group) + 1), parts_of(a, s, cut).tiles);
    if (parts <= 1) continue;  // written by its only part
    // 32 bits: states_at_most() times 128 floats.
    const uint32_t next = (uint32_t)(rows * a.hkv);
    uint32_t state = (uint32_t)(((small ? small_states[b] : states_before(a)[b]) + row) * a.hkv + kvh) + first * next;
    float m = -FLT_MAX, l = 0.f;
    f32x4 o = {};
    for (int p = first; p < parts; p += 4 * stride) {  // four parts' loads at once
      f32x2 top[4];
      f32x4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        top[k] = f32x2{-FLT_MAX, 0.f}, x[k] = f32x4{};
        if (p + k * stride < parts) {
          top[k] = *(const f32x2*)(a.tops + 2 * state);
          x[k] = *(const f32x4*)(a.sums + (state * kD + 4 * quad));
        }
        state += stride * next;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float mn = fmaxf(m, top[k][0]);
        const float c0 = __builtin_amdgcn_exp2f((m - mn) * kScaleLog2), c1 = __builtin_amdgcn_exp2f((top[k][0] - mn) * kScaleLog2);
        m = mn, l = l * c0 + top[k][1] * c1;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = o[j] * c0 + x[k][j] * c1;
      }
    }
    if (shared) {
      __syncthreads();  // the row before has been read
      part_sums[sub][quad] = o;
      if (quad == 0) part_m[sub] = m, part_l[sub] = l;
      __syncthreads();
      if (sub != 0) continue;
      for (int p = 1; p < kJoin; ++p) m = fmaxf(m, part_m[p]);
      l = 0.f, o = f32x4{};
      for (int p = 0; p < kJoin; ++p) {
        const float c = __builtin_amdgcn_exp2f((part_m[p] - m) * kScaleLog2);
        l += part_l[p] * c;
        const f32x4 x = part_sums[p][quad];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += x[j] * c;
      }
    }
    const float inv = last_key(s, tok) < 0 ? 0.f : 1.0f / l;
    *(u32x2*)(a.output + (((long)s.start + tok) * a.hq + head) * kRowBytes + 8 * quad) =
        u32x2{Elem::pack2(o[0] * inv, o[1] * inv), Elem::pack2(o[2] * inv, o[3] * inv)};
  }
}

// ---------------------------------------------------------------------------------
// Host.
// ---------------------------------------------------------------------------------
Divisor divisor(int d) {
  uint32_t shift = 0;
  while ((1u << shift) < (uint32_t)d) ++shift;
  return {(uint32_t)(((1ull << (31 + shift)) + d - 1) / d), shift};
}

int parts_wanted() { return 2 * pkv::compute_units(); }

// The blocks that a call can have, over all KV heads.
int64_t blocks_at_most(int64_t batch, int64_t tokens, int64_t group, int64_t hkv) {
  return (tokens * group / kRows + batch) * hkv;
}
size_t plan_bytes(int64_t batch) { return batch > kSmallBatch ? (size_t)((5 + 4 * batch) * 4 + 15) / 16 * 16 : 0; }

// Parts that a call can have beyond one a block, over all KV heads: none of its rows is large where
// all its tokens are one wave's.
int64_t parts_at_most(int64_t tokens, int64_t group) {
  return (int64_t)parts_wanted() * (tokens * group <= kWaveRows ? 1 : 1 + kFiner);
}

// Rows of states, over all KV heads.  A small row is cut only where its tiles pass C, into less than
// tiles / C + 1 parts, which is at most 2 tiles / C; a large one where they reach 1.5 C, into at most
// tiles / C + 1/2, which is at most 4/3 tiles / C.  So the parts of all blocks of a class are at most
// 2 W / C and 4/3 W / C, with C at least W / P and W / (kFiner P): of 32 and of 128 rows each, and of
// no more than the call has.  With 256 compute units that is 199 MB for calls of 128 rows and more
// and 17 MB for those of at most 32.
int64_t states_at_most(int64_t tokens, int64_t group) {
  const int64_t all = tokens * group, small = all < kWaveRows ? all : kWaveRows, large = all < kRows ? all : kRows;
  const int64_t parts = parts_wanted();
  return 2 * parts * small + (all > kWaveRows ? (4 * kFiner * parts * large + 2) / 3 : 0);
}
// The joins address their floats in 32 bits.
constexpr int64_t kMostUnits = 1024;  // compute units of any one GPU
static_assert(2 * kMostUnits * (2 * kWaveRows + (4 * kFiner * kRows + 2) / 3) * kStateFloats <= UINT32_MAX);

}  // namespace

extern "C" {

size_t pkv_paged_prefill_workspace_bytes(int32_t batch, int32_t tokens, int32_t num_q_heads, int32_t num_kv_heads) {
  if (batch <= 0 || tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads) return 0;
  const int64_t group = num_q_heads / num_kv_heads;
  return plan_bytes(batch) + (size_t)states_at_most(tokens, group) * kStateFloats * sizeof(float);
}

int pkv_paged_prefill_attention(const void* q, int64_t q_stride, const void* k_pages, const void* v_pages,
                                const int32_t* block_table, const int32_t* seq_lens,
                                const int32_t* token_offsets, void* output, void* workspace,
                                size_t workspace_size, int32_t batch, int32_t tokens, int32_t num_q_heads,
                                int32_t num_kv_heads, int32_t head_dim, int32_t num_pages,
                                int32_t page_size, int32_t max_pages, int32_t dtype, void* stream) {
  using pkv::fail;
  const char* const op = "paged_prefill_attention";
  if (batch < 0 || tokens < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_pages <= 0 || page_size <= 0 || max_pages <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT,
                "%s: batch %d, tokens %d, num_q_heads %d, num_kv_heads %d, num_pages %d, page_size %d, max_pages %d", op,
                batch, tokens, num_q_heads, num_kv_heads, num_pages, page_size, max_pages);
  if (head_dim != kD) return fail(PKV_ERR_UNSUPPORTED, "%s: head_dim %d (only 128)", op, head_dim);
  if (dtype != PKV_DTYPE_F16 && dtype != PKV_DTYPE_BF16) return fail(PKV_ERR_UNSUPPORTED, "%s: unknown dtype %d", op, dtype);
  if (num_q_heads % num_kv_heads) return fail(PKV_ERR_INVALID_ARGUMENT, "%s: Hq must be divisible by Hkv", op);
  const int32_t group = num_q_heads / num_kv_heads;
  if (group > PKV_MAX_GROUP) return fail(PKV_ERR_UNSUPPORTED, "%s: G=Hq/Hkv %d (at most %d)", op, group, PKV_MAX_GROUP);
  if (q_stride < (int64_t)num_q_heads * kD || q_stride % 8)
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: the token stride must hold q's heads and be a multiple of 8 elements", op);
  const int64_t page_bytes = (int64_t)num_kv_heads * page_size * kRowBytes;
  if ((int64_t)max_pages * page_size > INT32_MAX - kKeys || page_bytes > INT32_MAX)
    return fail(PKV_ERR_UNSUPPORTED, "%s: max_pages * page_size must be below 2^31 - 32, and a page below 2 GiB", op);
  const int64_t groups = blocks_at_most(batch, tokens, group, num_kv_heads) +
                         (parts_at_most(tokens, group) / num_kv_heads + 1 + kFiner) * num_kv_heads;
  if ((int64_t)tokens * group > INT32_MAX || !pkv::fits_grid(groups, kWaves * 64))
    return fail(PKV_ERR_UNSUPPORTED, "%s: too many tokens or sequences", op);
  if (batch == 0 || tokens == 0) return pkv::ok();
  if (!q || !k_pages || !v_pages || !block_table || !seq_lens || !token_offsets || !output)
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: null pointer", op);
  if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)output) & 15)
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: tensors must be 16-byte aligned", op);
  const size_t need = pkv_paged_prefill_workspace_bytes(batch, tokens, num_q_heads, num_kv_heads);
  if (!workspace || workspace_size < need || ((uintptr_t)workspace & 15))
    return fail(PKV_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes is smaller than %zu, or misaligned", op,
                workspace_size, need);
  // Rows of q are read until the last part of their block ends, behind which the output of another
  // may have been written: only a q whose rows are the output's own may be written over.
  const int64_t row = (int64_t)num_q_heads * kRowBytes;
  if (!(output == q && (tokens == 1 || 2 * q_stride == row)) &&
      pkv::meets_rows(output, tokens * row, q, tokens, 2 * q_stride, row))
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: output must be a contiguous q itself, or not overlap q", op);
  float* const states = (float*)((uint8_t*)workspace + plan_bytes(batch));
  const ChunkArgs a{(const uint8_t*)q, (const uint8_t*)k_pages, (const uint8_t*)v_pages, block_table, seq_lens, token_offsets,
                    (uint8_t*)output, (int32_t*)workspace, states, states + states_at_most(tokens, group) * kD,
                    2 * q_stride, batch, tokens, num_q_heads, num_kv_heads, group, num_pages, max_pages, page_size,
                    (uint32_t)page_bytes, divisor(page_size), divisor(group), divisor(num_kv_heads), 1.0f / (float)group,
                    (float)num_kv_heads / (float)parts_wanted() * 1.0001f};
  const hipStream_t st = (hipStream_t)stream;
  const bool bf16 = dtype == PKV_DTYPE_BF16;
  if (batch > kSmallBatch) plan_kernel<<<1, kPlanThreads, 0, st>>>(a);
  auto* const kernel = bf16 ? chunk_kernel<BFloat> : chunk_kernel<Half>;
  kernel<<<dim3((unsigned)groups), dim3(kWaves * 64), 0, st>>>(a);
  auto* const join = bf16 ? join_kernel<BFloat> : join_kernel<Half>;
  const int64_t joins = (int64_t)tokens * num_q_heads, most = 4L * pkv::compute_units();
  join<<<dim3((unsigned)(joins < most ? joins : most)), dim3(32 * kJoin), 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? pkv::ok() : fail(PKV_ERR_LAUNCH, "%s launch: %s", op, hipGetErrorString(e));
}

}  // extern "C"
