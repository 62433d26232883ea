// pkv_prefill.hip — causal GQA attention over whole prompts, packed one after another
// (the reference has decode only; its harness starts from a filled pool,
// tests/benchmark_serving_trace.py:285-298).
//
//   o[i] = sum_{j <= i} p_ij v[j],  p_ij = exp(q[i] k[j] / sqrt(128) - m_i) / l_i
//
// Rows of work.  The G query heads of a KV head are rows of one matrix product over the same K
// and V: row r of a (sequence, KV head) is token r / G, head kvh * G + r % G.  A workgroup of
// four waves owns 128 consecutive rows (for G = 4: 32 tokens), a wave 32 of them, so K/V
// tiles are read from L2 once for all heads of the group, any G is served by one kernel, and
// the masked part of a diagonal tile covers few tokens.  Consecutive workgroups take the KV
// heads in turn: with 8 heads, or a multiple, each XCD's L2 holds the K/V of its own.
//
// Per wave and tile of 32 keys, with v_mfma_f32_32x32x16:
//   S^T[key, row] = K Q^T   K from LDS as the A operand, Q in registers as the B operand.
//   A lane then holds 16 keys of ONE row: maximum and sum of the softmax are lane-local but
//   for one exchange between the wave's halves.
//   O^T[dim, row] += V^T P^T   P^T's B operand is S^T's own register layout, packed to 16 bits
//   (the k order of a product is free as long as both operands agree), V^T's A operand comes
//   from row-major V in LDS through the transposing reads (ds_read_b64_tr_b16).
// P is rounded to the activation type (half a step of it, as the operand must be), and the sum
// that divides is that of the rounded weights; scores, sums and outputs are in 32 bits.  The
// decode kernels add a second bf16 term of P: they wait for memory, and its products cost
// little.  Here products are what bounds it, and a second term is half as many again: bf16
// outputs are 1.9e-3 to 2.0e-3 from the exact ones (relative 2-norm), where 32-bit weights give
// 1.5e-3 to 1.6e-3, the output's own rounding.
//
// Three workgroups run on a CU (168 registers, 48 KB of LDS each), so that one's softmax and
// waits lie under another's products; K/V pass from memory to LDS without registers, two tiles
// ahead.  The compiler spills 4 (fp16) or 6 (bf16) vector registers to 20 bytes of scratch and 43
// scalars to lanes of vector registers, and brings them back before the first tile, right
// behind its scores or after the last one; the kernel for few blocks spills 55 scalars.  Two
// prompts of 8192 (Hq 32, Hkv 8, bf16): 0.965-0.98 ms, 1.12-1.14 PFLOP/s, 0.9 of what a library
// product of 8192^3 reaches; bounded by power (1.55-1.7 GHz with the matrix units busy 62-64 %
// of the cycles; the products alone take 0.815 ms).  32 prompts of 16-1024: 126 us, 630 TFLOP/s,
// a third of it the start and end of each workgroup.

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

constexpr uint32_t kRsrcWord3 = 0x00020000u;  // raw buffer, 32-bit data format (gfx9 family)

struct PrefillArgs {
  const uint8_t* q;  // token t, head h at q + t * q_stride + h * 256 (bytes)
  const uint8_t* k;
  const uint8_t* v;
  const int32_t* token_offsets;  // [B + 1]
  uint8_t* output;               // [T, Hq, 128]
  long q_stride, k_stride, v_stride;
  int32_t batch, tokens, hq, hkv, group;
  float inv_group;
};

__device__ inline int offset_of(const PrefillArgs& a, int b) {
  return min(max(a.token_offsets[b], 0), a.tokens);
}
template <int ROWS>  // of a block
__device__ inline int blocks_of(const PrefillArgs& a, int len) {
  return (int)(((uint32_t)(len * a.group) + ROWS - 1) / ROWS);
}

// A block of rows: block `index` of the sequence of `len` tokens from `start` on.  index < 0: none.
struct Block {
  int start, len, index;
};

// The `slot`-th block of up to 64 sequences: those longer than half the longest first, then
// those longer than a quarter, an eighth, and the others; sequence after sequence in each
// class, its longest block first.  So the blocks that start last, and that the GPU waits for
// at the end, are short, and the blocks at work at one time still share their K/V in L2 (all
// blocks by length would not: slower).
template <int ROWS>
__device__ inline Block by_length(const PrefillArgs& a, int slot, int lane) {
  const int start = offset_of(a, min(lane, a.batch));
  const int len = max(offset_of(a, min(lane + 1, a.batch)) - start, 0);
  const int blocks = blocks_of<ROWS>(a, len), top = wave_max(blocks);
  for (int k = 0; k < 4; ++k) {
    const int n = blocks <= top >> k && (k == 3 || blocks > top >> (k + 1)) ? blocks : 0;
    const int sums = wave_scan(n);
    const uint64_t past = __builtin_amdgcn_ballot_w64(sums > slot);
    if (past) {
      const int b = __builtin_ctzll(past);
      return {__builtin_amdgcn_readlane(start, b), __builtin_amdgcn_readlane(len, b),
              __builtin_amdgcn_readlane(sums, b) - 1 - slot};
    }
    slot -= __builtin_amdgcn_readlane(sums, 63);
  }
  return {0, 0, -1};
}

// The `slot`-th block of more sequences: sequence after sequence, its longest block first.
// Sequence b, whose rows start at x = offset * G, has the slots from x / ROWS + b on, which
// are, up to the next sequence's, at least as many as its blocks.  It is the last one whose
// first slot is at most `slot`, found among 63 candidates at a time; the last round's lanes
// hold its offset and its successor's.
template <int ROWS>
__device__ inline Block packed_order(const PrefillArgs& a, int slot, int lane) {
  auto first_slot = [&](int offset, int b) { return (int)((uint32_t)(offset * a.group) / ROWS) + b; };
  int b = 0, n = a.batch, stride, offset, found;
  do {
    stride = (n + 62) / 63;
    const int at = b + min(lane * stride, n);
    offset = offset_of(a, min(at, a.batch));
    const uint64_t fits = __builtin_amdgcn_ballot_w64(lane * stride < n && first_slot(offset, at) <= slot);
    found = fits ? 63 - __builtin_clzll(fits) : 0;
    b += found * stride;
    n = min(stride, n - found * stride);
  } while (stride > 1);
  const int start = __builtin_amdgcn_readlane(offset, found);
  const int len = max(__builtin_amdgcn_readlane(offset, found + 1) - start, 0);
  const int blocks = blocks_of<ROWS>(a, len), index = blocks - 1 - (slot - first_slot(start, b));
  return {start, len, index < blocks ? index : -1};
}

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// 64 x 16 bytes from a buffer straight to LDS, lane l's to `lds` + 16 l.  In assembly because the
// compiler lets every LDS read wait for every such load in flight, the next tile's among them;
// landed() is the wait, before the barrier behind which the tile is read.  The compiler keeps no
// distances to instructions in assembly, so this text carries them: a scalar register written by a
// vector instruction (the descriptor's, by readfirstlane or as a spilled one brought back) must
// lie five wait states before the load that reads it (s_mov, and four of s_nop 3), m0 one.  No
// registers are written but m0, which nothing else in these kernels uses.
__device__ inline void load_to_lds(uint32_t lds, i32x4 rsrc, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds), "v"(offset), "s"(rsrc) : "memory");
}

// GROUPS = 2: two waves for 64 rows' even tiles and two for their odd ones, whose states are
// joined at the end.  A step takes about 0.65 us however little the GPU has to do, so where
// blocks are few, half the steps on twice the CUs count for more than the second reading of
// K/V: one prompt of 500 tokens (8 KV heads) 15.2 -> 12.7 us, 4000 (1 KV head) 82 -> 52 us; with
// blocks for every CU it is no faster.
template <class Elem, int GROUPS>
__global__ __launch_bounds__(kWaves * 64, GROUPS == 1 ? 3 : 1) void prefill_kernel(PrefillArgs a) {
  constexpr int kGroupWaves = kWaves / GROUPS, kRows = kGroupWaves * kWaveRows;
  constexpr int kGroupBytes = kBuffers * 2 * kTileBytes;
  __shared__ __attribute__((aligned(1024))) uint8_t all_lds[GROUPS * kGroupBytes];
  const int tid = threadIdx.x, lane = tid & 63;
  const int group = GROUPS == 1 ? 0 : uniform(tid >> 6) / kGroupWaves, wave = (tid >> 6) - group * kGroupWaves;
  uint8_t* const lds = all_lds + group * kGroupBytes;  // K and V of the group's tiles
  const int col = lane & 31, half = lane >> 5;
  const int kvh = uniform((int)(blockIdx.x % (unsigned)a.hkv));
  const int slot = uniform((int)(blockIdx.x / (unsigned)a.hkv));
  const Block work = a.batch <= 64 ? by_length<kRows>(a, slot, lane) : packed_order<kRows>(a, slot, lane);
  if (work.index < 0) return;
  const int start = uniform(work.start), len = uniform(work.len), block = uniform(work.index);
  const int rows = len * a.group;

  // Row row0 + r of the wave is token tok0 + (rem + r) / G: a quotient of numbers below 64, which
  // the product with 1 / G in 32 bits gives exactly (it is off by less than 1 / (2 G)).
  const int row0 = uniform(min(block * kRows + wave * kWaveRows, rows));
  const int tok0 = row0 / a.group, rem = row0 - tok0 * a.group, live = rows - row0;  // may be 0
  auto token_of = [&](int r) { return (int)(((float)(rem + r) + 0.5f) * a.inv_group); };
  const int last_row = max(min(kWaveRows, live) - 1, 0);
  const int r = min(col, last_row), dt = token_of(r);
  const int tok = min(tok0 + dt, len - 1);  // a wave past the last row takes the last token's
  const int wave_first = tok0, wave_last = live > 0 ? tok0 + uniform(token_of(last_row)) : -1;
  const int last = (min((block + 1) * kRows, rows) - 1) / a.group;
  const int all_tiles = last / kKeys + 1;
  const int tiles = (all_tiles - group + GROUPS - 1) / GROUPS;  // the group's: GROUPS i + group
  const int steps = (all_tiles + GROUPS - 1) / GROUPS;

  // A wave moves rows kMoved wave + 4 i + lane / 16 of a tile, 256 bytes a row.  16-byte chunk p of
  // row r in LDS is chunk p ^ r of K's row (p ^ 4 r of V's), so that reads of one chunk column
  // (K) or of 64 bytes of four rows (V) spread over all banks.
  constexpr int kMoved = kKeys / kGroupWaves;
  const int srow = wave * kMoved + (lane >> 4), chunk = lane & 15;
  const uint32_t lds0 = (uint32_t)uniform((int)((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds +
                                                (uint32_t)(wave * kMoved * kRowBytes)));
  const uint8_t* const kbase = a.k + (long)start * a.k_stride + (long)kvh * kRowBytes;
  const uint8_t* const vbase = a.v + (long)start * a.v_stride + (long)kvh * kRowBytes;
  const uint32_t koff = (uint32_t)(srow * (int)a.k_stride), kchunk = (chunk ^ (srow & 15)) << 4;
  const uint32_t voff = (uint32_t)(srow * (int)a.v_stride) + ((chunk ^ ((srow & 3) << 2)) << 4);
  constexpr int kLoads = kMoved / 4;  // per wave and tile of K, and of V
  // The next tile to fetch: where it lies, and the rows from it to the sequence's end.
  uint64_t kp, vp;
  int left;
  auto fetch = [&](int buf) __attribute__((always_inline)) {
    // Rows past the sequence's end read as zero: the descriptor ends with its last row.
    const int n = min(kKeys, left) - 1;
    const i32x4 rk{uniform((int)kp), uniform((int)(kp >> 32) & 0xffff),
                   uniform(n * (int)a.k_stride + kRowBytes), (int)kRsrcWord3};
    const i32x4 rv{uniform((int)vp), uniform((int)(vp >> 32) & 0xffff),
                   uniform(n * (int)a.v_stride + kRowBytes), (int)kRsrcWord3};
    const uint32_t to = (uint32_t)uniform((int)(lds0 + buf * 2 * kTileBytes));
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      load_to_lds(to + i * 4 * kRowBytes, rk, koff + (kchunk ^ (i << 6)) + i * 4 * (uint32_t)a.k_stride);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      load_to_lds(to + kTileBytes + i * 4 * kRowBytes, rv, voff + i * 4 * (uint32_t)a.v_stride);
    kp += (uint64_t)(GROUPS * kKeys * a.k_stride);
    vp += (uint64_t)(GROUPS * kKeys * a.v_stride);
    left -= GROUPS * kKeys;
  };
  auto begin = [&]() __attribute__((always_inline)) {
    kp = (uint64_t)uniform_ptr(kbase + (long)group * kKeys * a.k_stride);
    vp = (uint64_t)uniform_ptr(vbase + (long)group * kKeys * a.v_stride);
    left = len - group * kKeys;
    if (tiles > 0) fetch(0);
    if (tiles > 1) fetch(1);
  };
  begin();  // before Q's loads: nothing that waits for those comes between

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
  const uint8_t* kat[8];
  const uint8_t* vat[4];
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) kat[kk] = lds + (ksrc ^ (kk << 5));
#pragma unroll
  for (int db = 0; db < 4; ++db) vat[db] = lds + kTileBytes + (vsrc ^ (db << 6));

  // A masked weight is 0, and 0 times an infinity or NaN in V is NaN.  So where a row comes out
  // not finite, its workgroup computes once more, `careful`: such values are taken out of the
  // tiles that a row of it masks in part, those of the steps from `masked` on, and put back at the end for
  // the rows from their token on.
  bool careful = false;
  const int masked = block * kRows / a.group / kKeys / GROUPS;  // a step: the same for all groups
  auto clean = [&](int buf) {
    u32x4* const v = (u32x4*)(lds + buf * 2 * kTileBytes + kTileBytes) + wave * 64 + lane;
    for (int i = 0; i < kTileBytes / 16; i += kGroupWaves * 64) {
      u32x4 x = v[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = drop_nonfinite<Elem>(x[j]);
      v[i] = x;
    }
    __syncthreads();
  };

  // The group's i-th tile, which lies in buffer `buf`; `first`: i = 0, which sets the running
  // maximum, sums and output.
  auto step = [&](int i0, int buf, auto first) __attribute__((always_inline)) {
    constexpr bool kFirst = decltype(first)::value;
    const int at = buf * 2 * kTileBytes;
    if (careful && i0 >= masked) clean(buf);
    if (i0 + 2 < tiles) fetch(buf >= 1 ? buf - 1 : buf + 2);
    const int k0 = (GROUPS * i0 + group) * kKeys;
    if ((kFirst && GROUPS == 1) || (k0 <= wave_last && (GROUPS == 1 || i0 < tiles))) {
      f32x16 s = {};
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) s = Elem::mma(*(const u32x4*)(kat[kk] + at), q[kk], s);
      auto value = [&](int c, int db) __attribute__((always_inline)) {  // keys 16 c ..., dims 32 db + lane % 32
        typedef __attribute__((address_space(3))) s16x4* Lds;
        const uint8_t* v = vat[db] + at + c * 16 * kRowBytes;
        const u32x2 v0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)v));
        const u32x2 v1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(v + 8 * kRowBytes)));
        return u32x4{v0[0], v0[1], v1[0], v1[1]};
      };
      u32x4 v0[4];
#pragma unroll
      for (int db = 0; db < 4; ++db) v0[db] = value(0, db);
      if (k0 + kKeys - 1 > wave_first) {
        const int visible = tok - k0 - 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i >> 2) + (i & 3) > visible) s[i] = -INFINITY;
      }
      float mx = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
      if constexpr (kFirst) {
        // Finite where a row sees no key of the tile, or none but of score -inf: weights 0, not NaN.
        m = fmaxf(fmaxf(mx, __shfl_xor(mx, 32)), -FLT_MAX);
        l = 0.f;
        large = __builtin_amdgcn_ballot_w64(fabsf(m) >= kLargeScore) != 0;
      } else if (__builtin_amdgcn_ballot_w64(mx > m + kSlack) != 0) {
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
        const uint32_t x = Elem::pack2(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i], kScaleLog2, -ms)),
                                       __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + 1], kScaleLog2, -ms)));
        p[i >> 3][(i & 7) >> 1] = x;
        l = Elem::sum2(x, l);
      }
      u32x4 v1[4];
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        v1[db] = value(1, db);
        o[db] = Elem::mma(v0[db], p[0], kFirst ? f32x16{} : o[db]);
      }
#pragma unroll
      for (int db = 0; db < 4; ++db) o[db] = Elem::mma(v1[db], p[1], o[db]);
    }
    // The next tile has landed, and behind the barrier this one's place is free.
    if (i0 + 2 < tiles) landed<2 * kLoads>();
    else landed<0>();
    __syncthreads();
  };
  u32x2 out[16];
  for (;;) {
    landed<0>();
    __syncthreads();
    if constexpr (GROUPS > 1) {  // a wave without a key: weight 0
      m = -FLT_MAX, l = 0.f;
#pragma unroll
      for (int db = 0; db < 4; ++db) o[db] = f32x16{};
    }
    step(0, 0, std::true_type{});
    for (int i = 1; i < steps; i += kBuffers) {  // LDS places known at compile time
      step(i, 1, std::false_type{});
      if (i + 1 >= steps) break;
      step(i + 1, 2, std::false_type{});
      if (i + 2 >= steps) break;
      step(i + 2, 0, std::false_type{});
    }
    if constexpr (GROUPS > 1) {  // the second group's states to the first's waves
      float* const at = (float*)all_lds + wave * 66 * 64 + lane;
      if (group == 1) {
#pragma unroll
        for (int j = 0; j < 64; ++j) at[j * 64] = o[j >> 4][j & 15];
        at[64 * 64] = m, at[65 * 64] = l;
      }
      __syncthreads();
      if (group == 0) {
        const float m1 = at[64 * 64], l1 = at[65 * 64], mn = fmaxf(m, m1);
        const float c0 = __builtin_amdgcn_exp2f((m - mn) * kScaleLog2), c1 = __builtin_amdgcn_exp2f((m1 - mn) * kScaleLog2);
        m = mn, l = l * c0 + l1 * c1;
#pragma unroll
        for (int j = 0; j < 64; ++j) o[j >> 4][j & 15] = o[j >> 4][j & 15] * c0 + at[j * 64] * c1;
      }
      __syncthreads();  // the places are free
    }
    if (careful) {
      for (int key = masked * GROUPS * kKeys; key <= tok; ++key) {
        const u32x2* const x = (const u32x2*)(vbase + (long)key * a.v_stride) + half;
#pragma unroll
        for (int c = 0; c < 16; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float y = Elem::widen(x[2 * c][i >> 1], i & 1);
            o[c >> 2][4 * (c & 3) + i] += __builtin_isfinite(y) ? 0.f : y;
          }
      }
    }
    // The rows in the output's type; `zero` turns NaN where a value is not finite.
    const float inv = 1.0f / (l + __shfl_xor(l, 32));
    float zero = 0.f;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const uint32_t x = Elem::pack2(o[db][i] * inv, o[db][i + 1] * inv);
        out[4 * db + (i >> 2)][(i >> 1) & 1] = x;
        zero = Elem::times0(x, zero);
      }
    if (careful || !__syncthreads_or(group == 0 && live > 0 && zero != 0.f)) break;
    careful = true;
    begin();
  }

  if (group != 0) return;
  // The wave's 32 rows pass through LDS, so that 16 lanes write one row of 256 bytes; 16-byte
  // chunks lie under an exclusive or with the row.
  uint8_t* const mine = lds + wave * kWaveRows * kRowBytes;
#pragma unroll
  for (int c = 0; c < 16; ++c) *(u32x2*)(mine + col * kRowBytes + ((c ^ (col & 15)) << 4) + 8 * half) = out[c];
  // Row R of the (sequence, KV head), a row of its token t, is row R + t (Hq - G) of the output.
  uint8_t* const to = a.output + ((long)start * a.hq + kvh * a.group + row0 + (long)tok0 * (a.hq - a.group)) * kRowBytes +
                      (lane & 15) * 16;
#pragma unroll
  for (int i = 0; i < kWaveRows / 4; ++i) {
    const int j = 4 * i + (lane >> 4);
    if (j < live)
      *(u32x4*)(to + (long)(j + token_of(j) * (a.hq - a.group)) * kRowBytes) =
          *(const u32x4*)(mine + j * kRowBytes + (((lane & 15) ^ (j & 15)) << 4));
  }
}

}  // namespace

extern "C" int pkv_prefill_attention(
    const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
    int64_t v_stride, const int32_t* token_offsets, void* output, int32_t batch, int32_t tokens,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t dtype, void* stream) {
  using pkv::fail;
  if (batch < 0 || tokens < 0 || num_q_heads <= 0 || num_kv_heads <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "prefill_attention: batch %d, tokens %d, num_q_heads %d, num_kv_heads %d",
                batch, tokens, num_q_heads, num_kv_heads);
  if (head_dim != kD) return fail(PKV_ERR_UNSUPPORTED, "prefill_attention: head_dim %d (only 128)", head_dim);
  if (dtype != PKV_DTYPE_F16 && dtype != PKV_DTYPE_BF16)
    return fail(PKV_ERR_UNSUPPORTED, "prefill_attention: unknown dtype %d", dtype);
  if (num_q_heads % num_kv_heads)
    return fail(PKV_ERR_INVALID_ARGUMENT, "prefill_attention: Hq must be divisible by Hkv");
  const int32_t group = num_q_heads / num_kv_heads;
  if (group > PKV_MAX_GROUP)
    return fail(PKV_ERR_UNSUPPORTED, "prefill_attention: G=Hq/Hkv %d (at most %d)", group, PKV_MAX_GROUP);
  if (q_stride < (int64_t)num_q_heads * kD || k_stride < (int64_t)num_kv_heads * kD ||
      v_stride < (int64_t)num_kv_heads * kD || (q_stride | k_stride | v_stride) % 8)
    return fail(PKV_ERR_INVALID_ARGUMENT,
                "prefill_attention: a token stride must hold its heads and be a multiple of 8 elements");
  if (k_stride > (1 << 23) || v_stride > (1 << 23))  // a tile's rows lie within 2 GiB
    return fail(PKV_ERR_UNSUPPORTED, "prefill_attention: token strides of K and V up to 2^23 elements");
  auto slots = [&](int rows) { return ((int64_t)tokens * group / rows + batch) * num_kv_heads; };
  if ((int64_t)tokens * group > INT32_MAX || !pkv::fits_grid(slots(kWaves * kWaveRows), kWaves * 64))
    return fail(PKV_ERR_UNSUPPORTED, "prefill_attention: too many tokens or sequences");
  if (batch == 0 || tokens == 0) return pkv::ok();
  if (!q || !k || !v || !token_offsets || !output)
    return fail(PKV_ERR_INVALID_ARGUMENT, "prefill_attention: null pointer");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)output) & 15)
    return fail(PKV_ERR_INVALID_ARGUMENT, "prefill_attention: tensors must be 16-byte aligned");
  // Blocks read K and V, and other blocks' rows of q, until the last one ends: only a q whose rows
  // are the output's own may be written over.
  const int64_t row = (int64_t)num_q_heads * kRowBytes, kv_row = (int64_t)num_kv_heads * kRowBytes;
  if (pkv::meets_rows(output, tokens * row, k, tokens, 2 * k_stride, kv_row) ||
      pkv::meets_rows(output, tokens * row, v, tokens, 2 * v_stride, kv_row))
    return fail(PKV_ERR_INVALID_ARGUMENT, "prefill_attention: output must not be k or v, nor overlap them");
  if (!(output == q && (tokens == 1 || 2 * q_stride == row)) &&
      pkv::meets_rows(output, tokens * row, q, tokens, 2 * q_stride, row))
    return fail(PKV_ERR_INVALID_ARGUMENT,
                "prefill_attention: output must be a contiguous q itself, or not overlap q");
  const PrefillArgs a{(const uint8_t*)q, (const uint8_t*)k, (const uint8_t*)v, token_offsets,
                      (uint8_t*)output, 2 * q_stride, 2 * k_stride, 2 * v_stride,
                      batch, tokens, num_q_heads, num_kv_heads, group, 1.0f / (float)group};
  // Blocks of 128 rows that leave more than half of the CUs without one become blocks of 64
  // rows whose tiles two pairs of waves share.
  const bool split = slots(kWaves * kWaveRows) <= pkv::compute_units() / 2, bf16 = dtype == PKV_DTYPE_BF16;
  auto* const kernel = split ? (bf16 ? prefill_kernel<BFloat, 2> : prefill_kernel<Half, 2>)
                             : (bf16 ? prefill_kernel<BFloat, 1> : prefill_kernel<Half, 1>);
  kernel<<<dim3((unsigned)slots(kWaves * kWaveRows / (split ? 2 : 1))), dim3(kWaves * 64), 0, (hipStream_t)stream>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? pkv::ok()
                         : fail(PKV_ERR_LAUNCH, "prefill_attention launch: %s", hipGetErrorString(e));
}
