// pkv_write.hip — writes packed K/V tokens (a batch of prompts, or one token a row) into the
// page pools, each token to a slot (page * page_size + offset): a copy into fp16 / bf16 pools,
// or a quantisation to fp8 (OCP e4m3) with one scale per (page, KV head), K and V apart.
// The reference never writes K/V (tests/benchmark_serving_trace.py:285-298).
//
// Block scales are powers of two in [2^-60, 2^60], the smallest with amax <= 448 scale over the
// finite values of the block.  A power of two makes x / scale exact, and growing a scale later
// (a token with a larger magnitude joins a part-filled page) leaves every stored value as it is
// but those that become subnormal, which round once; an arbitrary scale would round every value
// of the page again at each growth.  It costs nothing in precision: e4m3 is a floating format.
//
// Tokens outside the pools (slot < 0 or past the last page) are skipped.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pkv.h"
#include "pkv_device.h"
#include "pkv_e4m3.h"

namespace pkv {
int fail(int status, const char* fmt, ...);  // pkv_decode.hip: sets pkv_last_error()
int ok();
}  // namespace pkv

namespace {

constexpr int kD = 128;
constexpr int kRowBytes = 2 * kD;
constexpr int kScaleExp = 60;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct WriteArgs {
  const uint8_t* k_new;  // token t, head h at k_new + t * k_stride + h * 256 (bytes)
  const uint8_t* v_new;
  uint8_t* k_pages;      // [num_pages, Hkv, ps, 128]
  uint8_t* v_pages;
  float* kv_scales;      // [num_pages, Hkv, 2] (block-scaled fp8)
  const int32_t* slots;  // [tokens]
  long k_stride, v_stride;
  int32_t tokens, hkv, page_size;
  int32_t num_slots;     // num_pages * page_size
};

// Sixteen lanes copy one (token, head) row of 256 bytes, K and V.  Bound by memory: 46257 tokens,
// 8 heads, 379 MB in 73.5 us, the rate of a plain copy (5.1 TB/s).
__global__ __launch_bounds__(256) void write_kernel(WriteArgs a) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long row = i >> 4;
  const int t = (int)(row / a.hkv), h = (int)(row - (long)t * a.hkv);
  if (t >= a.tokens) return;
  const int slot = a.slots[t];
  if (slot < 0 || slot >= a.num_slots) return;
  const int c = (int)(i & 15) * 16;
  const int page = slot / a.page_size, off = slot - page * a.page_size;
  const long to = (((long)page * a.hkv + h) * a.page_size + off) * kRowBytes + c;
  const u32x4 k = *(const u32x4*)(a.k_new + t * a.k_stride + (long)h * kRowBytes + c);
  const u32x4 v = *(const u32x4*)(a.v_new + t * a.v_stride + (long)h * kRowBytes + c);
  *(u32x4*)(a.k_pages + to) = k;
  *(u32x4*)(a.v_pages + to) = v;
}

// ---------------------------------------------------------------------------------
// Block-scaled fp8.
// ---------------------------------------------------------------------------------
// Magnitudes of two 16-bit floats in an order in which every infinity and NaN lies below
// every finite value: (|x| + one step of the exponent) mod 2^15.
template <bool BF16>
__device__ inline uint32_t finite_order(uint32_t x2) {
  return ((x2 & 0x7fff7fffu) + (BF16 ? 0x00800080u : 0x04000400u)) & 0x7fff7fffu;
}
__device__ inline uint32_t max2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}
template <bool BF16>
__device__ inline uint32_t finite_max(uint32_t m, u32x4 x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max2(m, finite_order<BF16>(x[i]));
  return m;
}
template <bool BF16>
__device__ inline uint32_t wave_max(uint32_t m) {
#pragma unroll
  for (int d = 32; d; d >>= 1) m = max2(m, __shfl_xor(m, d));
  return m;
}
// The largest finite magnitude, from the largest of its finite_order.
template <bool BF16>
__device__ inline float finite_value(uint32_t m) {
  const uint32_t z = max(m & 0xffffu, m >> 16), one = BF16 ? 0x80u : 0x400u;
  return pkv::half_bits_to_float<BF16>(z > one ? z - one : 0u);
}

// 2^e of the smallest power of two >= x, within the range of block scales (x not positive or
// NaN: the smallest).  `top`: the mantissa up to which 2^exponent(x) itself is large enough.
__device__ inline int pow2_exponent(float x, uint32_t top) {
  const uint32_t b = __float_as_uint(x);
  const int e = (int)(b >> 23) - 127 + ((b & 0x7fffffu) > top ? 1 : 0);
  return x > 0.f ? e : -kScaleExp;
}
__device__ inline int clamp_exponent(int e) { return min(max(e, -kScaleExp), kScaleExp); }
__device__ inline float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// 448 = 1.75 * 2^8: amax = m 2^e needs 2^(e - 8) if m <= 1.75 and 2^(e - 7) otherwise.
__device__ inline int scale_exponent(float amax) {
  return clamp_exponent(pow2_exponent(amax, 0x600000u) - 8);
}
__device__ inline int old_exponent(float scale) {
  return scale > 0.f ? clamp_exponent(pow2_exponent(scale, 0u)) : -kScaleExp;
}

template <bool BF16>
__device__ inline u32x2 encode8(u32x4 x, float inv) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    b[i] = pkv::e4m3_encode2(pkv::half_bits_to_float<BF16>(x[i] & 0xffffu) * inv,
                             pkv::half_bits_to_float<BF16>(x[i] >> 16) * inv);
  return u32x2{b[0] | b[1] << 16, b[2] | b[3] << 16};
}

// x * r in 32 bits rounded to odd: a later rounding to fewer bits is then the exact product's
// (an old scale need not be a power of two, and x * r could otherwise round to a tie first).
__device__ inline float mul_odd(float x, float r) {
  const float p = x * r, err = __builtin_fmaf(x, r, -p);
  const uint32_t b = __float_as_uint(p);
  if (err == 0.f || (b & 1u)) return p;
  return __uint_as_float((err > 0.f) == (p > 0.f) ? b + 1 : b - 1);
}

// The stored rows first, first + step, ... below `rows` of one (page, head) block, times r (at
// most 1), rounded again; lane c % 16 takes dims 8 c ... of each.
__device__ inline void rescale_rows(uint8_t* block, int first, int step, int rows, float r, int lane) {
  for (int t = first; t < rows; t += step) {
    u32x2* const p = (u32x2*)(block + (long)t * kD + (lane & 15) * 8);
    u32x2 x = *p;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[i], false);
      const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[i], true);
      x[i] = pkv::e4m3_encode2(mul_odd(lo[0], r), mul_odd(lo[1], r)) |
             pkv::e4m3_encode2(mul_odd(hi[0], r), mul_odd(hi[1], r)) << 16;
    }
    *p = x;
  }
}

// One of K and V: the run's tensor, and its page's block.
struct Run {
  const uint8_t* from;  // the run's first token
  long stride;          // bytes between tokens
  uint8_t* block;       // [ps, 128] e4m3
  float* scale;
  int count, off;       // tokens, and the slot of the first in its page
};

// WAVES waves write one run.  Up to 4 * WAVES * ROWS tokens stay in registers between the search
// for the largest magnitude and the rounding (all of their loads are in flight at once); those
// of longer runs are read again.  `lds`: WAVES + 1 words.
template <bool BF16, int WAVES, int ROWS>
__device__ void write_run(const Run& r, int wave, int lane, uint32_t* lds) {
  constexpr int kStep = 4 * WAVES;  // tokens that the waves take at once, four each
  const int sub = 4 * wave + (lane >> 4);
  const uint8_t* const from = r.from + (lane & 15) * 16;
  float old = 1.f;
  if (r.off > 0 && wave == 0) old = *r.scale;
  u32x4 x[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int t = kStep * i + sub;
    x[i] = t < r.count ? *(const u32x4*)(from + t * r.stride) : u32x4{0, 0, 0, 0};
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) m = finite_max<BF16>(m, x[i]);
  for (int t = kStep * ROWS + sub; t < r.count; t += kStep)
    m = finite_max<BF16>(m, *(const u32x4*)(from + t * r.stride));
  m = wave_max<BF16>(m);
  if constexpr (WAVES > 1) {  // the old scale too: read before, and written after, the barrier
    __syncthreads();          // the run before is done with `lds`
    if (lane == 0) lds[wave] = m;
    if (wave == 0 && lane == 0) lds[WAVES] = __float_as_uint(old);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = max2(m, lds[w]);
    old = __uint_as_float(lds[WAVES]);
  }
  int e = scale_exponent(finite_value<BF16>(m));
  if (r.off > 0) {  // earlier tokens share the block: its scale can only grow
    old = fminf(fmaxf(old, pow2(-kScaleExp)), pow2(kScaleExp));
    e = max(e, old_exponent(old));
    if (old != pow2(e)) rescale_rows(r.block, sub, kStep, r.off, old * pow2(-e), lane);
  }
  const float inv = pow2(-e);
  uint8_t* const to = r.block + (long)r.off * kD + (lane & 15) * 8;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int t = kStep * i + sub;
    if (t < r.count) *(u32x2*)(to + (long)t * kD) = encode8<BF16>(x[i], inv);
  }
  for (int t = kStep * ROWS + sub; t < r.count; t += kStep)
    *(u32x2*)(to + (long)t * kD) = encode8<BF16>(*(const u32x4*)(from + t * r.stride), inv);
  if (wave == 0 && lane == 0) *r.scale = pow2(e);
}

// WAVES waves take the runs that begin in their `window` (at most 32) tokens, for one head and
// K or V.  Heads vary fastest, K's before V's: a token's lie next to one another in memory, and
// are read at about the same time.  Every wave's lanes hold the slots of 64 tokens from the one
// before the window on.  A run of up to 64 tokens is one wave's, in its registers; the runs of
// longer pages are shared by the workgroup (one wave took 25 us for the longest of two rows of
// 8270 tokens in pages of 128, four take 9.6) unless they are short.
//
// Bound by memory: 46257 tokens, 8 heads, some continuing a page, 284 MB: 59.7 us in pages of 16
// (4.8 TB/s, where a copy reaches 5.1), 59 of 32, 76 of 64, 115 of 128 (a token's heads are read
// further apart in time).  Four waves a run from pages of 32 on: 95 us of 32, 107 of 64.
template <bool BF16, int WAVES, int ROWS>
__global__ __launch_bounds__(256) void write_block_kernel(WriteArgs a, int window) {
  __shared__ uint32_t lds[WAVES + 1];
  const int id = blockIdx.x * (4 / WAVES) + (WAVES == 1 ? threadIdx.x >> 6 : 0);
  const int wave = WAVES == 1 ? 0 : threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(id / (2 * a.hkv));
  const int part = __builtin_amdgcn_readfirstlane(id - w * (2 * a.hkv));
  const bool is_v = part >= a.hkv;
  const int h = is_v ? part - a.hkv : part;
  const int first = (int)min((long)w * window, (long)a.tokens);
  const int t = first - 1 + lane;
  const int slot = t >= 0 && t < a.tokens ? a.slots[t] : -1;
  const bool valid = slot >= 0 && slot < a.num_slots;
  const int page = valid ? slot / a.page_size : 0, off = slot - page * a.page_size;
  const int before = __shfl_up(slot, 1);  // by every lane: a lane out of step would read as 0
  const bool follows = valid && off > 0 && lane > 0 && before == slot - 1;
  const uint64_t joined = __builtin_amdgcn_ballot_w64(follows);
  const uint64_t mine = ((1ull << window) - 1) << 1;  // lanes of the window's tokens
  uint64_t starts = __builtin_amdgcn_ballot_w64(valid && !follows) & mine;
  int turn = 0;
  while (starts) {
    const int i = __builtin_ctzll(starts);
    starts &= starts - 1;
    const int s0 = __builtin_amdgcn_readlane(slot, i), t0 = first - 1 + i;
    const int p0 = __builtin_amdgcn_readlane(page, i), o0 = __builtin_amdgcn_readlane(off, i);
    // 1 + the lanes behind lane i that follow one another; past lane 63, 64 tokens at a time.
    int count = 1 + min(__builtin_ctzll(~(joined >> (i + 1)) | 1ull << (63 - i)), 63 - i);
    if (i + count == 64) {
      const int most = min(a.page_size - o0, a.tokens - t0);
      for (bool more = true; more && count < most;) {
        const int j = count + lane;
        const uint64_t out = ~__builtin_amdgcn_ballot_w64(j < most && a.slots[t0 + j] == s0 + j);
        const int n = out ? __builtin_ctzll(out) : 64;
        count += n;
        more = n == 64;
      }
    }
    const long block = (long)p0 * a.hkv + h, stride = is_v ? a.v_stride : a.k_stride;
    const Run run{(is_v ? a.v_new : a.k_new) + t0 * stride + (long)h * kRowBytes, stride,
                  (is_v ? a.v_pages : a.k_pages) + block * a.page_size * kD,
                  a.kv_scales + 2 * block + (is_v ? 1 : 0), count, o0};
    if (WAVES > 1 && window > 1 && count <= 16) {  // short runs: a wave each, in turn
      if (turn++ % WAVES == wave) write_run<BF16, 1, 4>(run, 0, lane, lds);
    } else {
      write_run<BF16, WAVES, ROWS>(run, wave, lane, lds);
    }
  }
}

int check_write(const char* op, const WriteArgs& a, int32_t head_dim, int32_t num_pages, int32_t dtype) {
  using pkv::fail;
  if (a.tokens < 0 || a.hkv <= 0 || a.page_size <= 0 || num_pages <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: tokens %d, num_kv_heads %d, page_size %d, num_pages %d",
                op, a.tokens, a.hkv, a.page_size, num_pages);
  if (head_dim != kD) return fail(PKV_ERR_UNSUPPORTED, "%s: head_dim %d (only 128)", op, head_dim);
  if (dtype != PKV_DTYPE_F16 && dtype != PKV_DTYPE_BF16)
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, dtype);
  if ((long)num_pages * a.page_size > INT32_MAX)
    return fail(PKV_ERR_UNSUPPORTED, "%s: num_pages * page_size does not fit in int32", op);
  if ((long)a.tokens * a.hkv > (1L << 30) - 64)
    return fail(PKV_ERR_UNSUPPORTED, "%s: tokens * num_kv_heads too large", op);
  if (a.k_stride < (long)a.hkv * kRowBytes || a.v_stride < (long)a.hkv * kRowBytes ||
      a.k_stride % 16 || a.v_stride % 16)
    return fail(PKV_ERR_INVALID_ARGUMENT,
                "%s: a token stride must hold num_kv_heads * 128 elements and be a multiple of 8", op);
  if (a.tokens == 0) return PKV_OK;
  if (!a.k_new || !a.v_new || !a.k_pages || !a.v_pages || !a.slots)
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: null pointer", op);
  if (((uintptr_t)a.k_new | (uintptr_t)a.v_new | (uintptr_t)a.k_pages | (uintptr_t)a.v_pages) & 15)
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: K and V must be 16-byte aligned", op);
  return PKV_OK;
}

int launched(const char* op) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? pkv::ok() : pkv::fail(PKV_ERR_LAUNCH, "%s launch: %s", op, hipGetErrorString(e));
}

}  // namespace

extern "C" {

int pkv_write_kv(const void* k_new, int64_t k_stride, const void* v_new, int64_t v_stride,
                 void* k_pages, void* v_pages, const int32_t* slot_mapping, int32_t tokens,
                 int32_t num_kv_heads, int32_t head_dim, int32_t num_pages, int32_t page_size,
                 int32_t dtype, void* stream) {
  const WriteArgs a{(const uint8_t*)k_new, (const uint8_t*)v_new, (uint8_t*)k_pages,
                    (uint8_t*)v_pages, nullptr, slot_mapping, 2 * k_stride, 2 * v_stride, tokens,
                    num_kv_heads, page_size, (int32_t)((int64_t)num_pages * page_size)};
  const int st = check_write("write_kv", a, head_dim, num_pages, dtype);
  if (st != PKV_OK || tokens == 0) return st == PKV_OK ? pkv::ok() : st;
  const long lanes = (long)tokens * num_kv_heads * 16;
  const long groups = (lanes + 255) / 256;
  if (!pkv::fits_grid(groups, 256))
    return pkv::fail(PKV_ERR_UNSUPPORTED, "write_kv: tokens * num_kv_heads too large (below 2^28)");
  write_kernel<<<dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream>>>(a);
  return launched("write_kv");
}

int pkv_write_kv_fp8_block(const void* k_new, int64_t k_stride, const void* v_new,
                           int64_t v_stride, void* k_pages, void* v_pages, float* kv_scales,
                           const int32_t* slot_mapping, int32_t tokens, int32_t num_kv_heads,
                           int32_t head_dim, int32_t num_pages, int32_t page_size, int32_t dtype,
                           void* stream) {
  const WriteArgs a{(const uint8_t*)k_new, (const uint8_t*)v_new, (uint8_t*)k_pages,
                    (uint8_t*)v_pages, kv_scales, slot_mapping, 2 * k_stride, 2 * v_stride, tokens,
                    num_kv_heads, page_size, (int32_t)((int64_t)num_pages * page_size)};
  const int st = check_write("write_kv_fp8_block", a, head_dim, num_pages, dtype);
  if (st != PKV_OK || tokens == 0) return st == PKV_OK ? pkv::ok() : st;
  if (!kv_scales || ((uintptr_t)kv_scales & 7))
    return pkv::fail(PKV_ERR_INVALID_ARGUMENT, "write_kv_fp8_block: kv_scales null or not 8-byte aligned");
  // Few tokens: a window each, so that runs that lie next to one another (a decode step's) are
  // not written one after another; else windows of 16 tokens for pages of up to 16, a start or
  // two each, and of 32 for larger ones.  Of long prompts in pages of 64 and 128 every second
  // window and three of four hold no start, and one without still costs 2 us of a CU's place.
  const bool bf16 = dtype == PKV_DTYPE_BF16, shared = page_size > 64;
  const int window = (long)tokens * num_kv_heads <= 4096 ? 1 : page_size > 16 ? 32 : 16;
  const long units = (long)((tokens + window - 1) / window) * num_kv_heads * 2;
  const long groups = shared ? units : (units + 3) / 4;
  if (!pkv::fits_grid(groups, 256))
    return pkv::fail(PKV_ERR_UNSUPPORTED, "write_kv_fp8_block: tokens * num_kv_heads too large (below 2^28)");
  auto* const kernel = shared           ? (bf16 ? write_block_kernel<true, 4, 8> : write_block_kernel<false, 4, 8>)
                       : page_size <= 16 ? (bf16 ? write_block_kernel<true, 1, 4> : write_block_kernel<false, 1, 4>)
                       : page_size <= 32 ? (bf16 ? write_block_kernel<true, 1, 8> : write_block_kernel<false, 1, 8>)
                                         : (bf16 ? write_block_kernel<true, 1, 16> : write_block_kernel<false, 1, 16>);
  kernel<<<dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream>>>(a, window);
  return launched("write_kv_fp8_block");
}

}  // extern "C"
