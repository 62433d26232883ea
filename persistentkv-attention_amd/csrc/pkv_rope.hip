// pkv_rope.hip — the norm of every query and key head and its rotation by position, in one pass
// over packed tokens, with K and V left packed or stored straight into the page pools by slot.
// The reference has neither (its harness draws q and filled pools, tests/benchmark_serving_trace.py
// :285-298).
//
//   y = x (mean(x^2) + eps)^(-1/2) w          x: the 128 dims of one (token, head); or y = x
//   a' = a cos - b sin,  b' = b cos + a sin   pairs (a, b) of the first `rot` dims: (i, i + rot / 2)
//                                             or (2 i, 2 i + 1), angle i of the token's position
//
// All in 32 bits, rounded once.  Cosines and sines come from the caller's table: angles of far
// positions need 64 bits, which a program spends once per model, not per token.
//
// Sixteen lanes hold one head, eight dims each; a wave's four groups of them take four tokens and
// HEADS heads one after another, so that angles and weights are read once for those heads and
// all of the heads' loads are in flight together.
//
// Bound by memory: 53,000 tokens, 32 / 8 heads, into the pools, 1.31 GB: 239 us (5.5 TB/s, where a copy
// reaches 5.1); 9,000 tokens of 32 / 32 heads, packed, 293 MB: 57 us (5.2).  64 tokens: 4.8 us, the launch.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pkv.h"
#include "pkv_device.h"

namespace pkv {
int fail(int status, const char* fmt, ...);  // pkv_decode.hip: sets pkv_last_error()
int ok();
}  // namespace pkv

namespace {

constexpr int kD = 128;
constexpr int kRowBytes = 2 * kD;
constexpr int kTokens = 4;  // of a wave

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

struct RopeArgs {
  const uint8_t* x[3];  // q, k, v: token t, head h at x + t * stride + h * 256 (bytes)
  long stride[3];
  uint8_t* out[3];      // q_out, and k_out (packed) or the pools (slots)
  long out_stride[2];
  const float* weight[2];  // of q and k, or null: no norm
  int32_t weight_step[2];  // elements between heads: 0 or 128
  const float* cos_sin;    // [positions, rot]
  const int32_t* positions;
  const int32_t* slots;    // or null: K stays packed
  int32_t tokens, heads[3], parts[3];  // parts: of up to HEADS heads
  int32_t rot, last_position, page_size, num_slots, pairs;
  float eps;
};

template <bool BF16>
__device__ inline float widen(uint32_t x2, int high) {
  if constexpr (BF16) return __uint_as_float(high ? x2 & 0xffff0000u : x2 << 16);
  return (float)__builtin_bit_cast(f16x2, x2)[high];
}
template <bool BF16>
__device__ inline uint32_t narrow2(float a, float b) {
  if constexpr (BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
}

// The sum over the 16 lanes of a head, in all of them.
template <int CTRL>
__device__ inline float add_rotated(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ inline float sum16(float x) {
  x = add_rotated<0x128>(x);  // row_ror 8, 4, 2, 1
  x = add_rotated<0x124>(x);
  x = add_rotated<0x122>(x);
  return add_rotated<0x121>(x);
}

// Sums of squares past 2^128: again with the values 2^-70 times as large (eps no longer counts).
constexpr float kDown = 0x1p-70f;
__device__ inline float norm_factor(const float (&y)[8], float squares, float eps) {
  if (squares < INFINITY) return __builtin_amdgcn_rsqf(squares * (1.0f / kD) + eps);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = __builtin_fmaf(y[i] * kDown, y[i] * kDown, s);
  return __builtin_amdgcn_rsqf(sum16(s) * (1.0f / kD)) * kDown;
}

template <bool BF16, int HEADS>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
  const int lane = threadIdx.x & 63, c = lane & 15;
  const int parts = a.parts[0] + a.parts[1] + a.parts[2];
  const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int block = __builtin_amdgcn_readfirstlane((int)(id / parts));
  int part = __builtin_amdgcn_readfirstlane((int)(id - (long)block * parts));
  int which = 0;  // q, k, v
  while (which < 2 && part >= a.parts[which]) part -= a.parts[which++];
  const int t = block * kTokens + (lane >> 4);
  const int h0 = part * HEADS, count = min(HEADS, a.heads[which] - h0);
  if (t >= a.tokens) return;

  u32x4 x[HEADS];
  const uint8_t* const from = a.x[which] + t * a.stride[which] + (long)h0 * kRowBytes + c * 16;
#pragma unroll
  for (int i = 0; i < HEADS; ++i)
    if (i < count) x[i] = *(const u32x4*)(from + i * kRowBytes);

  uint8_t* to;
  long step = kRowBytes;
  if (which > 0 && a.slots) {
    const int slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots) return;
    const int page = slot / a.page_size, off = slot - page * a.page_size;
    step *= a.page_size;
    to = a.out[which] + ((long)page * a.heads[which] + h0) * step + (long)off * kRowBytes + c * 16;
  } else {
    to = a.out[which] + t * a.out_stride[which & 1] + (long)h0 * kRowBytes + c * 16;
  }
  if (which < 2) {
    // The lane's dims turn by cs[i] and sn[i]: a' = a cs - b sn with its partner b, and the second
    // of a pair with -sn.  Dims from `rot` on turn by nothing.
    const int half = a.rot >> 4;  // lanes of half the dims that turn
    const bool turns = c < 2 * half;
    const int pos = min(max(a.positions[t], 0), a.last_position);
    const float* const angles = a.cos_sin + (long)pos * a.rot;
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i] = 1.f, sn[i] = 0.f;
    if (turns) {
      if (a.pairs) {
        const f32x4 u = *(const f32x4*)(angles + 4 * c), v = *(const f32x4*)(angles + 8 * half + 4 * c);
#pragma unroll
        for (int i = 0; i < 8; ++i) cs[i] = u[i >> 1], sn[i] = i & 1 ? -v[i >> 1] : v[i >> 1];
      } else {
        const float* const p = angles + 8 * (c < half ? c : c - half);
        const f32x4 u0 = *(const f32x4*)p, u1 = *(const f32x4*)(p + 4);
        const f32x4 v0 = *(const f32x4*)(p + 8 * half), v1 = *(const f32x4*)(p + 8 * half + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          cs[i] = i < 4 ? u0[i & 3] : u1[i & 3];
          sn[i] = i < 4 ? v0[i & 3] : v1[i & 3];
          if (c >= half) sn[i] = -sn[i];
        }
      }
    }
    const int partner = (lane & 48) | (turns ? (c < half ? c + half : c - half) : c);
    const float* const weight = a.weight[which];
    float w[8];
    auto read_weight = [&](int h) {
      const f32x4 w0 = *(const f32x4*)(weight + (long)h * a.weight_step[which] + 8 * c);
      const f32x4 w1 = *(const f32x4*)(weight + (long)h * a.weight_step[which] + 8 * c + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = i < 4 ? w0[i & 3] : w1[i & 3];
    };
    if (weight) read_weight(h0);
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      if (i >= count) break;
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = widen<BF16>(x[i][j >> 1], j & 1);
      if (weight) {
        if (i > 0 && a.weight_step[which]) read_weight(h0 + i);
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s = __builtin_fmaf(y[j], y[j], s);
        const float f = norm_factor(y, sum16(s), a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = y[j] * f * w[j];
      }
      float b[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = a.pairs ? y[j ^ 1] : __shfl(y[j], partner);
      if (turns) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = __builtin_fmaf(y[j], cs[j], -b[j] * sn[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; j += 2) x[i][j >> 1] = narrow2<BF16>(y[j], y[j + 1]);
    }
  }
#pragma unroll
  for (int i = 0; i < HEADS; ++i)
    if (i < count) *(u32x4*)(to + i * step) = x[i];
}

// Whether rows of `row` bytes `stride` apart from a on, and such of b, have a byte in common; rows
// whose strides differ count as if they did where the ranges meet.
bool rows_meet(const uint8_t* a, long row_a, long stride_a, const uint8_t* b, long row_b, long stride_b, long rows) {
  if (rows == 0 || a + (rows - 1) * stride_a + row_a <= b || b + (rows - 1) * stride_b + row_b <= a) return false;
  if (rows == 1 || stride_a != stride_b) return true;
  const long d = (((long)(b - a)) % stride_a + stride_a) % stride_a;
  return d < row_a || d + row_b > stride_a;
}

int run(const char* op, RopeArgs& a, int32_t head_dim, int64_t num_pages, int32_t dtype, void* stream) {
  using pkv::fail;
  const bool write = a.heads[2] > 0;
  if (a.tokens < 0 || a.heads[0] <= 0 || a.heads[1] <= 0 || a.last_position < 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: tokens %d, num_q_heads %d, num_kv_heads %d, max_positions %d", op,
                a.tokens, a.heads[0], a.heads[1], a.last_position + 1);
  if (head_dim != kD) return fail(PKV_ERR_UNSUPPORTED, "%s: head_dim %d (only 128)", op, head_dim);
  if (dtype != PKV_DTYPE_F16 && dtype != PKV_DTYPE_BF16)
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, dtype);
  if (a.rot < 16 || a.rot > kD || a.rot % 16)
    return fail(PKV_ERR_UNSUPPORTED, "%s: rotary_dim %d (a multiple of 16, at most 128)", op, a.rot);
  if ((a.weight[0] || a.weight[1]) && !(a.eps >= 0x1p-100f && a.eps <= 0x1p100f))
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: eps %g (2^-100 to 2^100)", op, (double)a.eps);
  if (write && (a.page_size <= 0 || num_pages <= 0))
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: page_size %d, num_pages %ld", op, a.page_size, (long)num_pages);
  if (write && num_pages * a.page_size > INT32_MAX)
    return fail(PKV_ERR_UNSUPPORTED, "%s: num_pages * page_size does not fit in int32", op);
  const int outs = write ? 1 : 2, ins = write ? 3 : 2;
  for (int i = 0; i < ins; ++i)
    if (a.stride[i] < (long)a.heads[i] * kRowBytes || a.stride[i] % 16 ||
        (i < outs && (a.out_stride[i] < (long)a.heads[i] * kRowBytes || a.out_stride[i] % 16)))
      return fail(PKV_ERR_INVALID_ARGUMENT, "%s: a token stride must hold its heads and be a multiple of 8 elements", op);
  // Heads a wave.  Few in all: one, so that none waits for another's (16 tokens of 56 heads 4.7 us for
  // 5.2 with two, 5.7 with four); then two (4096 tokens: 20.7 us for 23.6 with one, 22.4 with four and
  // 26 with eight); four where memory is what all wait for (53,000 tokens: 241 us for 249 with two,
  // 328 with one, 244 with eight).
  const long rows = (long)a.tokens * (a.heads[0] + (ins - 1) * (long)a.heads[1]);
  const int each = rows <= 2048 ? 1 : rows <= 1 << 20 ? 2 : 4;
  long parts = 0;
  for (int i = 0; i < 3; ++i) parts += a.parts[i] = (int32_t)(((long)a.heads[i] + each - 1) / each);
  const long waves = ((long)a.tokens + kTokens - 1) / kTokens * parts, groups = (waves + 3) / 4;
  if (!pkv::fits_grid(groups, 256) || parts > INT32_MAX)
    return fail(PKV_ERR_UNSUPPORTED, "%s: too many tokens or heads", op);
  if (a.tokens == 0) return pkv::ok();
  uintptr_t all = (uintptr_t)a.cos_sin | (uintptr_t)a.weight[0] | (uintptr_t)a.weight[1];
  for (int i = 0; i < ins; ++i) {
    if (!a.x[i] || !a.out[i]) return fail(PKV_ERR_INVALID_ARGUMENT, "%s: null pointer", op);
    all |= (uintptr_t)a.x[i] | (uintptr_t)a.out[i];
  }
  if (!a.cos_sin || !a.positions || (write && !a.slots)) return fail(PKV_ERR_INVALID_ARGUMENT, "%s: null pointer", op);
  if (all & 15) return fail(PKV_ERR_INVALID_ARGUMENT, "%s: tensors must be 16-byte aligned", op);
  // A head is read and written by the same lanes, so an output may be its own input; any other
  // overlap would be written while others read it.
  for (int o = 0; o < outs; ++o) {
    const long row = (long)a.heads[o] * kRowBytes;
    for (int i = 0; i < ins; ++i)
      if (!(i == o && a.out[o] == a.x[o] && (a.tokens == 1 || a.out_stride[o] == a.stride[o])) &&
          rows_meet(a.out[o], row, a.out_stride[o], a.x[i], (long)a.heads[i] * kRowBytes, a.stride[i], a.tokens))
        return fail(PKV_ERR_INVALID_ARGUMENT, "%s: %s must be its own input or overlap none", op, o ? "k_out" : "q_out");
  }
  if (outs == 2 && rows_meet(a.out[0], (long)a.heads[0] * kRowBytes, a.out_stride[0], a.out[1],
                             (long)a.heads[1] * kRowBytes, a.out_stride[1], a.tokens))
    return fail(PKV_ERR_INVALID_ARGUMENT, "%s: q_out and k_out must not overlap", op);
  const bool bf16 = dtype == PKV_DTYPE_BF16;
  auto* const kernel = each == 1   ? (bf16 ? rope_kernel<true, 1> : rope_kernel<false, 1>)
                       : each == 2 ? (bf16 ? rope_kernel<true, 2> : rope_kernel<false, 2>)
                                   : (bf16 ? rope_kernel<true, 4> : rope_kernel<false, 4>);
  kernel<<<dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? pkv::ok() : fail(PKV_ERR_LAUNCH, "%s launch: %s", op, hipGetErrorString(e));
}

}  // namespace

extern "C" {

int pkv_norm_rope(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                  const float* q_weight, int32_t q_weight_heads, const float* k_weight,
                  int32_t k_weight_heads, const float* cos_sin, const int32_t* positions, void* q_out,
                  int64_t q_out_stride, void* k_out, int64_t k_out_stride, int32_t tokens,
                  int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t rotary_dim,
                  int32_t max_positions, int32_t interleaved, float eps, int32_t dtype, void* stream) {
  if ((q_weight && q_weight_heads != 1 && q_weight_heads != num_q_heads) ||
      (k_weight && k_weight_heads != 1 && k_weight_heads != num_kv_heads))
    return pkv::fail(PKV_ERR_INVALID_ARGUMENT, "norm_rope: weights of one head, or of every head");
  RopeArgs a{{(const uint8_t*)q, (const uint8_t*)k, nullptr}, {2 * q_stride, 2 * k_stride, 0},
             {(uint8_t*)q_out, (uint8_t*)k_out, nullptr}, {2 * q_out_stride, 2 * k_out_stride},
             {q_weight, k_weight}, {q_weight_heads > 1 ? kD : 0, k_weight_heads > 1 ? kD : 0},
             cos_sin, positions, nullptr, tokens, {num_q_heads, num_kv_heads, 0}, {}, rotary_dim,
             max_positions - 1, 0, 0, interleaved, eps};
  return run("norm_rope", a, head_dim, 0, dtype, stream);
}

int pkv_norm_rope_write_kv(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                           const void* v, int64_t v_stride, const float* q_weight,
                           int32_t q_weight_heads, const float* k_weight, int32_t k_weight_heads,
                           const float* cos_sin, const int32_t* positions, void* q_out,
                           int64_t q_out_stride, void* k_pages, void* v_pages,
                           const int32_t* slot_mapping, int32_t tokens, int32_t num_q_heads,
                           int32_t num_kv_heads, int32_t head_dim, int32_t rotary_dim,
                           int32_t max_positions, int32_t interleaved, float eps, int32_t num_pages,
                           int32_t page_size, int32_t dtype, void* stream) {
  if ((q_weight && q_weight_heads != 1 && q_weight_heads != num_q_heads) ||
      (k_weight && k_weight_heads != 1 && k_weight_heads != num_kv_heads))
    return pkv::fail(PKV_ERR_INVALID_ARGUMENT, "norm_rope_write_kv: weights of one head, or of every head");
  RopeArgs a{{(const uint8_t*)q, (const uint8_t*)k, (const uint8_t*)v}, {2 * q_stride, 2 * k_stride, 2 * v_stride},
             {(uint8_t*)q_out, (uint8_t*)k_pages, (uint8_t*)v_pages}, {2 * q_out_stride, 0},
             {q_weight, k_weight}, {q_weight_heads > 1 ? kD : 0, k_weight_heads > 1 ? kD : 0},
             cos_sin, positions, slot_mapping, tokens, {num_q_heads, num_kv_heads, num_kv_heads}, {},
             rotary_dim, max_positions - 1, page_size,
             (int32_t)((int64_t)num_pages * page_size <= INT32_MAX ? (int64_t)num_pages * page_size : 0),
             interleaved, eps};
  return run("norm_rope_write_kv", a, head_dim, num_pages, dtype, stream);
}

}  // extern "C"
