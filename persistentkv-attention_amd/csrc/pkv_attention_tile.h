// pkv_attention_tile.h — what the attention kernels over tiles of 32 keys in LDS share: element
// types with their matrix instruction, the softmax's constants, wave-wide sums, the wait for loads
// to LDS, and values that are not finite.
#pragma once

#include <hip/hip_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

namespace {

constexpr int kD = 128;
constexpr int kRowBytes = 2 * kD;
constexpr int kKeys = 32;    // keys per tile
constexpr int kWaves = 4;
constexpr int kWaveRows = 32;
constexpr int kTileBytes = kKeys * kRowBytes;
constexpr int kBuffers = 3;  // tiles in LDS: one read, one landed, one on its way
constexpr float kScaleLog2 = 0.08838834764831845f * 1.4426950408889634f;  // log2(e) / sqrt(128)
// The running maximum is replaced only when a score passes it by more than 2^8 in weight:
// the output is rescaled in few tiles, and weights stay below 2^8, far inside fp16's range.
constexpr float kSlack = 8.0f / kScaleLog2;
// Weights are 2^(s c - M c), c = kScaleLog2, in one multiply-add.  M c is rounded: a factor that all
// of a row's weights share, within 2^-13 of 1 for |M| below 2^14 but of any size for larger ones
// (2^32 at |M| = 2^32: past fp16's range, or below it).  From 2^14 on it is (s - M) c.
constexpr float kLargeScore = 0x1p14f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

struct Half {
  static constexpr uint32_t kExponentStep = 0x04000400u;  // one step of both halves' exponents
  static constexpr uint32_t kOne = 0x3c00u;
  __device__ static inline float widen(uint32_t x2, bool high) {
    return (float)__builtin_bit_cast(f16x2, x2)[high];
  }
  // c plus both halves; c where both are finite, else NaN.
  __device__ static inline float sum2(uint32_t x, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x), __builtin_bit_cast(f16x2, kOne * 0x10001u), c, false);
  }
  __device__ static inline float times0(uint32_t x, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x), f16x2{0, 0}, c, false);
  }
  __device__ static inline f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  __device__ static inline uint32_t pack2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
  }
};
struct BFloat {
  static constexpr uint32_t kExponentStep = 0x00800080u;
  static constexpr uint32_t kOne = 0x3f80u;
  __device__ static inline float widen(uint32_t x2, bool high) {
    return __uint_as_float(high ? x2 & 0xffff0000u : x2 << 16);
  }
  __device__ static inline float sum2(uint32_t x, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), __builtin_bit_cast(bf16x2, kOne * 0x10001u), c, false);
  }
  __device__ static inline float times0(uint32_t x, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), bf16x2{0, 0}, c, false);
  }
  __device__ static inline f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  __device__ static inline uint32_t pack2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
  }
};

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline void* uniform_ptr(const void* p) {
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = (uint32_t)uniform((int)(uint32_t)v), hi = (uint32_t)uniform((int)(v >> 32));
  return (void*)(((uint64_t)hi << 32) | lo);
}

template <int CTRL, int ROW_MASK>
__device__ inline int from_lane(int x) {  // 0 where the lane has no source
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROW_MASK, 0xf, false);
}
__device__ inline int wave_scan(int x) {  // inclusive sums
  x += from_lane<0x111, 0xf>(x);          // row_shr 1, 2, 4, 8: within 16 lanes
  x += from_lane<0x112, 0xf>(x);
  x += from_lane<0x114, 0xf>(x);
  x += from_lane<0x118, 0xf>(x);
  x += from_lane<0x142, 0xa>(x);          // row_bcast 15, 31
  return x + from_lane<0x143, 0xc>(x);
}
__device__ inline int wave_max(int x) {  // of values that are not negative
  x = max(x, from_lane<0x111, 0xf>(x));
  x = max(x, from_lane<0x112, 0xf>(x));
  x = max(x, from_lane<0x114, 0xf>(x));
  x = max(x, from_lane<0x118, 0xf>(x));
  x = max(x, from_lane<0x142, 0xa>(x));
  return __builtin_amdgcn_readlane(max(x, from_lane<0x143, 0xc>(x)), 63);
}

// Waits until at most N of the wave's loads are in flight.
template <int N>
__device__ inline void landed() {
  static_assert(N < 16);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70 | N);  // vmcnt(N), nothing else
  asm volatile("" ::: "memory");
}

// The top bits of those halves of a pair of 16-bit floats that are infinite or NaN.
template <class Elem>
__device__ inline uint32_t nonfinite_halves(uint32_t x2) {
  return ((x2 & 0x7fff7fffu) + Elem::kExponentStep) & 0x80008000u;
}
template <class Elem>
__device__ inline uint32_t drop_nonfinite(uint32_t x2) {
  const uint32_t y = nonfinite_halves<Elem>(x2);
  return x2 & ~((y >> 15) * 0xffffu);
}

}  // namespace
