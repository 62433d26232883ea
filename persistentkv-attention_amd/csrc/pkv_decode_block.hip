// pkv_decode_block.hip — paged GQA decode attention over fp8 (OCP e4m3) K/V with one scale per
// (page, KV head), K and V apart: K = ks[p] K8, V = vs[p] V8 (pkv_write_kv_fp8_block writes
// such pools).  The reference names dequantising paged decode as future work
// (paper/persistentkv_mlsys_workshop.tex:688-690).
//
// Mathematics.  With x_j = ks q.k8_j / sqrt(128) (in units of log2) and y_j = x_j + log2 vs_j,
//   out = sum_j 2^x_j vs_j v8_j / sum_j 2^x_j = sum_j 2^(y_j - M) v8_j / sum_j 2^(y_j - M) / vs_j
// where M is the running maximum of y, not of x.  The weights 2^(y - M) enter the product with
// V in 16 bits, so those that matter for the output are the ones near 1, whatever the scales
// of their pages: weights 2^(x - m) vs_j would be subnormal in fp16 where vs is small.  V8 is
// exact in 16 bits, and the scales cost one add and one multiply-add per 16 tokens, since a
// block of 16 tokens lies in one page and its scales are wave-uniform.
//
// Schedule.  All (row, KV head) pairs' 32-token tiles, and kPieceCost positions for the start
// of each pair, form one line, cut into equal shares, one a wave; the grid fills the GPU
// once.  Every workgroup computes the cut from the lengths (a scan in LDS), so nothing is
// planned on the host and the call can be captured for lengths that change.  A pair inside one
// share is written to the output, the others as partial states, at most two a wave, and
// joined by the merge kernel.  Tables of few tokens take one launch instead, a workgroup a pair
// (short_block_kernel).
//
// Per wave and tile: K and V straight from the pages into registers (16- and 8-byte buffer
// loads whose descriptor ends with the row's last token), S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_16x16x32, heads padded to 16 a block.  Two tiles (16 KB) in flight in each of a CU's
// four waves keep HBM busy: 64 Zipf rows (bf16, G = 8, 600 MB) 97-99 us, 6.1 TB/s; 8 bimodal
// rows (fp16, G = 4, 95 MB) 19.5 us, 4.9 TB/s, of which about 3 us pass before the first bytes;
// then 4 to 6 us of merge.  For G above 16 a wave holds two blocks of heads in 254 registers and
// takes twice the products a tile: 128 rows of 8192, 32 / 1 heads (268 MB), 62 us and 4.3 TB/s, 64 / 2
// heads (537 MB) 119 us and 4.5, where 32 rows of 8192 at 32 / 8 (537 MB) take 91 us and 5.9.

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
constexpr int kTile = 32;
constexpr int kWaves = 4;            // per workgroup, one workgroup per CU
constexpr int kPieceCost = 2;        // positions that a pair's start counts for
constexpr int kMinShare = 2;         // positions of a share
constexpr int kMaxRows = 16000;      // an LDS prefix of 4 bytes a row
constexpr int kStateFloats = kD + 2; // acc, m, l
constexpr int kMergeWaves = 4;
constexpr int kShortWaves = 8;       // of a workgroup that takes a (row, KV head) of a short table,
constexpr int kShortTokens = 512;    // which addresses at most this many tokens (see there)
constexpr int kKvLoadPolicy = 2;     // non-temporal: K/V bytes are read once
constexpr uint32_t kRsrcWord3 = 0x00020000u;  // raw buffer, 32-bit data format (gfx9 family)
constexpr float kScaleLog2 = 0.08838834764831845f * 1.4426950408889634f;  // log2(e) / sqrt(128)
constexpr float kSlack = 8.0f;       // the running maximum lags by at most this (log2)
constexpr float kScaleMin = 0x1p-60f, kScaleMax = 0x1p60f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// P enters the PV product in the activation type; bf16 keeps 8 bits, so its P is split into
// two terms (two products), as the framework's other decode kernels split it.
//
// kLift: the state's m lies this far below the maximum of y, so that the largest weights are
// 2^kLift.  Where pages' scales of V are 2^120 apart, a token of a small-scaled page that counts
// in the sum has a weight next to 2^-126, the end of fp32's range (v_exp gives 0 below it); with
// 2^30 in hand what is lost there is below 2^-36 of the largest token's share.  fp16's weights
// have no such room, and scales of V so far apart have no output in fp16.
struct Half {
  static constexpr int kPasses = 1;
  static constexpr float kLift = 0.f;
  __device__ static inline f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  __device__ static inline uint32_t pack2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
  }
  template <bool HI>  // e4m3 bytes 2 HI and 2 HI + 1 of x, exactly
  __device__ static inline uint32_t fp8_pair(uint32_t x) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x, 1.0f, HI));
  }
};
struct BFloat {
  static constexpr int kPasses = 2;
  static constexpr float kLift = 30.f;
  __device__ static inline f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  __device__ static inline uint32_t pack2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
  }
  template <bool HI>
  __device__ static inline uint32_t fp8_pair(uint32_t x) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x, 1.0f, HI));
  }
};

struct BlockArgs {
  const uint8_t* q;           // [B, Hq, 128]
  const uint8_t* k_pages;     // [num_pages, Hkv, ps, 128] e4m3
  const uint8_t* v_pages;
  const float* kv_scales;     // [num_pages, Hkv, 2]
  const int32_t* block_table; // [B, max_pages]
  const int32_t* seq_lens;    // [B]
  uint8_t* output;            // [B, Hq, 128]
  float* acc;                 // [2 * waves, G, 128] partial states: sum 2^(y - m) v8,
  f32x2* ml;                  // [2 * waves, G] m, and sum 2^(y - m) / vs
  int2* plan;                 // [B * Hkv] first and last wave of the pair (first > last: empty)
  int32_t batch, hkv, group, num_pages, page_size, page_shift, max_pages, waves;
};

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline void* uniform_ptr(const void* p) {
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = (uint32_t)uniform((int)(uint32_t)v), hi = (uint32_t)uniform((int)(v >> 32));
  return (void*)(((uint64_t)hi << 32) | lo);
}
// Wave-uniform reads through the scalar cache: waiting for them never waits for K/V loads.
__device__ inline int load_scalar(const int32_t* p) {
  return uniform(*(const __attribute__((address_space(4))) int32_t*)p);
}

// Tokens of a row, at most what its table row can address (below 2^31, see the launch).
__device__ inline int clamp_length(const BlockArgs& a, int n) {
  return min(max(n, 0), a.max_pages * a.page_size);
}
__device__ inline int row_positions(const BlockArgs& a, int row) {
  const int n = clamp_length(a, a.seq_lens[row]);
  return n ? (n + kTile - 1) / kTile + kPieceCost : 0;
}

struct Tile {
  u32x4 k[2][2];  // [block of 16 tokens][16-byte half]: token lane % 16, dims 32 (lane / 16) ...
  u32x2 v[8];     // token 16 (j / 4) + 4 (lane / 16) + j % 4, dims 8 (lane % 16) ...
  float ks[2], vs[2];
};

struct Pages {
  int page[2];
};

struct Stream {
  const BlockArgs& a;
  const int32_t* table;
  int kvh, len, lane;

  __device__ inline void page_of(int token, int& logical, int& in_page) const {
    logical = a.page_shift >= 0 ? token >> a.page_shift : token / a.page_size;
    in_page = token - logical * a.page_size;
    logical = min(logical, a.max_pages - 1);
  }
  __device__ inline Pages lookup(int tile) const {
    Pages p;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      int logical, in_page;
      page_of(tile * kTile + b * 16, logical, in_page);
      p.page[b] = load_scalar(table + logical);
    }
    return p;
  }
  __device__ inline void issue(int tile, const Pages& p, Tile& r) const {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int tok0 = tile * kTile + b * 16;
      const int valid = min(max(len - tok0, 0), 16);
      int logical, in_page;
      page_of(tok0, logical, in_page);
      const long block = (long)min(max(p.page[b], 0), a.num_pages - 1) * a.hkv + kvh;
      const long off = valid ? (block * a.page_size + in_page) * kD : 0;
      const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
          uniform_ptr(a.k_pages + off), (short)0, uniform(valid * kD), kRsrcWord3);
      const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
          uniform_ptr(a.v_pages + off), (short)0, uniform(valid * kD), kRsrcWord3);
      const int c = lane & 15, g = lane >> 4;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        r.k[b][h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
            rk, c * kD + g * 32 + h * 16, 0, kKvLoadPolicy));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        r.v[4 * b + j] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(
            rv, (4 * g + j) * kD + c * 8, 0, kKvLoadPolicy));
      const int32_t* s = (const int32_t*)a.kv_scales + 2 * block;
      r.ks[b] = __builtin_bit_cast(float, load_scalar(s));
      r.vs[b] = __builtin_bit_cast(float, load_scalar(s + 1));
    }
  }
};

template <int HB>
struct State {
  float m[HB], l[HB];   // l: this lane's tokens only
  f32x4 o[HB][8];       // o[hb][jj][i]: dim 8 (4 (lane / 16) + i) + jj of head 16 hb + lane % 16
};

// The square root of 2^x.  A state's l is a sum of weights over scales of V, up to 2^60 and more
// times its weights: 2^x, taken by itself, may be below fp32's range where l 2^x is not.
__device__ inline float half_weight(float x) { return __builtin_amdgcn_exp2f(0.5f * x); }

template <class Elem, int HB>
__device__ inline void compute(State<HB>& st, const Tile& r, const u32x4 (&q)[HB][4], int tile,
                               int len, int lane) {
  const int g = lane >> 4;
  float qk[2], lv[2], iv[2];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const float vs = fminf(fmaxf(r.vs[b], kScaleMin), kScaleMax);
    qk[b] = fminf(fmaxf(r.ks[b], kScaleMin), kScaleMax) * kScaleLog2;
    lv[b] = __builtin_amdgcn_logf(vs);
    iv[b] = __builtin_amdgcn_rcpf(vs);
  }
  u32x4 vt[8];  // vt[jj]: the lane's 8 tokens of dim 8 (lane % 16) + jj
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      // (token 2t dim 2m, token 2t + 1 dim 2m, token 2t dim 2m + 1, token 2t + 1 dim 2m + 1)
      const uint32_t x = __builtin_amdgcn_perm(r.v[2 * t + 1][m >> 1], r.v[2 * t][m >> 1],
                                               (m & 1) ? 0x07030602u : 0x05010400u);
      vt[2 * m][t] = Elem::template fp8_pair<false>(x);
      vt[2 * m + 1][t] = Elem::template fp8_pair<true>(x);
    }
#pragma unroll
  for (int hb = 0; hb < HB; ++hb) {
    float y[8];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const uint32_t x0 = r.k[b][kk >> 1][2 * (kk & 1)], x1 = r.k[b][kk >> 1][2 * (kk & 1) + 1];
        s = Elem::mma(u32x4{Elem::template fp8_pair<false>(x0), Elem::template fp8_pair<true>(x0),
                            Elem::template fp8_pair<false>(x1), Elem::template fp8_pair<true>(x1)},
                      q[hb][kk], s);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) y[4 * b + i] = __builtin_fmaf(s[i], qk[b], lv[b]);
    }
    if ((tile + 1) * kTile > len) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (tile * kTile + 16 * (j >> 2) + 4 * g + (j & 3) >= len) y[j] = -INFINITY;
    }
    float mx = y[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mx = fmaxf(mx, y[j]);
    if (__builtin_amdgcn_ballot_w64(mx > st.m[hb] + (Elem::kLift + kSlack)) != 0) {
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(st.m[hb], fmaxf(mx, __shfl_xor(mx, 32)) - Elem::kLift);
      const float root = half_weight(st.m[hb] - mx), c = root * root;
      st.m[hb] = mx;
      st.l[hb] = st.l[hb] * root * root;
#pragma unroll
      for (int jj = 0; jj < 8; ++jj) st.o[hb][jj] *= c;
    }
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(y[j] - st.m[hb]);
    st.l[hb] = __builtin_fmaf((p[0] + p[1]) + (p[2] + p[3]), iv[0],
                              __builtin_fmaf((p[4] + p[5]) + (p[6] + p[7]), iv[1], st.l[hb]));
    u32x4 pa;
#pragma unroll
    for (int t = 0; t < 4; ++t) pa[t] = Elem::pack2(p[2 * t], p[2 * t + 1]);
#pragma unroll
    for (int pass = 0; pass < Elem::kPasses; ++pass) {
      if (pass == 1) {  // what the first rounding left (a bf16 value is its bits << 16)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          pa[t] = Elem::pack2(p[2 * t] - __builtin_bit_cast(float, pa[t] << 16),
                              p[2 * t + 1] - __builtin_bit_cast(float, pa[t] & 0xffff0000u));
      }
#pragma unroll
      for (int jj = 0; jj < 8; ++jj) st.o[hb][jj] = Elem::mma(vt[jj], pa, st.o[hb][jj]);
    }
  }
}

template <class Elem>
__device__ inline u32x4 pack8(const f32x4 (&o)[8], int i, float f) {
  return u32x4{Elem::pack2(o[0][i] * f, o[1][i] * f), Elem::pack2(o[2][i] * f, o[3][i] * f),
               Elem::pack2(o[4][i] * f, o[5][i] * f), Elem::pack2(o[6][i] * f, o[7][i] * f)};
}

// Tiles [t0, t1) of (row, kvh).  `state` < 0: the whole pair, written to the output; else that
// place in `states` and `ml`.
template <class Elem, int HB>
__device__ void piece(const BlockArgs& a, int row, int kvh, int t0, int t1, int state, float* states,
                      f32x2* ml, int lane) {
  const int c = lane & 15, g = lane >> 4;
  Stream stream{a, a.block_table + (long)row * a.max_pages, kvh, 0, lane};
  Pages pa = stream.lookup(t0), pb = stream.lookup(t0 + 1);
  stream.len = min(clamp_length(a, load_scalar(a.seq_lens + row)), t1 * kTile);
  u32x4 q[HB][4];
#pragma unroll
  for (int hb = 0; hb < HB; ++hb) {
    const int head = min(16 * hb + c, a.group - 1);
    const uint8_t* p = a.q + (((long)row * a.hkv + kvh) * a.group + head) * (2 * kD) + g * 64;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) q[hb][kk] = *(const u32x4*)(p + kk * 16);
  }
  State<HB> st;
#pragma unroll
  for (int hb = 0; hb < HB; ++hb) {
    st.m[hb] = -INFINITY;
    st.l[hb] = 0.f;
#pragma unroll
    for (int jj = 0; jj < 8; ++jj) st.o[hb][jj] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Two tiles in flight; loads of tile t1 cover no tokens and read nothing.
  Tile ra, rb;
  stream.issue(t0, pa, ra);
  int t = t0;
  for (; t + 1 < t1; t += 2) {
    stream.issue(t + 1, pb, rb);
    pa = stream.lookup(t + 2);
    compute<Elem, HB>(st, ra, q, t, stream.len, lane);
    stream.issue(t + 2, pa, ra);
    pb = stream.lookup(t + 3);
    compute<Elem, HB>(st, rb, q, t + 1, stream.len, lane);
  }
  if (t < t1) compute<Elem, HB>(st, ra, q, t, stream.len, lane);

#pragma unroll
  for (int hb = 0; hb < HB; ++hb) {
    float l = st.l[hb] + __shfl_xor(st.l[hb], 16);
    l += __shfl_xor(l, 32);
    const int head = 16 * hb + c;
    if (head >= a.group) continue;
    if (state < 0) {
      const float inv = 1.0f / l;
      u32x4* out = (u32x4*)(a.output + (((long)row * a.hkv + kvh) * a.group + head) * (2 * kD) + g * 64);
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = pack8<Elem>(st.o[hb], i, inv);
    } else {
      const long at = (long)state * a.group + head;
      if (g == 0) ml[at] = f32x2{st.m[hb], l};
      f32x4* acc = (f32x4*)(states + at * kD + g * 32);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int jj = 0; jj < 8; jj += 4)
          acc[2 * i + jj / 4] = f32x4{st.o[hb][jj][i], st.o[hb][jj + 1][i], st.o[hb][jj + 2][i], st.o[hb][jj + 3][i]};
    }
  }
}

template <int CTRL, int ROW_MASK>
__device__ inline uint32_t dpp_add(uint32_t x) {
  return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROW_MASK, 0xf, false);
}
__device__ inline uint32_t wave_scan(uint32_t x) {  // inclusive sums
  x = dpp_add<0x111, 0xf>(x);                       // row_shr 1, 2, 4, 8: within 16 lanes
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);                       // row_bcast 15, 31
  return dpp_add<0x143, 0xc>(x);
}

template <class Elem, int HB>
__global__ __launch_bounds__(kWaves * 64) void decode_block_kernel(BlockArgs a) {
  extern __shared__ uint32_t prefix[];  // [B + 1] exclusive prefix of the rows' positions, then sums
  uint32_t* const sums = prefix + a.batch + 1;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t before = 0;
  for (int base = 0; base < a.batch; base += kWaves * 64) {
    const int row = base + tid;
    uint32_t x = row < a.batch ? (uint32_t)row_positions(a, row) : 0;
    x = wave_scan(x);
    if (lane == 63) sums[wave] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) x += sums[w];
    }
    if (row < a.batch) prefix[row + 1] = before + x;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) before += sums[w];
    __syncthreads();
  }
  if (tid == 0) prefix[0] = 0;
  __syncthreads();
  const uint32_t total = before * (uint32_t)a.hkv;
  const uint32_t share = max((total + a.waves - 1) / (uint32_t)a.waves, (uint32_t)kMinShare);

  // The waves of each pair, for the merge.
  for (int pair = blockIdx.x * kWaves * 64 + tid; pair < a.batch * a.hkv; pair += gridDim.x * kWaves * 64) {
    const int row = pair / a.hkv, h = pair - row * a.hkv;
    const uint32_t n = prefix[row + 1] - prefix[row];
    const uint32_t at = prefix[row] * (uint32_t)a.hkv + h * n;
    a.plan[pair] = n ? int2{(int)((at + kPieceCost) / share), (int)((at + n - 1) / share)} : int2{0, -1};
  }

  const uint32_t w = uniform((int)(blockIdx.x * kWaves + wave));
  uint32_t x = w * share;
  const uint32_t end = min(x + share, total);
  if (x >= end) return;
  int row = 0;
  {
    int hi = a.batch;  // prefix[row] * hkv <= x < prefix[hi] * hkv
    while (hi - row > 1) {
      const int mid = (row + hi) >> 1;
      if (prefix[mid] * (uint32_t)a.hkv <= x) row = mid;
      else hi = mid;
    }
  }
  row = uniform(row);
  while (x < end) {
    const uint32_t n = (uint32_t)uniform((int)(prefix[row + 1] - prefix[row]));
    const uint32_t row0 = (uint32_t)uniform((int)(prefix[row] * (uint32_t)a.hkv));
    if (x >= row0 + n * (uint32_t)a.hkv) {
      ++row;
      continue;
    }
    const uint32_t h = (x - row0) / n, at = row0 + h * n;
    const uint32_t stop = min(at + n, end);
    const int t0 = max((int)(x - at) - kPieceCost, 0), t1 = (int)(stop - at) - kPieceCost;
    if (t1 > t0) {
      const bool first = at + kPieceCost >= w * share, last = stop == at + n;
      piece<Elem, HB>(a, row, (int)h, t0, t1, first && last ? -1 : (int)(2 * w + (first ? 1 : 0)), a.acc, a.ml, lane);
    }
    x = stop;
  }
}

// Joins the partial states of one (pair, head); an empty row's output is zero.  Every wave
// computes the states' weights 2^(m - M) for itself, a state a lane; then half a wave reads one
// state's 512 bytes of sums, so that a workgroup has 8 states in flight in each of kUnroll steps.
// (One wave a head, a state after another, took 10 to 22 us where this takes 4 to 6.)
template <class Elem>
__global__ __launch_bounds__(kMergeWaves * 64) void merge_block_kernel(BlockArgs a) {
  constexpr int kUnroll = 4, kHalves = 2 * kMergeWaves;
  __shared__ f32x4 part[kHalves][kD / 4];
  const int id = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int pair = id / a.group, head = id - pair * a.group;
  const int2 p = a.plan[pair];
  uint8_t* const out = a.output + (long)id * (2 * kD);
  if (p.x == p.y) return;
  if (p.x > p.y) {
    if (tid < kD / 4) *(u32x2*)(out + tid * 8) = u32x2{0, 0};
    return;
  }
  const int n = p.y - p.x + 1;  // state i is wave p.x + i's: its last piece for i = 0, else its first
  auto state = [&](int i) { return (long)(2 * (p.x + i) + (i == 0 ? 1 : 0)) * a.group + head; };
  // The sums' first loads go out before the maxima are known: only the pair's waves place them.
  const int half = tid >> 5, c = tid & 31;
  f32x4 x[kUnroll];
  float w[kUnroll];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long at = state(min(i0 + u * kHalves, n - 1));
      x[u] = *(const f32x4*)(a.acc + at * kD + 4 * c);
      w[u] = a.ml[at][0];
    }
  };
  load(half);
  float m = -INFINITY;
  const f32x2 own = lane < n ? a.ml[state(lane)] : f32x2{-INFINITY, 0.f};
  for (int i = lane + 64; i < n; i += 64) m = fmaxf(m, a.ml[state(i)][0]);
  m = fmaxf(m, own[0]);
#pragma unroll
  for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  const float root = half_weight(own[0] - m);
  float l = own[1] * root * root;
  for (int i = lane + 64; i < n; i += 64) {
    const f32x2 y = a.ml[state(i)];
    const float r = half_weight(y[0] - m);
    l = __builtin_fmaf(y[1] * r, r, l);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = half;;) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i0 + u * kHalves < n) {
        const float f = __builtin_amdgcn_exp2f(w[u] - m);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = __builtin_fmaf(x[u][j], f, acc[j]);
      }
    i0 += kHalves * kUnroll;
    if (i0 >= n) break;
    load(i0);
  }
  part[half][c] = acc;
  __syncthreads();
  if (tid < kD / 4) {
    f32x4 sum = part[0][tid];
#pragma unroll
    for (int h = 1; h < kHalves; ++h) sum += part[h][tid];
    *(u32x2*)(out + tid * 8) = u32x2{Elem::pack2(sum[0] / l, sum[1] / l), Elem::pack2(sum[2] / l, sum[3] / l)};
  }
}

// Tables of few tokens: a workgroup takes a (row, KV head), its waves the tiles in equal parts,
// and joins their states in LDS.  One launch, no cut and no plan (32 / 8 heads, fp16, 1 row: 64
// tokens 3.8 us where the cut takes 6.6, 512 tokens 7.1 and 8.4; 32 rows: 4.1 and 7.0, 9.1 and
// 14.2; 64 rows of 512: 16.3 and 20.1).  A CU by itself gets 34 GB/s, so 1024 tokens of one row
// take 10.9 where the cut over all CUs takes 8.9; only pairs for every CU make up for that (32
// rows of 1024: 14.0 and 19.2, of 1-1024: 12.6 and 14.7; 40 rows, the worst: 23.3 and 22.1).  Past two
// pairs a CU the starts count: 128 rows of 512 take 30.1 and 26.3.  For G up to 16 only: the states of
// 32 heads would take 128 KB of LDS; larger groups go through the cut (1 row of 400 tokens, 32 / 1
// heads: 10.4 us).
template <class Elem>
__global__ __launch_bounds__(kShortWaves * 64) void short_block_kernel(BlockArgs a) {
  __shared__ __attribute__((aligned(16))) float states[kShortWaves * 16 * kD];  // [wave, head, 128]
  __shared__ f32x2 ml[kShortWaves * 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int row = uniform((int)(blockIdx.x / (unsigned)a.hkv)), kvh = uniform((int)(blockIdx.x % (unsigned)a.hkv));
  const int tiles = (clamp_length(a, load_scalar(a.seq_lens + row)) + kTile - 1) / kTile;
  const int n = min(tiles, kShortWaves);
  if (wave < n)
    piece<Elem, 1>(a, row, kvh, wave * tiles / n, (wave + 1) * tiles / n, n == 1 ? -1 : wave, states, ml, lane);
  if (n == 1) return;
  __syncthreads();
  uint8_t* const out = a.output + (long)blockIdx.x * a.group * (2 * kD);
  for (int i = tid; i < a.group * (kD / 4); i += kShortWaves * 64) {
    const int head = i / (kD / 4);
    float m = -INFINITY, l = 0.f;
    for (int w = 0; w < n; ++w) m = fmaxf(m, ml[w * a.group + head][0]);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < n; ++w) {
      const f32x2 y = ml[w * a.group + head];
      const float root = half_weight(y[0] - m), f = root * root;
      const f32x4 x = *(const f32x4*)(states + w * a.group * kD + 4 * i);
      l = __builtin_fmaf(y[1] * root, root, l);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] = __builtin_fmaf(x[j], f, sum[j]);
    }
    const float inv = n ? 1.0f / l : 0.f;  // no token: zero
    *(u32x2*)(out + i * 8) = u32x2{Elem::pack2(sum[0] * inv, sum[1] * inv), Elem::pack2(sum[2] * inv, sum[3] * inv)};
  }
}

size_t workspace_bytes(int64_t batch, int64_t hkv, int64_t group) {
  const size_t states = 2 * (size_t)pkv::compute_units() * kWaves * group * kStateFloats * sizeof(float);
  return states + (size_t)batch * hkv * sizeof(int2);
}

template <class Elem, int HB>
void launch(const BlockArgs& a, hipStream_t s) {
  if constexpr (HB == 1) {
    const int pairs = a.batch * a.hkv, cus = a.waves / kWaves;
    if (a.max_pages * a.page_size <= (pairs < cus ? kShortTokens : 2 * kShortTokens) && pairs <= 2 * cus) {
      short_block_kernel<Elem><<<dim3((unsigned)(a.batch * a.hkv)), dim3(kShortWaves * 64), 0, s>>>(a);
      return;
    }
  }
  const size_t lds = (size_t)(a.batch + 1 + kWaves) * sizeof(uint32_t);
  decode_block_kernel<Elem, HB><<<dim3((unsigned)(a.waves / kWaves)), dim3(kWaves * 64), lds, s>>>(a);
  const long heads = (long)a.batch * a.hkv * a.group;
  merge_block_kernel<Elem><<<dim3((unsigned)heads), dim3(kMergeWaves * 64), 0, s>>>(a);
}

}  // namespace

extern "C" {

size_t pkv_fp8_block_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads) {
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads) return 0;
  return workspace_bytes(batch, num_kv_heads, num_q_heads / num_kv_heads);
}

int pkv_paged_attention_fp8_block(
    const void* q, const void* k_pages, const void* v_pages, const float* kv_scales,
    const int32_t* block_table, const int32_t* seq_lens, void* output, void* workspace,
    size_t workspace_size, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t num_pages, int32_t page_size, int32_t max_pages, int32_t dtype,
    void* stream) {
  using pkv::fail;
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_pages <= 0 || page_size <= 0 || max_pages <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT,
                "paged_attention_fp8_block: batch %d, num_q_heads %d, num_kv_heads %d, num_pages %d, "
                "page_size %d, max_pages %d",
                batch, num_q_heads, num_kv_heads, num_pages, page_size, max_pages);
  if (head_dim != kD) return fail(PKV_ERR_UNSUPPORTED, "paged_attention_fp8_block: d=%d (only d=128)", head_dim);
  if (dtype != PKV_DTYPE_F16 && dtype != PKV_DTYPE_BF16)
    return fail(PKV_ERR_UNSUPPORTED, "paged_attention_fp8_block: unknown dtype %d", dtype);
  if (num_q_heads % num_kv_heads)
    return fail(PKV_ERR_INVALID_ARGUMENT, "paged_attention_fp8_block: Hq must be divisible by Hkv");
  const int32_t group = num_q_heads / num_kv_heads;
  if (group > PKV_MAX_GROUP)
    return fail(PKV_ERR_UNSUPPORTED, "paged_attention_fp8_block: G=Hq/Hkv %d (at most %d)", group, PKV_MAX_GROUP);
  if (page_size % 16)
    return fail(PKV_ERR_UNSUPPORTED, "paged_attention_fp8_block: page_size %d is not a multiple of 16", page_size);
  if (batch > kMaxRows)
    return fail(PKV_ERR_UNSUPPORTED, "paged_attention_fp8_block: batch %d (at most %d)", batch, kMaxRows);
  const int64_t tokens = (int64_t)max_pages * page_size;
  const int64_t capacity = tokens < INT32_MAX ? tokens : INT32_MAX;
  if (tokens > INT32_MAX - 256 || (capacity / kTile + 1 + kPieceCost) * batch * num_kv_heads > INT32_MAX)
    return fail(PKV_ERR_UNSUPPORTED, "paged_attention_fp8_block: the block table addresses too many tokens");
  if (!pkv::fits_grid((int64_t)batch * num_q_heads, kMergeWaves * 64))
    return fail(PKV_ERR_UNSUPPORTED, "paged_attention_fp8_block: batch * num_q_heads too large (below 2^24)");
  if (batch == 0) return pkv::ok();
  if (!q || !k_pages || !v_pages || !kv_scales || !block_table || !seq_lens || !output)
    return fail(PKV_ERR_INVALID_ARGUMENT, "paged_attention_fp8_block: null pointer");
  if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)output | (uintptr_t)workspace) & 15 ||
      (uintptr_t)kv_scales & 7)
    return fail(PKV_ERR_INVALID_ARGUMENT, "paged_attention_fp8_block: tensors must be 16-byte aligned");
  const int64_t bytes = (int64_t)batch * num_q_heads * (2 * kD);
  if (output != q && pkv::meets_rows(output, bytes, q, 1, bytes, bytes))
    return fail(PKV_ERR_INVALID_ARGUMENT, "paged_attention_fp8_block: output must be q itself, or not overlap q");
  const size_t need = workspace_bytes(batch, num_kv_heads, group);
  if (!workspace || workspace_size < need)
    return fail(PKV_ERR_WORKSPACE_TOO_SMALL, "paged_attention_fp8_block: workspace of %zu bytes, %zu needed",
                workspace_size, need);
  const int waves = pkv::compute_units() * kWaves;
  BlockArgs a{};
  a.q = (const uint8_t*)q;
  a.k_pages = (const uint8_t*)k_pages;
  a.v_pages = (const uint8_t*)v_pages;
  a.kv_scales = kv_scales;
  a.block_table = block_table;
  a.seq_lens = seq_lens;
  a.output = (uint8_t*)output;
  a.acc = (float*)workspace;
  a.ml = (f32x2*)(a.acc + 2 * (size_t)waves * group * kD);
  a.plan = (int2*)((uint8_t*)workspace + need - (size_t)batch * num_kv_heads * sizeof(int2));
  a.batch = batch;
  a.hkv = num_kv_heads;
  a.group = group;
  a.num_pages = num_pages;
  a.page_size = page_size;
  a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1;
  a.max_pages = max_pages;
  a.waves = waves;
  hipStream_t s = (hipStream_t)stream;
  const bool bf16 = dtype == PKV_DTYPE_BF16;
  if (group <= 16) bf16 ? launch<BFloat, 1>(a, s) : launch<Half, 1>(a, s);
  else bf16 ? launch<BFloat, 2>(a, s) : launch<Half, 2>(a, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? pkv::ok()
                         : fail(PKV_ERR_LAUNCH, "paged_attention_fp8_block launch: %s", hipGetErrorString(e));
}

}  // extern "C"
