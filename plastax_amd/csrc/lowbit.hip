// lowbit.hip -- level pairs as whole matrices in few bits: quantisation to
// 4-bit blocks, activations kept in 8-bit blocks with the activation's
// gradient from them, and the products of a level pair and of its backward.
// No counterpart in the reference, whose weights and activations are float32.

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/plastax_hip.h"
#include "px_common.h"
#include "px_lowbit.h"
#include "px_lowbit_gemm.h"

using plx_detail::check_launch;
using plx_detail::cu_count;
using plx_detail::fail;

namespace {

using namespace px;

constexpr int kBlock = 256;
// Workgroups of a launch at most: 2^30 lanes, past which a kernel's lanes go
// round again (a grid of 2^32 lanes leaves values unwritten without an error).
constexpr int64_t kMaxGroups = (int64_t{1} << 30) / kBlock;

__host__ __device__ constexpr int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ---------------------------------------------------------------------------
// Lines of values and their blocks: one pass each, bound by memory (8192 x 8192
// bf16 quantised 30 us, 5.7 TB/s; 4096 x 784 float32 the other way round 5 us).
// "Along" kernels: the line's values lie
// next to each other; a lane takes 8 of them, four lanes a block, so that a
// wave reads and writes whole cache lines. "Across" kernels: any strides; a
// lane takes a whole block and its neighbours the same block of the next
// lines, which coalesces where lines are next to each other (a matrix kept
// the other way round).
// ---------------------------------------------------------------------------
// Lanes beside each other along a line, for a line of `chunks` groups of 8.
inline int lanes_along(int64_t chunks) {
  int lx = 4;
  while (lx < kBlock && lx < chunks) lx *= 2;
  return lx;
}
inline unsigned groups_along(int64_t lines, int lx) {
  const int64_t g = div_up(lines, kBlock / lx);
  return static_cast<unsigned>(g < kMaxGroups ? g : kMaxGroups);
}
// The largest of 4 neighbouring lanes' values.
__device__ __forceinline__ uint32_t max4(uint32_t m) {
  uint32_t o = __shfl_xor(m, 1, 64);
  m = m > o ? m : o;
  o = __shfl_xor(m, 2, 64);
  return m > o ? m : o;
}

template <typename T>
__global__ __launch_bounds__(kBlock) void k_mx4_along(int64_t lines, int64_t n, const T* x, int64_t stride,
                                                      uint8_t* codes, uint8_t* scales, int lx) {
  const int64_t chunks = div_up(n, 128) * 16;  // a multiple of lx's quads
  const int tx = threadIdx.x & (lx - 1), ly = kBlock / lx, ty = threadIdx.x / lx;
  for (int64_t line = static_cast<int64_t>(blockIdx.x) * ly + ty; line < lines;
       line += static_cast<int64_t>(gridDim.x) * ly) {
    const T* row = x + line * stride;
    uint32_t* out = reinterpret_cast<uint32_t*>(codes) + line * chunks;
    for (int64_t c = tx; c < chunks; c += lx) {
      const int64_t left = n - c * 8;
      float v[8];
      load8<true>(row + c * 8, 1, left > 8 ? 8 : left < 0 ? 0 : static_cast<int>(left), v);
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = m > abs_bits(v[i]) ? m : abs_bits(v[i]);
      m = max4(m);
      const bool fine = m < kInfBits;
      const int e = exponent4(m);
      out[c] = fine ? codes4(v, pow2(fine ? e : 0)) : 0u;
      if ((tx & 3) == 0) scales[line * (chunks / 4) + c / 4] = static_cast<uint8_t>(fine ? e + 127 : 255);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void k_mx4_across(int64_t lines, int64_t n, const T* x, int64_t sl, int64_t se,
                                                       uint8_t* codes, uint8_t* scales) {
  const int64_t blocks = div_up(n, 128) * 4;
  const int64_t total = div_up(lines, 64) * blocks * 64;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; t < total;
       t += static_cast<int64_t>(gridDim.x) * kBlock) {
    const int64_t w = t >> 6, b = w % blocks, line = (w / blocks) * 64 + (t & 63);
    if (line >= lines) continue;
    const T* p = x + line * sl + b * 32 * se;
    const int64_t left = n - b * 32;
    float v[4][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      v[i / 8][i % 8] = i < left ? to_f32(p[i * se]) : 0.0f;
      const uint32_t a = abs_bits(v[i / 8][i % 8]);
      m = m > a ? m : a;
    }
    const bool fine = m < kInfBits;
    const int e = exponent4(m);
    const float scale = pow2(fine ? e : 0);
    uint4 c = make_uint4(0, 0, 0, 0);
    if (fine) c = make_uint4(codes4(v[0], scale), codes4(v[1], scale), codes4(v[2], scale), codes4(v[3], scale));
    reinterpret_cast<uint4*>(codes)[line * blocks + b] = c;
    scales[line * blocks + b] = static_cast<uint8_t>(fine ? e + 127 : 255);
  }
}

// BITS 4 or 8: the values that codes stand for, lines of n next to each other.
// A lane writes 16 bytes, 4 values of float32 or 8 of the others, so that a
// wave's store is whole lines (8192 x 8192 as float32 50 us; with 32 bytes a
// lane in two stores 57).
template <int BITS, typename T>
__global__ __launch_bounds__(kBlock) void k_mx_values(int64_t lines, int64_t n, const uint8_t* codes,
                                                      const uint8_t* scales, T* out, int lx) {
  constexpr int W = 16 / sizeof(T);
  typedef T tw __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  const int64_t blocks = BITS == 4 ? div_up(n, 128) * 4 : div_up(n, 32), chunks = div_up(n, W);
  const int tx = threadIdx.x & (lx - 1), ly = kBlock / lx, ty = threadIdx.x / lx;
  for (int64_t line = static_cast<int64_t>(blockIdx.x) * ly + ty; line < lines;
       line += static_cast<int64_t>(gridDim.x) * ly) {
    for (int64_t c = tx; c < chunks; c += lx) {
      const float scale = scale_value(scales[line * blocks + c * W / 32]);
      const int64_t at = line * blocks * (32 / W) + c;
      float v[8];
      if (BITS == 4)
        values4(W == 8 ? reinterpret_cast<const uint32_t*>(codes)[at] : reinterpret_cast<const uint16_t*>(codes)[at],
                scale, v);
      else
        values8(W == 8 ? reinterpret_cast<const uint2*>(codes)[at]
                       : make_uint2(reinterpret_cast<const uint32_t*>(codes)[at], 0),
                scale, v);
      T* p = out + line * n + c * W;
      const int64_t left = n - c * W;
      if (left >= W) {
        tw r;
#pragma unroll
        for (int i = 0; i < W; ++i) r[i] = from_f32<T>(v[i]);
        __builtin_nontemporal_store(r, reinterpret_cast<tw*>(p));
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
          if (i < left) p[i] = from_f32<T>(v[i]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Activations. y = fn(h) from h itself; fn'(q) from what was kept. Bound by
// memory as long as a value costs below some 30 instructions: silu of 8192 x
// 8192 bf16 72 us on average and its gradient 74 (62 and 64 at least), 338 MB
// each, 4.6 TB/s (5.4).
// ---------------------------------------------------------------------------
// exp(-a), a >= 0, to 2 steps: the hardware's 2^f (1 step) of the fraction of
// -a log2(e), whose rounding error goes on as a factor 1 + r ln 2, and ldexp,
// which rounds once below the normal numbers.
__device__ __forceinline__ float exp_neg(float a) {
  a = a > 150.0f ? 150.0f : a;  // (a NaN stays)
  const float hi = a * -1.44269502162933349609375f;
  float lo = __builtin_fmaf(a, -1.44269502162933349609375f, -hi);
  lo = __builtin_fmaf(a, -1.925963033500011e-8f, lo);
  const float n = __builtin_rintf(hi);
  const float p = __builtin_amdgcn_exp2f(hi - n);
  return __builtin_ldexpf(__builtin_fmaf(p * lo, 0.693147182464599609375f, p), static_cast<int>(n));
}
// 1 / d, 1 <= d <= 2: the hardware's (1 step) and one Newton step.
__device__ __forceinline__ float inverse(float d) {
  const float r = __builtin_amdgcn_rcpf(d);
  return __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
}

// By exp(-|h|), so that nothing overflows and the tails keep their values:
// sigmoid = 1 / (1 + t) or t / (1 + t), tanh = (1 - u) / (1 + u) with
// u = exp(-2|h|), and below 0.625 Cephes' polynomial, which has no
// cancellation.
template <int FN>
__device__ __forceinline__ float act(float h) {
  if (FN == PLX_LB_RELU) return h <= 0.0f ? 0.0f : h;  // (a NaN passes)
  const float a = fabsf(h);
  const float t = exp_neg(FN == PLX_LB_TANH ? 2.0f * a : a), r = inverse(1.0f + t);
  if (FN == PLX_LB_TANH) {
    const float y = h * h;
    float p = -5.70498872745e-3f;
    p = __builtin_fmaf(p, y, 2.06390887954e-2f);
    p = __builtin_fmaf(p, y, -5.37397155531e-2f);
    p = __builtin_fmaf(p, y, 1.33314422036e-1f);
    p = __builtin_fmaf(p, y, -3.33332819422e-1f);
    return a < 0.625f ? __builtin_fmaf(p * y, h, h) : __builtin_copysignf((1.0f - t) * r, h);
  }
  const float s = h < 0.0f ? t * r : r;
  return FN == PLX_LB_SIGMOID ? s : h * s;
}
// tanh' = 4u / (1 + u)^2, sigmoid' = t / (1 + t)^2 and
// silu' = sigmoid(q) + q sigmoid'(q).
template <int FN>
__device__ __forceinline__ float act_grad(float q) {
  const float a = fabsf(q);
  const float t = exp_neg(FN == PLX_LB_TANH ? 2.0f * a : a), r = inverse(1.0f + t), d = t * r * r;
  if (FN == PLX_LB_TANH) return 4.0f * d;
  if (FN == PLX_LB_SIGMOID) return d;
  return (q >= 0.0f ? r : t * r) + (t == 0.0f ? 0.0f : q * d);  // (an infinite q has the slope 0 or 1)
}
// The slopes at 8 kept values. The rectifier's goes by the codes: 1 unless the
// sign is set or all else is zero, so 1 at a kept infinity or NaN (0x7f), whose
// result the forward passed on, and 0 at a negative infinity (0xff).
template <int FN>
__device__ __forceinline__ void act_grads8(uint2 c, float scale, float d[8]) {
  if (FN == PLX_LB_RELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = i < 4 ? c.x : c.y;
      const uint32_t set = (((w & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) & ~w & 0x80808080u) >> 7;  // (1 in those bytes)
      d[i] = static_cast<float>(set >> (i % 4 * 8) & 0xFFu);
    }
    return;
  }
  values8(c, scale, d);
#pragma unroll
  for (int i = 0; i < 8; ++i) d[i] = act_grad<FN>(d[i]);
}

template <int FN, typename T>
__global__ __launch_bounds__(kBlock) void k_act_along(int64_t lines, int64_t n, const T* h, int64_t sh, T* y,
                                                      int64_t sy, uint8_t* codes, uint8_t* scales, int lx) {
  const int64_t chunks = div_up(n, 32) * 4;
  const int tx = threadIdx.x & (lx - 1), ly = kBlock / lx, ty = threadIdx.x / lx;
  for (int64_t line = static_cast<int64_t>(blockIdx.x) * ly + ty; line < lines;
       line += static_cast<int64_t>(gridDim.x) * ly) {
    for (int64_t c = tx; c < chunks; c += lx) {
      const int64_t left64 = n - c * 8;
      const int left = left64 > 8 ? 8 : left64 < 0 ? 0 : static_cast<int>(left64);
      float v[8], f[8];
      load8<true>(h + line * sh + c * 8, 1, left, v);
      uint32_t m = largest8<false>(0, v);
      const bool fine = m < kInfBits;
      if (!fine) m = largest8<true>(0, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = act<FN>(v[i]);
      if (y) store8<true>(y + line * sy + c * 8, left, f);
      const int e = exponent8(max4(m));
      uint2 k = codes8(v, pow2(-e));
      if (!fine) k = mark8(k, v);
      reinterpret_cast<uint2*>(codes)[line * chunks + c] = k;
      if ((tx & 3) == 0) scales[line * (chunks / 4) + c / 4] = static_cast<uint8_t>(e + 127);
    }
  }
}

template <int FN, typename T>
__global__ __launch_bounds__(kBlock) void k_act_across(int64_t lines, int64_t n, const T* h, int64_t sl, int64_t se,
                                                       T* y, int64_t yl, int64_t ye, uint8_t* codes, uint8_t* scales) {
  const int64_t blocks = div_up(n, 32);
  const int64_t total = div_up(lines, 64) * blocks * 64;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; t < total;
       t += static_cast<int64_t>(gridDim.x) * kBlock) {
    const int64_t w = t >> 6, b = w % blocks, line = (w / blocks) * 64 + (t & 63);
    if (line >= lines) continue;
    const T* p = h + line * sl + b * 32 * se;
    T* o = y + line * yl + b * 32 * ye;
    const int64_t left = n - b * 32;
    float v[4][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {  // (loads without a condition, 32 in flight)
      const float at = to_f32(p[(i < left ? i : left - 1) * se]);
      v[i / 8][i % 8] = i < left ? at : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) m = largest8<false>(m, v[i]);
    const bool fine = m < kInfBits;
    if (!fine) {
      m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) m = largest8<true>(m, v[i]);
    }
    const int e = exponent8(m);
    uint2 k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = codes8(v[i], pow2(-e));
    if (!fine) {
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = mark8(k[i], v[i]);
    }
    uint2* c = reinterpret_cast<uint2*>(codes) + (line * blocks + b) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = k[i];
    scales[line * blocks + b] = static_cast<uint8_t>(e + 127);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (y && i < left) o[i * ye] = from_f32<T>(act<FN>(v[i / 8][i % 8]));
  }
}

template <int FN, typename T>
__global__ __launch_bounds__(kBlock) void k_grad_along(int64_t lines, int64_t n, const T* dy, int64_t sy,
                                                       const uint8_t* codes, const uint8_t* scales, T* dh, int64_t sh,
                                                       int lx) {
  const int64_t kept = div_up(n, 32) * 4, chunks = div_up(n, 8);
  const int tx = threadIdx.x & (lx - 1), ly = kBlock / lx, ty = threadIdx.x / lx;
  for (int64_t line = static_cast<int64_t>(blockIdx.x) * ly + ty; line < lines;
       line += static_cast<int64_t>(gridDim.x) * ly) {
    for (int64_t c = tx; c < chunks; c += lx) {
      const int64_t left64 = n - c * 8;
      const int left = left64 > 8 ? 8 : static_cast<int>(left64);
      float v[8], d[8];
      load8<true>(dy + line * sy + c * 8, 1, left, v);
      act_grads8<FN>(reinterpret_cast<const uint2*>(codes)[line * kept + c],
                     scale_value(scales[line * (kept / 4) + c / 4]), d);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= d[i];
      store8<true>(dh + line * sh + c * 8, left, v);
    }
  }
}

template <int FN, typename T>
__global__ __launch_bounds__(kBlock) void k_grad_across(int64_t lines, int64_t n, const T* dy, int64_t sl, int64_t se,
                                                        const uint8_t* codes, const uint8_t* scales, T* dh, int64_t hl,
                                                        int64_t he) {
  const int64_t blocks = div_up(n, 32);
  const int64_t total = div_up(lines, 64) * blocks * 64;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; t < total;
       t += static_cast<int64_t>(gridDim.x) * kBlock) {
    const int64_t w = t >> 6, b = w % blocks, line = (w / blocks) * 64 + (t & 63);
    if (line >= lines) continue;
    const uint2* c = reinterpret_cast<const uint2*>(codes) + (line * blocks + b) * 4;
    const float scale = scale_value(scales[line * blocks + b]);
    const int64_t left = n - b * 32;
    const T* p = dy + line * sl + b * 32 * se;
    T* o = dh + line * hl + b * 32 * he;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float d[8];
      act_grads8<FN>(c[i], scale, d);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i * 8 + j < left) o[(i * 8 + j) * he] = from_f32<T>(to_f32(p[(i * 8 + j) * se]) * d[j]);
    }
  }
}

// ---------------------------------------------------------------------------
// Products: out[m][n] = sum over k of a(m, k) b(n, k), a from memory at any
// strides, b from codes:
//   kW    4-bit weights, lines n, blocks along k      (y = x w^T)
//   kWT   4-bit weights, lines k, blocks along n      (dx = g w)
//   kX    8-bit values, lines k, blocks along n       (dw = g^T x, token-major)
//   kXT   8-bit values, lines n, blocks along k       (the same, unit-major)
// Every b is exact in bf16, and a is split into the bf16 pieces that hold it
// exactly (pieces8), so every product is exact and only the float32 sums of
// the matrix instruction round. Pieces of different units have sums of their own,
// joined at the end.
// ---------------------------------------------------------------------------
enum { kW = 0, kWT = 1, kX = 2, kXT = 3 };

struct GemmArgs {
  const void* a;
  int64_t sm, sk;
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t blocks;  // blocks of a line of codes
  void* out;       // [m][n]
  float* part;     // [splits][m][n], where splits > 1
  int M, N, K, kper, tiles_n;
};

__device__ __forceinline__ void unit_pieces(Unit<__bf16>::type v, uint4 out[1]) {
  out[0] = __builtin_bit_cast(uint4, v);
}
template <typename T8, int P>
__device__ __forceinline__ void unit_pieces(T8 v, uint4 (&out)[P]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32(v[i]);
  pieces8<P>(f, out);
}

// The sums of a tile of TS x TS, a wave's quarter of its group's in acc (with b's
// rows as the matrix instruction's first operand a lane holds four consecutive
// n of one m): the groups' sums are added in order through LDS.
template <int TS, int KS, typename OT>
__device__ __forceinline__ void tile_store(const f32x4 (&acc)[TS / 32][TS / 32], void* lds, int group, int wm, int wn, int m0,
                                           int n0, int M, int N, OT* out, float* parts) {
  const int tid = threadIdx.x, l15 = tid & 15, q = (tid & 63) >> 4;
  float* part = gridDim.y > 1 ? parts + static_cast<int64_t>(blockIdx.y) * M * N : nullptr;
  auto store = [&](int m, int n, f32x4 v) {
    if (m >= M || n >= N) return;
    const int64_t at = static_cast<int64_t>(m) * N + n;
    if (part)
      store4(part + at, N - n, v);
    else
      store4(out + at, N - n, v);
  };
  constexpr int F = TS / 32, kRow = TS / 4, kTileSums = TS * kRow;
  if (KS == 1) {
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int j = 0; j < F; ++j) store(m0 + wm + j * 16 + l15, n0 + wn + i * 16 + q * 4, acc[i][j]);
    return;
  }
  __syncthreads();
  f32x4* sums = static_cast<f32x4*>(lds);  // [group][m][TS / 4 of n], four n at c ^ (m & (TS / 4 - 1))
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) {
      const int m = wm + j * 16 + l15, c = (wn >> 2) + i * 4 + q;
      sums[group * kTileSums + m * kRow + (c ^ (m & (kRow - 1)))] = acc[i][j];
    }
  __syncthreads();
  for (int t = tid; t < kTileSums; t += 256 * KS) {
    const int m = t / kRow, c = t % kRow;
    f32x4 v = sums[m * kRow + (c ^ (m & (kRow - 1)))];
#pragma unroll
    for (int k = 1; k < KS; ++k) v += sums[k * kTileSums + m * kRow + (c ^ (m & (kRow - 1)))];
    store(m0 + m, n0 + c * 4, v);
  }
}

// TS x TS (64 or 32) of the output by KS groups of four waves, k in steps
// of 64 KS, a group's share 64 of them: both operands go through registers
// (as bf16 pieces) into LDS, the next step's loads in flight during this
// step's matrix instructions, and the groups' sums are added in order at the
// end. Threads load 8 consecutive values of a line. A line of k ("along") is
// a row of LDS, 8 chunks of 16 bytes with chunk c of row r at c ^ (r & 7), so
// that the rows of a fragment's read fall on different banks; lines of m or n
// ("across") are rows too, pairs of chunks at p ^ (k & 3) (k & 1 of 32), and their
// fragments are read transposed. What bounds it is that a step's phases follow
// each other: bf16 256 x 4096 x 4096 takes 19 us, 36 % of a CU's cycles
// conversions and addresses, 33 % LDS, 16 % matrix instructions.
// Four waves a SIMD at least: float32's sums for each unit would leave three
// (1 x 4096 x 4096's weight gradient 22.4 us, so 19.0).
template <typename T, int KIND, typename OT, int TS, int KS, bool AA>
__global__ __launch_bounds__(256 * KS, 4) void k_mx_gemm(GemmArgs g) {
  constexpr int P = Pieces<T>::n, S = Pieces<T>::sums;
  constexpr bool BA = KIND == kWT || KIND == kX;
  constexpr int BITS = KIND == kW || KIND == kWT ? 4 : 8;
  constexpr int F = TS / 32, kLine = TS / 8;                // (fragments a wave and side; chunks of a line across)
  constexpr int kStep = 64 * KS, kSub = TS * 8, kU = TS / 32;  // (16-byte chunks of TS x 64 values; units a thread)
  constexpr int kUints = (P + 1) * KS * kSub, kSums = KS * TS * TS / 4;
  // Two buffers where they fit: a step's stores to LDS then go beside the
  // matrix instructions of the step before, with one barrier for both (bf16
  // 512 x 4096 x 4096 44 -> 35 us). Not for one group of waves, where several
  // workgroups of a CU do that already (float32 8192 x 512 x 512 25 -> 31).
  constexpr int kBufs = KS == 4 && 2 * kUints * 16 <= 128 * 1024 ? 2 : 1;
  __shared__ uint4 lds[KS > 1 && kBufs * kUints < kSums ? kSums : kBufs * kUints];
  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = wave >> 2;
  const int m0 = (blockIdx.x / g.tiles_n) * TS, n0 = (blockIdx.x % g.tiles_n) * TS;
  const int kbeg = blockIdx.y * g.kper, kend = kbeg + g.kper < g.K ? kbeg + g.kper : g.K;
  const T* a = static_cast<const T*>(g.a);
  typedef typename Unit<T>::type unit;

  struct {
    unit a[kU];
    uint2 b[kU];
    uint32_t s[kU];
  } r;
  // The line and the chunk of this thread's i-th unit, and its place in LDS.
  auto place = [&](bool across, int i, int* line, int* chunk) {
    const int u = tid + 256 * KS * i;
    if (across) {
      *line = u / kLine, *chunk = u % kLine;
      const int c = *chunk, k = *line;
      return (k >> 6) * kSub + (k & 63) * kLine + ((((c >> 1) ^ (k & (kLine / 2 - 1))) << 1) | (c & 1));
    }
    *line = u / (8 * KS), *chunk = u % (8 * KS);
    return (*chunk >> 3) * kSub + *line * 8 + ((*chunk & 7) ^ (*line & 7));
  };
  auto load = [&](int k0) {
    if (k0 >= kend) return;
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      int line, chunk;
      place(AA, i, &line, &chunk);
      const int m = m0 + (AA ? chunk * 8 : line), k = k0 + (AA ? line : chunk * 8);
      const int room = AA ? g.M - m : kend - k;
      const bool in = AA ? k < kend : m < g.M;
      r.a[i] = load_unit(a + m * g.sm + k * g.sk, AA ? g.sm : g.sk, in ? room : 0);
    }
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      int line, chunk;
      place(BA, i, &line, &chunk);
      const int64_t l = BA ? k0 + line : n0 + line;
      const int pos = (BA ? n0 : k0) + chunk * 8;
      r.b[i] = make_uint2(0, 0), r.s[i] = 127;
      if (l < (BA ? kend : g.N) && pos < (BA ? g.N : kend)) {
        const int64_t at = l * g.blocks * 4 + pos / 8;
        if (BITS == 4)
          r.b[i].x = reinterpret_cast<const uint32_t*>(g.codes)[at];
        else
          r.b[i] = reinterpret_cast<const uint2*>(g.codes)[at];
        r.s[i] = g.scales[l * g.blocks + pos / 32];
      }
    }
  };
  auto put = [&](int buf, int k0) {  // (k0: the loads' first k)
    uint4* la = lds + buf * kUints;
    uint4* lb = la + P * KS * kSub;
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      int line, chunk;
      const int at = place(AA, i, &line, &chunk);
      uint4 p[P];
      unit_pieces(r.a[i], p);
#pragma unroll
      for (int j = 0; j < P; ++j) la[j * KS * kSub + at] = p[j];
    }
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      int line, chunk;
      const int at = place(BA, i, &line, &chunk);
      const float scale = scale_value(r.s[i]);
      if (KIND == kXT) r.b[i] = first_codes8(r.b[i], kend - k0 - chunk * 8);
      lb[at] = BITS == 4 ? bf16_of4(r.b[i].x, scale) : bf16_of8(r.b[i], scale);
    }
  };
  auto frag = [&](const uint4* t, bool across, int row, int s) {
    if (across) {
      typedef __attribute__((address_space(3))) s16x4* p4;
      const int k = s * 32 + q * 8 + (l15 >> 2);
      const char* p = reinterpret_cast<const char*>(t) + k * kLine * 16 +
                      (((row >> 4) ^ ((l15 >> 2) & (kLine / 2 - 1))) << 5) + (l15 & 3) * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(p + 4 * kLine * 16));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    const int r = row + l15;
    return as_bf16x8(t[r * 8 + ((s * 4 + q) ^ (r & 7))]);
  };

  f32x4 acc[F][F][S] = {};
  const int wn = (wave & 1) * (TS / 2), wm = ((wave >> 1) & 1) * (TS / 2);
  auto compute = [&](int buf, int k0) {
    const uint4* la = lds + buf * kUints;
    const uint4* lb = la + P * KS * kSub;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (KS == 1 && k0 + s * 32 >= kend) break;  // (zeros from there on)
      bf16x8 fb[F], fa[F][P];
#pragma unroll
      for (int i = 0; i < F; ++i) {
        fb[i] = frag(lb + group * kSub, BA, wn + i * 16, s);
#pragma unroll
        for (int p = 0; p < P; ++p) fa[i][p] = frag(la + (p * KS + group) * kSub, AA, wm + i * 16, s);
      }
#pragma unroll
      for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
          for (int j = 0; j < F; ++j)
            acc[i][j][p % S] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[i], fa[j][p], acc[i][j][p % S], 0, 0, 0);
    }
  };
  load(kbeg);
  if (kBufs == 2) {
    if (kbeg < kend) put(0, kbeg);
    load(kbeg + kStep);
    int buf = 0;
    for (int k0 = kbeg; k0 < kend; k0 += kStep) {
      __syncthreads();
      if (k0 + kStep < kend) put(buf ^ 1, k0 + kStep);
      load(k0 + 2 * kStep);
      compute(buf, k0);
      buf ^= 1;
    }
  } else {
    for (int k0 = kbeg; k0 < kend; k0 += kStep) {
      __syncthreads();
      put(0, k0);
      __syncthreads();
      load(k0 + kStep);
      compute(0, k0);
    }
  }
  f32x4 sums[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) sums[i][j] = join_sums(acc[i][j]);
  tile_store<TS, KS, OT>(sums, lds, group, wm, wn, m0, n0, g.M, g.N, static_cast<OT*>(g.out), g.part);
}

// out = the partial sums of the k ranges, in their order.
template <typename OT>
__global__ __launch_bounds__(kBlock) void k_mx_join(int64_t n, int splits, const float* part, OT* out) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kBlock) {
    float s = part[i];
    for (int k = 1; k < splits; ++k) s += part[k * n + i];
    out[i] = from_f32<OT>(s);
  }
}

// y = x w^T of up to 16 tokens: 16 rows of w by the waves of a workgroup, each
// with every kFewWaves-th group of 4 blocks; a lane takes a block and its 32
// inputs of one token, straight into the matrix instruction, and the waves'
// sums are added in order. Weights are read once, so what counts is how many
// loads are in flight: one token through 4096 x 4096 takes 5.6 us (8.9 MB),
// with 8 waves 8.3; small tiles take 10.5 and the sum of their ranges 3.7 (in a
// captured graph 5.1, in float32 8.4).
constexpr int kFew = 16;
template <bool ALONG>
constexpr int kFewWaves = ALONG ? 16 : 8;
// The unit of p[0..left), left < 8, of a row of 8 or more: the row's last
// eight values moved down.
template <typename T>
__device__ __forceinline__ typename Unit<T>::type load_tail(const T* p, int left) {
  typename Unit<T>::type r = load_unit(p - (8 - left), 1, 8), z = {};
  const int by = 8 - left;
  if (by & 4) r = __builtin_shufflevector(r, z, 4, 5, 6, 7, 8, 8, 8, 8);
  if (by & 2) r = __builtin_shufflevector(r, z, 2, 3, 4, 5, 6, 7, 8, 8);
  if (by & 1) r = __builtin_shufflevector(r, z, 1, 2, 3, 4, 5, 6, 7, 8);
  return r;
}
// ALONG: inputs next to each other, 8 of them or more.
template <typename T, bool ALONG>
__global__ __launch_bounds__(64 * kFewWaves<ALONG>) void k_mx_few(GemmArgs g) {
  constexpr int W = kFewWaves<ALONG>, P = Pieces<T>::n, S = Pieces<T>::sums, kAhead = ALONG ? 2 : 1;
  __shared__ f32x4 sums[W][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, q = lane >> 4;
  const int n = blockIdx.x * 16 + l15;
  const T* x = static_cast<const T*>(g.a) + l15 * g.sm;
  const uint4* codes = reinterpret_cast<const uint4*>(g.codes) + n * g.blocks;
  const uint8_t* scales = g.scales + n * g.blocks;
  const int blocks = static_cast<int>(div_up(g.K, 32));  // (what is behind a line's end counts for nothing)
  f32x4 of[S] = {};
  for (int b0 = wave * 4 + q; b0 - q < blocks; b0 += kAhead * W * 4) {
    uint4 c[kAhead];
    uint32_t s[kAhead];
    typename Unit<T>::type v[kAhead][4];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int b = b0 + i * W * 4;
      c[i] = make_uint4(0, 0, 0, 0), s[i] = 127;
      if (b < blocks && n < g.N) c[i] = codes[b], s[i] = scales[b];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t k = int64_t{b} * 32 + j * 8;
        const int64_t left = l15 < g.M ? g.K - k : 0;
        if (ALONG) {
          v[i][j] = typename Unit<T>::type{};
          if (left >= 8)
            v[i][j] = load_unit(x + k, 1, 8);
          else if (left > 0)
            v[i][j] = load_tail(x + k, static_cast<int>(left));
        } else {
          v[i][j] = load_unit(x + k * g.sk, g.sk, left > 8 ? 8 : static_cast<int>(left));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float scale = scale_value(s[i]);
      const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint4 p[P];
        unit_pieces(v[i][j], p);
        const bf16x8 fw = as_bf16x8(bf16_of4(w[j], scale));
#pragma unroll
        for (int h = P - 1; h >= 0; --h)
          of[h % S] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw, as_bf16x8(p[h]), of[h % S], 0, 0, 0);
      }
    }
  }
  f32x4 acc = join_sums(of);
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave != 0 || l15 >= g.M) return;
#pragma unroll
  for (int w = 1; w < W; ++w) acc += sums[w][lane];
  const int at = blockIdx.x * 16 + q * 4;
  if (at < g.N) store4(static_cast<T*>(g.out) + static_cast<int64_t>(l15) * g.N + at, g.N - at, acc);
}

// 4-bit times 4-bit blocks: the scaled matrix instruction takes 128 k of both
// operands as they are kept, a block and its scale byte per lane (256 x 4096 x
// 4096 9.6 us; with fragments straight from memory 24). Tiles, groups
// and LDS as in k_mx_gemm, a chunk of 16 bytes being one block here: a step is
// 256 k a group.
template <typename OT, int TS, int KS>
__global__ __launch_bounds__(256 * KS) void k_mx4_gemm(int M, int N, int K, int blocks, const uint8_t* xc,
                                                       const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, OT* out,
                                                       float* parts, int tiles_n, int per) {
  constexpr int F = TS / 32, kSub = TS * 8, kStep = 8 * KS;  // blocks of a step
  constexpr int kUints = 2 * KS * kSub, kSums = KS * TS * TS / 4;
  constexpr int kBufs = KS == 4 ? 2 : 1;
  __shared__ uint4 lds[KS > 1 && kBufs * kUints < kSums ? kSums : kBufs * kUints];
  __shared__ uint8_t lss[kBufs * kUints];
  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = wave >> 2;
  const int m0 = (blockIdx.x / tiles_n) * TS, n0 = (blockIdx.x % tiles_n) * TS;
  const int used = (K + 31) / 32;  // blocks that hold values
  const int beg = blockIdx.y * per, end = beg + per < used ? beg + per : used;
  struct {
    uint4 c[2 * F];
    uint32_t s[2 * F];
  } r;
  auto load = [&](int b0) {
    if (b0 >= end) return;
#pragma unroll
    for (int i = 0; i < 2 * F; ++i) {  // x's, then w's
      const int u = tid + 256 * KS * (i % F), line = u / kStep, b = b0 + u % kStep;
      const int row = (i < F ? m0 : n0) + line;
      r.c[i] = make_uint4(0, 0, 0, 0), r.s[i] = 127;
      if (row < (i < F ? M : N) && b < end) {
        const int64_t at = static_cast<int64_t>(row) * blocks + b;
        r.c[i] = reinterpret_cast<const uint4*>(i < F ? xc : wc)[at];
        r.s[i] = (i < F ? xs : ws)[at];
      }
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int i = 0; i < 2 * F; ++i) {
      const int u = tid + 256 * KS * (i % F), line = u / kStep, b = u % kStep;
      const int at = buf * kUints + ((i < F ? 0 : KS) + (b >> 3)) * kSub + line * 8 + ((b & 7) ^ (line & 7));
      lds[at] = r.c[i];
      lss[at] = static_cast<uint8_t>(r.s[i]);
    }
  };
  f32x4 acc[F][F] = {};
  const int wn = (wave & 1) * (TS / 2), wm = ((wave >> 1) & 1) * (TS / 2);
  auto compute = [&](int buf) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x8 fx[F], fw[F];
      int sx[F], sw[F];
#pragma unroll
      for (int i = 0; i < F; ++i) {
        const int rm = wm + i * 16 + l15, rn = wn + i * 16 + l15;
        const int am = buf * kUints + group * kSub + rm * 8 + ((h * 4 + q) ^ (rm & 7));
        const int an = buf * kUints + (KS + group) * kSub + rn * 8 + ((h * 4 + q) ^ (rn & 7));
        fx[i] = as_i32x8(as_bf16x8(lds[am])), sx[i] = lss[am];
        fw[i] = as_i32x8(as_bf16x8(lds[an])), sw[i] = lss[an];
      }
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
          acc[i][j] =
              __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[i], fx[j], acc[i][j], 4, 4, 0, sw[i], 0, sx[j]);
    }
  };
  load(beg);
  if (kBufs == 2) {
    if (beg < end) put(0);
    load(beg + kStep);
    int buf = 0;
    for (int b0 = beg; b0 < end; b0 += kStep) {
      __syncthreads();
      if (b0 + kStep < end) put(buf ^ 1);
      load(b0 + 2 * kStep);
      compute(buf);
      buf ^= 1;
    }
  } else {
    for (int b0 = beg; b0 < end; b0 += kStep) {
      __syncthreads();
      put(0);
      __syncthreads();
      load(b0 + kStep);
      compute(0);
    }
  }
  tile_store<TS, KS, OT>(acc, lds, group, wm, wn, m0, n0, M, N, out, parts);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr int64_t kMaxDim = int64_t{1} << 30;
constexpr int64_t kBigLine = int64_t{1} << 22;  // elements of a large product's lines: 256 of them stay below 2^32 bytes

inline bool dims_fit(int64_t a, int64_t b) { return a >= 0 && b >= 0 && a <= kMaxDim && b <= kMaxDim; }
constexpr int64_t kMaxUnits = int64_t{1} << 24;  // of a level in products: a launch's tiles stay below 2^30 lanes
inline bool product_fits(int64_t tokens, int64_t inputs, int64_t outputs) {
  return tokens >= 0 && inputs >= 0 && outputs >= 0 && tokens <= kMaxDim && inputs <= kMaxUnits && outputs <= kMaxUnits;
}
inline bool known(int dtype) { return dtype == PLX_LB_F32 || dtype == PLX_LB_BF16 || dtype == PLX_LB_F16; }

template <typename F>
void with_type(int dtype, F f) {
  if (dtype == PLX_LB_F32)
    f(static_cast<float*>(nullptr));
  else if (dtype == PLX_LB_BF16)
    f(static_cast<__bf16*>(nullptr));
  else
    f(static_cast<_Float16*>(nullptr));
}
template <typename F>
void with_fn(int fn, F f) {
  if (fn == PLX_LB_RELU)
    f(std::integral_constant<int, PLX_LB_RELU>{});
  else if (fn == PLX_LB_TANH)
    f(std::integral_constant<int, PLX_LB_TANH>{});
  else if (fn == PLX_LB_SIGMOID)
    f(std::integral_constant<int, PLX_LB_SIGMOID>{});
  else
    f(std::integral_constant<int, PLX_LB_SILU>{});
}
#define PLX_TYPE(p) typename std::remove_pointer<decltype(p)>::type

inline unsigned groups_across(int64_t lines, int64_t blocks) {
  const int64_t g = div_up(div_up(lines, 64) * blocks * 64, kBlock);
  return static_cast<unsigned>(g < kMaxGroups ? g : kMaxGroups);
}

// A large product: 256 x 256 tiles have enough rows, columns and k (counted
// over a's pieces), and the operands' way through memory pays. Large against
// small tiles, us, from the least to the largest of the four products: bf16
// 8.6e9 (2048 cubed) 46 to 49 and 40 to 47, 10.1e9 (8192 x 4096 x 300) 39 to 67
// and 59 to 116, 17.2e9 56 to 61 and 63 to 80. float32, where small tiles split
// a in registers, 12.9e9 (1024 x 2048 x 2048, 32 tiles) 53 to 55 and 44 to 47,
// with a tile for every CU (4096 x 4096 of 256 tokens) 41 to 42 and 46, 14.7e9
// 59 to 60 and 52 to 68. In 4 bits 17.2e9 take 26 and 24, 25.2e9 31 and 34.
constexpr double kBigLeast = 9e9, kBigPieces = 14e9, kBig4Least = 25e9;
// (Beyond 2^30 lanes of a launch, products go in small tiles, cut into launches.)
inline bool large(int64_t m, int64_t n, int64_t k, double least) {
  return m >= 256 && n >= 256 && k >= 256 && static_cast<double>(m) * n * k >= least &&
         div_up(m, kBig) * div_up(n, kBig) <= int64_t{1} << 21 && n * k <= int64_t{1} << 34;
}

// How a product in small tiles runs: tiles of ts x ts, ks groups of waves in a
// workgroup, each with `share` of k in a step, and ranges of k over workgroups.
// By measurement (us in a captured graph, bf16 and float32, which has taken up
// to 5 % more on both sides since its pieces have units of their own):
//   ts 32 where tiles of 64 leave half the CUs idle and steps are few (256 x
//   777 of 1003 k: 5.6 and 7.5, with 64 8.2 and 13.0) or tiles very few (64 x
//   1024 of 4096 k: 8.1 and 10.1, 10.0 and 15.2), but not in between (256 x
//   1024 of 4096 k: 12.1 and 21.1, 12.1 and 18.8);
//   ks 4 until tiles fill the CUs four times (2048 x 512 of 2048 k: 14.2 and
//   30.6, with 1 28.7 and 45.7), from there on 1 (8192 x 512 of 512 k: 15.2 and
//   25.3, with 4 20.7 and 35.0).
struct Tiles {
  int ts, ks, splits, kper;
};
Tiles tiles_of(int64_t m, int64_t n, int64_t k, int64_t share) {
  Tiles t{};
  const int64_t wide = div_up(m, 64) * div_up(n, 64);
  t.ts = 2 * wide <= cu_count() && (k <= 16 * share || 8 * wide <= cu_count()) ? 32 : 64;
  const int64_t tiles = div_up(m, t.ts) * div_up(n, t.ts);
  t.ks = tiles >= 4 * cu_count() || k <= share ? 1 : 4;
  const int64_t steps = div_up(k, share * t.ks);
  int64_t s = cu_count() / (tiles > 0 ? tiles : 1);
  s = s < steps / 4 ? s : steps / 4;
  s = s < 1 ? 1 : s;
  t.kper = static_cast<int>(div_up(steps, s) * share * t.ks);
  t.splits = steps > 0 ? static_cast<int>(div_up(k, t.kper)) : 1;
  return t;
}

template <typename F>
void with_tiles(const Tiles& t, F f) {
  using std::integral_constant;
  if (t.ts == 64 && t.ks == 4)
    f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else if (t.ts == 64)
    f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (t.ks == 4)
    f(integral_constant<int, 32>{}, integral_constant<int, 4>{});
  else
    f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
}

// m, n, k and the kind of b of PLX_LB_* products.
struct Shape {
  int64_t m, n, k;
};
inline Shape shape_of(int kind, int64_t tokens, int64_t inputs, int64_t outputs) {
  if (kind == PLX_LB_PRODUCT) return {tokens, outputs, inputs};
  if (kind == PLX_LB_PRODUCT_GRAD) return {tokens, inputs, outputs};
  return {outputs, inputs, tokens};
}

constexpr int64_t round_up(int64_t a, int64_t b) { return div_up(a, b) * b; }

// How a product runs. `big`: through bf16 operands in memory (k_big_gemm); a
// itself where it is one already.
struct Plan {
  bool big;
  int splits;
  bool across, direct;  // a in lines of m; as it is
  int64_t kp, mp;       // padded k, and lines of m
  int64_t bytes_w, bytes_u, bytes;
};

// Workgroups that a large product should fill: one per CU, each with 8 steps
// or more, `each` of them from one of its range.
int big_splits(int64_t m, int64_t n, int64_t steps, int64_t each) {
  const int64_t tiles = div_up(m, kBig) * div_up(n, kBig);
  int64_t s = cu_count() / (tiles > 0 ? tiles : 1);
  s = s < steps * each / 8 ? s : steps * each / 8;
  if (s < 2) return 1;
  return static_cast<int>(div_up(steps, div_up(steps, s)));  // (no range is empty)
}

Plan plan_of(int kind, const Shape& s, int dtype, const void* a, int64_t sm, int64_t sk) {
  Plan p{};
  const int pieces = dtype == PLX_LB_F32 ? 3 : dtype == PLX_LB_F16 ? 2 : 1;
  const bool full = 2 * div_up(s.m, kBig) * div_up(s.n, kBig) >= cu_count();  // (no ranges of k)
  p.big = large(s.m, s.n, s.k * pieces, pieces == 1 || full ? kBigLeast : kBigPieces) && s.k * pieces <= kBigLine && s.m <= kBigLine;
  if (!p.big) {
    if (kind == PLX_LB_PRODUCT && s.m <= kFew) return p;
    p.splits = tiles_of(s.m, s.n, s.k, 64).splits;
    p.bytes = p.splits > 1 ? int64_t{4} * p.splits * s.m * s.n : 0;
    return p;
  }
  p.across = sm == 1 && sk != 1;
  p.kp = round_up(s.k, 64), p.mp = round_up(s.m, 8);
  const int64_t line = p.across ? sk : sm;
  p.direct = dtype == PLX_LB_BF16 && s.k % 64 == 0 && on16(a) && line % 8 == 0 && line >= 0 && line <= kBigLine &&
             (p.across ? s.m % 8 == 0 : sk == 1);
  p.bytes_w = round_up(2 * p.kp * s.n, 256);
  p.bytes_u = p.direct ? 0 : round_up(2 * pieces * p.kp * (p.across ? p.mp : s.m), 256);
  p.splits = pieces == 3 ? big_splits(s.m, s.n, p.kp / 64, 3) : big_splits(s.m, s.n, pieces * p.kp / 64, 1);
  p.bytes = p.bytes_w + p.bytes_u + (p.splits > 1 ? int64_t{4} * p.splits * s.m * s.n : 0);
  return p;
}

// out [n] = the joined sums of `splits` ranges.
template <typename OT>
void launch_join(int64_t n, int splits, const float* part, OT* out, hipStream_t s) {
  const int64_t groups = div_up(n, kBlock);
  k_mx_join<OT><<<static_cast<unsigned>(groups < kMaxGroups ? groups : kMaxGroups), kBlock, 0, s>>>(n, splits, part, out);
}

template <typename T, int KIND, typename OT>
void launch_big(const GemmArgs& g, const Plan& p, char* work, hipStream_t s) {
  constexpr int P = Pieces<T>::n;
  constexpr int BITS = KIND == kW || KIND == kWT ? 4 : 8;
  constexpr bool turned = KIND == kWT || KIND == kX;
  BigArgs b{};
  BigValues v{};
  v.lines = turned ? g.K : g.N, v.n = turned ? g.N : g.K, v.blocks = g.blocks;
  v.codes = g.codes, v.scales = g.scales, v.out = reinterpret_cast<uint16_t*>(work), v.kp = p.kp;
  v.tiles_n = static_cast<int>(div_up(g.N, 128)), v.lx = lanes_along(p.kp / 8);
  const unsigned groups = turned ? static_cast<unsigned>(p.kp / 64 * v.tiles_n) : groups_along(g.N, v.lx);
  b.w = work;
  b.ldw = 2 * p.kp;
  b.wrap = static_cast<int>(p.kp / 64), b.units = Pieces<T>::sums;
  b.steps = P / b.units * b.wrap;
  b.down[0] = kPiece2, b.down[1] = kPiece1;
  BigPieces u{};
  unsigned more = 0;
  if (p.direct) {
    b.u = static_cast<const char*>(g.a);
    b.ldu = 2 * (p.across ? g.sk : g.sm);
    b.rows_u = g.M;
  } else {
    u.x = g.a;
    u.lines = p.across ? g.K : g.M, u.n = p.across ? g.M : g.K;
    u.sl = p.across ? g.sk : g.sm, u.se = p.across ? g.sm : g.sk;
    u.out = reinterpret_cast<uint16_t*>(work + p.bytes_w);
    u.out_lines = p.across ? p.kp : g.M, u.out_n = p.across ? p.mp : p.kp;
    u.out_line = p.across ? p.mp : P * p.kp, u.piece = p.across ? p.kp * p.mp : p.kp;
    u.lx = lanes_along(u.out_n / 8);
    more = groups_along(u.out_lines, u.lx);
    b.u = work + p.bytes_w;
    b.ldu = 2 * u.out_line;
    b.rows_u = static_cast<int>(p.across ? p.mp : g.M);
  }
  k_big_operands<T, BITS, turned><<<groups + more, 256, 0, s>>>(v, u, groups);
  b.out = g.out;
  b.part = reinterpret_cast<float*>(work + p.bytes_w + p.bytes_u);
  b.M = g.M, b.N = g.N;
  b.split = static_cast<int>(div_up(b.steps, p.splits));
  b.tiles_m = static_cast<int>(div_up(g.M, kBig)), b.tiles_n = static_cast<int>(div_up(g.N, kBig));
  const dim3 grid(static_cast<unsigned>(b.tiles_m) * b.tiles_n, static_cast<unsigned>(p.splits));
  if (p.across)
    k_big_gemm<true, false, OT><<<grid, kBigThreads, 0, s>>>(b);
  else
    k_big_gemm<false, false, OT><<<grid, kBigThreads, 0, s>>>(b);
  if (p.splits > 1) launch_join(static_cast<int64_t>(g.M) * g.N, p.splits, b.part, static_cast<OT*>(g.out), s);
}

// How a product of two in 4 bits runs; `big` takes the scales in its order.
struct Plan4 {
  bool big;
  int steps, splits;
  int64_t bytes_w, bytes_u, bytes;
};
Plan4 plan4_of(int64_t m, int64_t n, int64_t k) {
  Plan4 p{};
  p.big = large(m, n, k, kBig4Least) && k <= 8 * kBigLine;
  if (!p.big) {
    p.splits = tiles_of(m, n, k, 256).splits;
    p.bytes = p.splits > 1 ? 4 * p.splits * m * n : 0;
    return p;
  }
  p.steps = static_cast<int>(div_up(k, 256));
  p.splits = big_splits(m, n, p.steps, 1);
  p.bytes_w = div_up(n, kBig) * p.steps * 2048, p.bytes_u = div_up(m, kBig) * p.steps * 2048;
  p.bytes = p.bytes_w + p.bytes_u + (p.splits > 1 ? 4 * p.splits * m * n : 0);
  return p;
}

template <typename T, int KIND, typename OT>
void launch_gemm(GemmArgs g, void* workspace, hipStream_t s) {
  const Tiles t = tiles_of(g.M, g.N, g.K, 64);
  const bool across = g.sm == 1 && g.sk != 1;
  g.kper = t.kper;
  g.tiles_n = static_cast<int>(div_up(g.N, t.ts));
  g.part = static_cast<float*>(workspace);
  const int64_t groups = kMaxGroups / (4 * t.splits);
  const int64_t rows = (groups / g.tiles_n > 0 ? groups / g.tiles_n : 1) * t.ts;  // of one launch
  const T* a = static_cast<const T*>(g.a);
  OT* out = static_cast<OT*>(g.out);
  const int64_t all = g.M;
  for (int64_t m = 0; m < all; m += rows) {  // (more than one launch only without splits)
    g.M = static_cast<int>(all - m < rows ? all - m : rows);
    g.a = a + m * g.sm;
    g.out = out + m * g.N;
    const dim3 grid(static_cast<unsigned>(div_up(g.M, t.ts) * g.tiles_n), static_cast<unsigned>(t.splits));
    with_tiles(t, [&](auto ts, auto ks) {
      constexpr int TS = decltype(ts)::value, KS = decltype(ks)::value;
      if (across)
        k_mx_gemm<T, KIND, OT, TS, KS, true><<<grid, 256 * KS, 0, s>>>(g);
      else
        k_mx_gemm<T, KIND, OT, TS, KS, false><<<grid, 256 * KS, 0, s>>>(g);
    });
  }
  if (t.splits > 1) launch_join(all * g.N, t.splits, g.part, out, s);
}

template <typename T, int KIND, typename OT>
void launch_product(const GemmArgs& g, const Plan& p, void* workspace, hipStream_t s) {
  if (p.big)
    launch_big<T, KIND, OT>(g, p, static_cast<char*>(workspace), s);
  else if (KIND == kW && g.M <= kFew && g.sk == 1 && g.K >= 8)
    k_mx_few<T, true><<<static_cast<unsigned>(div_up(g.N, 16)), 64 * kFewWaves<true>, 0, s>>>(g);
  else if (KIND == kW && g.M <= kFew)
    k_mx_few<T, false><<<static_cast<unsigned>(div_up(g.N, 16)), 64 * kFewWaves<false>, 0, s>>>(g);
  else
    launch_gemm<T, KIND, OT>(g, workspace, s);
}

}  // namespace

extern "C" {

int plx_mx4_quantise(int64_t lines, int64_t n, int32_t dtype, const void* x, int64_t line_stride, int64_t stride,
                     uint8_t* codes, uint8_t* scales, void* stream) {
  if (!dims_fit(lines, n)) return fail(PLX_ERR_INVALID, "plx_mx4_quantise: bad size");
  if (!known(dtype)) return fail(PLX_ERR_UNSUPPORTED, "plx_mx4_quantise: unknown element type");
  if (lines == 0 || n == 0) return PLX_OK;
  if (!x || !codes || !scales) return fail(PLX_ERR_INVALID, "plx_mx4_quantise: null pointer");
  if (!on16(codes)) return fail(PLX_ERR_INVALID, "plx_mx4_quantise: codes not on 16 bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(dtype, [&](auto* t) {
    using T = PLX_TYPE(t);
    const T* p = static_cast<const T*>(x);
    if (stride == 1) {
      const int lx = lanes_along(div_up(n, 128) * 16);
      k_mx4_along<T><<<groups_along(lines, lx), kBlock, 0, s>>>(lines, n, p, line_stride, codes, scales, lx);
    } else {
      k_mx4_across<T><<<groups_across(lines, div_up(n, 128) * 4), kBlock, 0, s>>>(lines, n, p, line_stride, stride,
                                                                                 codes, scales);
    }
  });
  return check_launch("plx_mx4_quantise");
}

int plx_mx_values(int32_t bits, int64_t lines, int64_t n, const uint8_t* codes, const uint8_t* scales, int32_t dtype,
                  void* out, void* stream) {
  if (bits != 4 && bits != 8) return fail(PLX_ERR_UNSUPPORTED, "plx_mx_values: 4 or 8 bits");
  if (!dims_fit(lines, n)) return fail(PLX_ERR_INVALID, "plx_mx_values: bad size");
  if (!known(dtype)) return fail(PLX_ERR_UNSUPPORTED, "plx_mx_values: unknown element type");
  if (lines == 0 || n == 0) return PLX_OK;
  if (!out || !codes || !scales) return fail(PLX_ERR_INVALID, "plx_mx_values: null pointer");
  if (!on16(codes)) return fail(PLX_ERR_INVALID, "plx_mx_values: codes not on 16 bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int lx = lanes_along(div_up(n, dtype == PLX_LB_F32 ? 4 : 8));
  with_type(dtype, [&](auto* t) {
    using T = PLX_TYPE(t);
    if (bits == 4)
      k_mx_values<4, T><<<groups_along(lines, lx), kBlock, 0, s>>>(lines, n, codes, scales, static_cast<T*>(out),
                                                                   lx);
    else
      k_mx_values<8, T><<<groups_along(lines, lx), kBlock, 0, s>>>(lines, n, codes, scales, static_cast<T*>(out),
                                                                   lx);
  });
  return check_launch("plx_mx_values");
}

int plx_mx8_activate(int64_t lines, int64_t n, int32_t dtype, int32_t fn, const void* h, int64_t h_line, int64_t h_elem,
                     void* y, int64_t y_line, int64_t y_elem, uint8_t* codes, uint8_t* scales, void* stream) {
  if (!dims_fit(lines, n)) return fail(PLX_ERR_INVALID, "plx_mx8_activate: bad size");
  if (!known(dtype)) return fail(PLX_ERR_UNSUPPORTED, "plx_mx8_activate: unknown element type");
  if (fn < PLX_LB_RELU || fn > PLX_LB_SILU) return fail(PLX_ERR_UNSUPPORTED, "plx_mx8_activate: unknown activation");
  if (lines == 0 || n == 0) return PLX_OK;
  if (!h || !codes || !scales) return fail(PLX_ERR_INVALID, "plx_mx8_activate: null pointer");
  if (!on16(codes)) return fail(PLX_ERR_INVALID, "plx_mx8_activate: codes not on 16 bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(dtype, [&](auto* t) {
    using T = PLX_TYPE(t);
    with_fn(fn, [&](auto f) {
      constexpr int FN = decltype(f)::value;
      if (h_elem == 1 && y_elem == 1) {
        const int lx = lanes_along(div_up(n, 32) * 4);
        k_act_along<FN, T><<<groups_along(lines, lx), kBlock, 0, s>>>(lines, n, static_cast<const T*>(h), h_line,
                                                                      static_cast<T*>(y), y_line, codes, scales,
                                                                      lx);
      } else {
        k_act_across<FN, T><<<groups_across(lines, div_up(n, 32)), kBlock, 0, s>>>(
            lines, n, static_cast<const T*>(h), h_line, h_elem, static_cast<T*>(y), y_line, y_elem, codes, scales);
      }
    });
  });
  return check_launch("plx_mx8_activate");
}

int plx_mx8_activate_grad(int64_t lines, int64_t n, int32_t dtype, int32_t fn, const void* dy, int64_t y_line,
                          int64_t y_elem, const uint8_t* codes, const uint8_t* scales, void* dh, int64_t h_line,
                          int64_t h_elem, void* stream) {
  if (!dims_fit(lines, n)) return fail(PLX_ERR_INVALID, "plx_mx8_activate_grad: bad size");
  if (!known(dtype)) return fail(PLX_ERR_UNSUPPORTED, "plx_mx8_activate_grad: unknown element type");
  if (fn < PLX_LB_RELU || fn > PLX_LB_SILU)
    return fail(PLX_ERR_UNSUPPORTED, "plx_mx8_activate_grad: unknown activation");
  if (lines == 0 || n == 0) return PLX_OK;
  if (!dy || !dh || !codes || !scales) return fail(PLX_ERR_INVALID, "plx_mx8_activate_grad: null pointer");
  if (!on16(codes)) return fail(PLX_ERR_INVALID, "plx_mx8_activate_grad: codes not on 16 bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(dtype, [&](auto* t) {
    using T = PLX_TYPE(t);
    with_fn(fn, [&](auto f) {
      constexpr int FN = decltype(f)::value;
      if (y_elem == 1 && h_elem == 1) {
        const int lx = lanes_along(div_up(n, 8));
        k_grad_along<FN, T><<<groups_along(lines, lx), kBlock, 0, s>>>(lines, n, static_cast<const T*>(dy), y_line,
                                                                       codes, scales, static_cast<T*>(dh), h_line,
                                                                       lx);
      } else {
        k_grad_across<FN, T><<<groups_across(lines, div_up(n, 32)), kBlock, 0, s>>>(
            lines, n, static_cast<const T*>(dy), y_line, y_elem, codes, scales, static_cast<T*>(dh), h_line, h_elem);
      }
    });
  });
  return check_launch("plx_mx8_activate_grad");
}

int64_t plx_mx_workspace(int32_t kind, int64_t tokens, int64_t inputs, int64_t outputs, int32_t dtype, const void* a,
                         int64_t token_stride, int64_t unit_stride) {
  if (kind < PLX_LB_PRODUCT || kind > PLX_LB_WEIGHT_GRAD_COLUMNS || !known(dtype) ||
      !product_fits(tokens, inputs, outputs))
    return -1;
  const bool grad = kind >= PLX_LB_WEIGHT_GRAD;
  return plan_of(kind, shape_of(kind, tokens, inputs, outputs), dtype, a, grad ? unit_stride : token_stride,
                 grad ? token_stride : unit_stride)
      .bytes;
}

int plx_mx_product(int32_t kind, int64_t tokens, int64_t inputs, int64_t outputs, int32_t dtype, const void* a,
                   int64_t token_stride, int64_t unit_stride, const uint8_t* codes, const uint8_t* scales, void* out,
                   void* workspace, int64_t workspace_bytes, void* stream) {
  if (kind < PLX_LB_PRODUCT || kind > PLX_LB_WEIGHT_GRAD_COLUMNS)
    return fail(PLX_ERR_UNSUPPORTED, "plx_mx_product: unknown kind");
  if (!product_fits(tokens, inputs, outputs)) return fail(PLX_ERR_INVALID, "plx_mx_product: bad size");
  if (!known(dtype)) return fail(PLX_ERR_UNSUPPORTED, "plx_mx_product: unknown element type");
  const Shape sh = shape_of(kind, tokens, inputs, outputs);
  if (sh.m == 0 || sh.n == 0) return PLX_OK;
  if (!out || (sh.k > 0 && (!a || !codes || !scales))) return fail(PLX_ERR_INVALID, "plx_mx_product: null pointer");
  if (!on16(codes)) return fail(PLX_ERR_INVALID, "plx_mx_product: codes not on 16 bytes");
  GemmArgs g{};
  g.a = a, g.codes = codes, g.scales = scales, g.out = out;
  g.M = static_cast<int>(sh.m), g.N = static_cast<int>(sh.n), g.K = static_cast<int>(sh.k);
  const bool grad = kind >= PLX_LB_WEIGHT_GRAD;
  g.sm = grad ? unit_stride : token_stride, g.sk = grad ? token_stride : unit_stride;
  g.blocks = grad ? div_up(kind == PLX_LB_WEIGHT_GRAD ? inputs : tokens, 32) : div_up(inputs, 128) * 4;
  const Plan p = plan_of(kind, sh, dtype, a, g.sm, g.sk);
  if (p.bytes > 0 && (!workspace || !on16(workspace) || workspace_bytes < p.bytes))
    return fail(PLX_ERR_INVALID, "plx_mx_product: plx_mx_workspace() bytes on 16 bytes needed");
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(dtype, [&](auto* t) {
    using T = PLX_TYPE(t);
    switch (kind) {
      case PLX_LB_PRODUCT: launch_product<T, kW, T>(g, p, workspace, s); break;
      case PLX_LB_PRODUCT_GRAD: launch_product<T, kWT, T>(g, p, workspace, s); break;
      case PLX_LB_WEIGHT_GRAD: launch_product<T, kX, float>(g, p, workspace, s); break;
      default: launch_product<T, kXT, float>(g, p, workspace, s); break;
    }
  });
  return check_launch("plx_mx_product");
}

int64_t plx_mx4_workspace(int64_t tokens, int64_t inputs, int64_t outputs) {
  if (!product_fits(tokens, inputs, outputs)) return -1;
  return plan4_of(tokens, outputs, inputs).bytes;
}

int plx_mx4_product(int64_t tokens, int64_t inputs, int64_t outputs, const uint8_t* x_codes, const uint8_t* x_scales,
                    const uint8_t* w_codes, const uint8_t* w_scales, int32_t dtype, void* out, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  if (!product_fits(tokens, inputs, outputs)) return fail(PLX_ERR_INVALID, "plx_mx4_product: bad size");
  if (!known(dtype)) return fail(PLX_ERR_UNSUPPORTED, "plx_mx4_product: unknown element type");
  if (tokens == 0 || outputs == 0) return PLX_OK;
  if (!out || (inputs > 0 && (!x_codes || !x_scales || !w_codes || !w_scales)))
    return fail(PLX_ERR_INVALID, "plx_mx4_product: null pointer");
  if (!on16(x_codes) || !on16(w_codes)) return fail(PLX_ERR_INVALID, "plx_mx4_product: codes not on 16 bytes");
  const Plan4 p = plan4_of(tokens, outputs, inputs);
  if (p.bytes > 0 && (!workspace || !on16(workspace) || workspace_bytes < p.bytes))
    return fail(PLX_ERR_INVALID, "plx_mx4_product: plx_mx4_workspace() bytes on 16 bytes needed");
  const int64_t blocks = div_up(inputs, 128) * 4;
  if (p.big) {
    hipStream_t s = static_cast<hipStream_t>(stream);
    char* work = static_cast<char*>(workspace);
    BigArgs g{};
    g.w = reinterpret_cast<const char*>(w_codes), g.u = reinterpret_cast<const char*>(x_codes);
    g.sw = work, g.su = work + p.bytes_w;
    g.out = out, g.part = reinterpret_cast<float*>(work + p.bytes_w + p.bytes_u);
    g.M = g.rows_u = static_cast<int>(tokens), g.N = static_cast<int>(outputs);
    g.ldw = g.ldu = blocks * 16;
    g.steps = g.wrap = p.steps, g.units = 1, g.split = static_cast<int>(div_up(p.steps, p.splits));
    g.tiles_m = static_cast<int>(div_up(tokens, kBig)), g.tiles_n = static_cast<int>(div_up(outputs, kBig));
    k_big_scales<<<static_cast<unsigned>((g.tiles_m + g.tiles_n) * div_up(p.steps, 8)), 256, 0, s>>>(
        g.N, g.M, blocks, div_up(inputs, 32), p.steps, w_scales, x_scales, reinterpret_cast<uint8_t*>(work),
        reinterpret_cast<uint8_t*>(work + p.bytes_w));
    with_type(dtype, [&](auto* t) {
      using T = PLX_TYPE(t);
      const dim3 grid(static_cast<unsigned>(g.tiles_m) * g.tiles_n, static_cast<unsigned>(p.splits));
      k_big_gemm<false, true, T><<<grid, kBigThreads, 0, s>>>(g);
      if (p.splits > 1) launch_join(tokens * outputs, p.splits, g.part, static_cast<T*>(out), s);
    });
    return check_launch("plx_mx4_product");
  }
  const Tiles t = tiles_of(tokens, outputs, inputs, 256);
  const int tiles_n = static_cast<int>(div_up(outputs, t.ts));
  const int64_t groups = kMaxGroups / (4 * t.splits);
  const int64_t rows = (groups / tiles_n > 0 ? groups / tiles_n : 1) * t.ts;  // of one launch
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(dtype, [&](auto* e) {
    using T = PLX_TYPE(e);
    for (int64_t m = 0; m < tokens; m += rows) {  // (more than one launch only without splits)
      const int64_t now = tokens - m < rows ? tokens - m : rows;
      const dim3 grid(static_cast<unsigned>(div_up(now, t.ts) * tiles_n), static_cast<unsigned>(t.splits));
      with_tiles(t, [&](auto ts, auto ks) {
        constexpr int TS = decltype(ts)::value, KS = decltype(ks)::value;
        k_mx4_gemm<T, TS, KS><<<grid, 256 * KS, 0, s>>>(
            static_cast<int>(now), static_cast<int>(outputs), static_cast<int>(inputs), static_cast<int>(blocks),
            x_codes + m * blocks * 16, x_scales + m * blocks, w_codes, w_scales, static_cast<T*>(out) + m * outputs,
            static_cast<float*>(workspace), tiles_n, t.kper / 32);
      });
    }
    if (t.splits > 1)
      launch_join(tokens * outputs, t.splits, static_cast<const float*>(workspace), static_cast<T*>(out), s);
  });
  return check_launch("plx_mx4_product");
}

}  // extern "C"
