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
#include "px_math.h"

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
// Lines of values and their blocks. "Along" kernels: the line's values lie
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
__global__ __launch_bounds__(kBlock) void k_mx4_along(int64_t lines, int64_t n, const T* x, int64_t stride, bool wide,
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
      load8(row + c * 8, 1, left > 8 ? 8 : left < 0 ? 0 : static_cast<int>(left), wide, v);
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
template <int BITS, typename T>
__global__ __launch_bounds__(kBlock) void k_mx_values(int64_t lines, int64_t n, const uint8_t* codes,
                                                      const uint8_t* scales, T* out, bool wide, int lx) {
  const int64_t kept = BITS == 4 ? div_up(n, 128) * 16 : div_up(n, 32) * 4, chunks = div_up(n, 8);
  const int tx = threadIdx.x & (lx - 1), ly = kBlock / lx, ty = threadIdx.x / lx;
  for (int64_t line = static_cast<int64_t>(blockIdx.x) * ly + ty; line < lines;
       line += static_cast<int64_t>(gridDim.x) * ly) {
    for (int64_t c = tx; c < chunks; c += lx) {
      const float scale = scale_value(scales[line * (kept / 4) + c / 4]);
      const int64_t left = n - c * 8;
      float v[8];
      if (BITS == 4)
        values4(reinterpret_cast<const uint32_t*>(codes)[line * kept + c], scale, v);
      else
        values8(reinterpret_cast<const uint2*>(codes)[line * kept + c], scale, v);
      store8(out + line * n + c * 8, 1, left > 8 ? 8 : static_cast<int>(left), wide, v);
    }
  }
}

// ---------------------------------------------------------------------------
// Activations. y = fn(h) from h itself; fn'(q) from what was kept.
// ---------------------------------------------------------------------------
template <int FN>
__device__ __forceinline__ float act(float h) {
  if (FN == PLX_LB_RELU) return h <= 0.0f ? 0.0f : h;  // (a NaN passes)
  if (FN == PLX_LB_TANH) return tanhf_(h);
  const float t = expf_(-fabsf(h)), d = 1.0f + t;  // (nothing overflows, so the tails keep their values)
  const float s = (h < 0.0f ? t : 1.0f) / d;
  return FN == PLX_LB_SIGMOID ? s : h * s;
}
// By exp(-|q|), so that nothing overflows: tanh' = 4u / (1 + u)^2 with
// u = exp(-2|q|), sigmoid' = t / (1 + t)^2 with t = exp(-|q|), and
// silu' = sigmoid(q) + q sigmoid'(q).
template <int FN>
__device__ __forceinline__ float act_grad(float q) {
  if (FN == PLX_LB_RELU) return q > 0.0f ? 1.0f : 0.0f;
  const float a = fabsf(q);
  const float t = expf_(FN == PLX_LB_TANH ? -2.0f * a : -a);
  const float r = 1.0f / (1.0f + t), d = t * r * r;
  if (FN == PLX_LB_TANH) return 4.0f * d;
  if (FN == PLX_LB_SIGMOID) return d;
  return (q >= 0.0f ? r : t * r) + (t == 0.0f ? 0.0f : q * d);  // (an infinite q has the slope 0 or 1)
}

template <int FN, typename T>
__global__ __launch_bounds__(kBlock) void k_act_along(int64_t lines, int64_t n, const T* h, int64_t sh, T* y,
                                                      int64_t sy, bool wide, uint8_t* codes, uint8_t* scales, int lx) {
  const int64_t chunks = div_up(n, 32) * 4;
  const int tx = threadIdx.x & (lx - 1), ly = kBlock / lx, ty = threadIdx.x / lx;
  for (int64_t line = static_cast<int64_t>(blockIdx.x) * ly + ty; line < lines;
       line += static_cast<int64_t>(gridDim.x) * ly) {
    for (int64_t c = tx; c < chunks; c += lx) {
      const int64_t left64 = n - c * 8;
      const int left = left64 > 8 ? 8 : left64 < 0 ? 0 : static_cast<int>(left64);
      float v[8], f[8];
      load8(h + line * sh + c * 8, 1, left, wide, v);
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = abs_bits(v[i]);
        m = a < kInfBits && a > m ? a : m;
        f[i] = act<FN>(v[i]);
      }
      store8(y + line * sy + c * 8, 1, left, wide, f);
      const int e = exponent8(max4(m));
      reinterpret_cast<uint2*>(codes)[line * chunks + c] = codes8(v, pow2(-e));
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
    for (int i = 0; i < 32; ++i) {
      v[i / 8][i % 8] = i < left ? to_f32(p[i * se]) : 0.0f;
      const uint32_t a = abs_bits(v[i / 8][i % 8]);
      m = a < kInfBits && a > m ? a : m;
    }
    const int e = exponent8(m);
    uint2* c = reinterpret_cast<uint2*>(codes) + (line * blocks + b) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = codes8(v[i], pow2(-e));
    scales[line * blocks + b] = static_cast<uint8_t>(e + 127);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < left) o[i * ye] = from_f32<T>(act<FN>(v[i / 8][i % 8]));
  }
}

template <int FN, typename T>
__global__ __launch_bounds__(kBlock) void k_grad_along(int64_t lines, int64_t n, const T* dy, int64_t sy,
                                                       const uint8_t* codes, const uint8_t* scales, T* dh, int64_t sh,
                                                       bool wide, int lx) {
  const int64_t kept = div_up(n, 32) * 4, chunks = div_up(n, 8);
  const int tx = threadIdx.x & (lx - 1), ly = kBlock / lx, ty = threadIdx.x / lx;
  for (int64_t line = static_cast<int64_t>(blockIdx.x) * ly + ty; line < lines;
       line += static_cast<int64_t>(gridDim.x) * ly) {
    for (int64_t c = tx; c < chunks; c += lx) {
      const int64_t left64 = n - c * 8;
      const int left = left64 > 8 ? 8 : static_cast<int>(left64);
      float v[8], q[8];
      load8(dy + line * sy + c * 8, 1, left, wide, v);
      values8(reinterpret_cast<const uint2*>(codes)[line * kept + c], scale_value(scales[line * (kept / 4) + c / 4]),
              q);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= act_grad<FN>(q[i]);
      store8(dh + line * sh + c * 8, 1, left, wide, v);
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
      float q[8];
      values8(c[i], scale, q);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i * 8 + j < left) o[(i * 8 + j) * he] = from_f32<T>(to_f32(p[(i * 8 + j) * se]) * act_grad<FN>(q[j]));
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
// the matrix instruction round.
// ---------------------------------------------------------------------------
enum { kW = 0, kWT = 1, kX = 2, kXT = 3 };

struct GemmArgs {
  const void* a;
  int64_t sm, sk;
  bool wide;
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t blocks;  // blocks of a line of codes
  void* out;       // [m][n]
  float* part;     // [splits][m][n], where splits > 1
  int M, N, K, kper, tiles_n;
};

constexpr int kTile = 64;

// 64 x 64 of the output by four waves of 32 x 32, k in steps of 64: both
// operands go through registers (converted to bf16 on the way) into LDS, the
// next step's loads in flight during this step's matrix instructions. In LDS
// a row is 64 k (8 chunks of 16 bytes), chunk c of row r at c ^ (r & 7): the
// 16 rows of a fragment's read then fall on different banks.
template <typename T, int KIND, typename OT>
__global__ __launch_bounds__(256) void k_mx_gemm(GemmArgs g) {
  constexpr int P = Pieces<T>::n;
  __shared__ uint4 la[P][kTile * 8];
  __shared__ uint4 lb[kTile * 8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m0 = (blockIdx.x / g.tiles_n) * kTile, n0 = (blockIdx.x % g.tiles_n) * kTile;
  const int kbeg = blockIdx.y * g.kper, kend = kbeg + g.kper < g.K ? kbeg + g.kper : g.K;
  const T* a = static_cast<const T*>(g.a);
  const bool along = g.sk == 1;

  float ra[2][8];
  uint4 rb = make_uint4(0, 0, 0, 0);
  uint2 rs = make_uint2(0, 0);

  auto load = [&](int k0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int u = tid + 256 * i;
      const int row = along ? u >> 3 : u & 63, c = along ? u & 7 : u >> 6;
      const int m = m0 + row, k = k0 + c * 8;
      const int left = m < g.M ? (kend - k > 8 ? 8 : kend - k) : 0;
      load8(a + m * g.sm + k * g.sk, g.sk, left, g.wide, ra[i]);
    }
    rb = make_uint4(0, 0, 0, 0), rs = make_uint2(0, 0);
    if (KIND == kW || KIND == kXT) {
      const int n = n0 + (tid >> 2), k = k0 + (tid & 3) * 16;
      if (n < g.N && k < kend) {  // (a started block is whole in memory)
        const int64_t b = n * g.blocks + k / 32;
        if (KIND == kW) {
          const uint2 c = *reinterpret_cast<const uint2*>(g.codes + b * 16 + (k & 16) / 2);
          rb.x = c.x, rb.y = c.y;
        } else {
          rb = *reinterpret_cast<const uint4*>(g.codes + b * 32 + (k & 16));
        }
        rs.x = g.scales[b];
      }
    } else {
      const int n = n0 + (tid & 31) * 2, k = k0 + (tid >> 5) * 8;
      uint32_t c[8], s[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = s[i] = 0;
        if (k + i < kend && n < g.N) {
          const int64_t b = (k + i) * g.blocks + n / 32;
          c[i] = KIND == kWT ? g.codes[b * 16 + (n & 31) / 2]
                             : *reinterpret_cast<const uint16_t*>(g.codes + b * 32 + (n & 31));
          s[i] = g.scales[b];
        }
      }
      if (KIND == kWT) {
        rb.x = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
        rb.y = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
      } else {
        rb = make_uint4(c[0] | c[1] << 16, c[2] | c[3] << 16, c[4] | c[5] << 16, c[6] | c[7] << 16);
      }
      rs.x = s[0] | s[1] << 8 | s[2] << 16 | s[3] << 24;
      rs.y = s[4] | s[5] << 8 | s[6] << 16 | s[7] << 24;
    }
  };
  auto put = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int u = tid + 256 * i;
      const int row = along ? u >> 3 : u & 63, c = along ? u & 7 : u >> 6;
      uint4 p[P];
      pieces8<P>(ra[i], p);
#pragma unroll
      for (int j = 0; j < P; ++j) la[j][row * 8 + (c ^ (row & 7))] = p[j];
    }
    if (KIND == kW || KIND == kXT) {
      const int row = tid >> 2, c = (tid & 3) * 2;
      const float scale = scale_value(rs.x);
      uint4 lo, hi;
      if (KIND == kW) {
        lo = bf16_of4(rb.x, scale), hi = bf16_of4(rb.y, scale);
      } else {
        lo = bf16_of8(make_uint2(rb.x, rb.y), scale), hi = bf16_of8(make_uint2(rb.z, rb.w), scale);
      }
      lb[row * 8 + (c ^ (row & 7))] = lo;
      lb[row * 8 + ((c + 1) ^ (row & 7))] = hi;
    } else {
      const int row = (tid & 31) * 2, c = tid >> 5;
      const uint32_t r[4] = {rb.x, rb.y, rb.z, rb.w}, s[2] = {rs.x, rs.y};
      float even[8], odd[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float scale = scale_value(s[i / 4] >> (8 * (i % 4)) & 255u);
        f32x2 v;
        if (KIND == kWT) {
          v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r[i / 4] >> (8 * (i % 4)), scale, 0);
        } else {
          v = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(r[i / 2] >> (16 * (i % 2))), false);
          v[0] *= scale, v[1] *= scale;
        }
        even[i] = v[0], odd[i] = v[1];
      }
      uint4 p[1];
      pieces8<1>(even, p);
      lb[row * 8 + (c ^ (row & 7))] = p[0];
      pieces8<1>(odd, p);
      lb[(row + 1) * 8 + (c ^ ((row + 1) & 7))] = p[0];
    }
  };

  f32x4 acc[2][2] = {};
  const int wn = (wave & 1) * 32, wm = (wave >> 1) * 32, l15 = lane & 15, q = lane >> 4;
  if (kbeg < kend) load(kbeg);
  for (int k0 = kbeg; k0 < kend; k0 += 64) {
    __syncthreads();
    put();
    __syncthreads();
    if (k0 + 64 < kend) load(k0 + 64);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 fb[2], fa[2][P];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rn = wn + i * 16 + l15, rm = wm + i * 16 + l15, c = s * 4 + q;
        fb[i] = as_bf16x8(lb[rn * 8 + (c ^ (rn & 7))]);
#pragma unroll
        for (int p = 0; p < P; ++p) fa[i][p] = as_bf16x8(la[p][rm * 8 + (c ^ (rm & 7))]);
      }
#pragma unroll
      for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[i], fa[j][p], acc[i][j], 0, 0, 0);
    }
  }
  // With b's rows as the instruction's first operand a lane holds four
  // consecutive n of one m.
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int m = m0 + wm + j * 16 + l15, n = n0 + wn + i * 16 + q * 4;
      if (m >= g.M) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (n + r >= g.N) break;
        const int64_t at = static_cast<int64_t>(m) * g.N + n + r;
        if (gridDim.y > 1)
          g.part[static_cast<int64_t>(blockIdx.y) * g.M * g.N + at] = acc[i][j][r];
        else
          static_cast<OT*>(g.out)[at] = from_f32<OT>(acc[i][j][r]);
      }
    }
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

// 4-bit times 4-bit blocks: the scaled matrix instruction takes 128 k of both
// operands as they are kept, one block and its scale byte per lane.
template <typename OT>
__global__ __launch_bounds__(256) void k_mx4_gemm(int M, int N, int64_t blocks, const uint8_t* xc, const uint8_t* xs,
                                                  const uint8_t* wc, const uint8_t* ws, OT* out, int tiles_n) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, q = lane >> 4;
  const int m0 = (blockIdx.x / tiles_n) * kTile + (wave >> 1) * 32;
  const int n0 = (blockIdx.x % tiles_n) * kTile + (wave & 1) * 32;
  f32x4 acc[2][2] = {};
  int64_t rm[2], rn[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // (rows past the end read the last one; their results are not written)
    const int m = m0 + i * 16 + l15, n = n0 + i * 16 + l15;
    rm[i] = (m < M ? m : M - 1) * blocks, rn[i] = (n < N ? n : N - 1) * blocks;
  }
  for (int64_t b = q; b < blocks; b += 4) {
    i32x8 fx[2], fw[2];
    int sx[2], sw[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 cx = reinterpret_cast<const uint4*>(xc)[rm[i] + b], cw = reinterpret_cast<const uint4*>(wc)[rn[i] + b];
      fx[i] = i32x8{static_cast<int>(cx.x), static_cast<int>(cx.y), static_cast<int>(cx.z), static_cast<int>(cx.w)};
      fw[i] = i32x8{static_cast<int>(cw.x), static_cast<int>(cw.y), static_cast<int>(cw.z), static_cast<int>(cw.w)};
      sx[i] = xs[rm[i] + b], sw[i] = ws[rn[i] + b];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[i], fx[j], acc[i][j], 4, 4, 0, sw[i], 0, sx[j]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int m = m0 + j * 16 + l15, n = n0 + i * 16 + q * 4;
      if (m >= M) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < N) out[static_cast<int64_t>(m) * N + n + r] = from_f32<OT>(acc[i][j][r]);
    }
}

// ---------------------------------------------------------------------------
// Operands of the large products: bf16 lines padded with zeros.
// ---------------------------------------------------------------------------
// Piece p of line l at out + p * piece + l * out_line.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_big_pieces(int64_t lines, int64_t n, const T* x, int64_t sl, int64_t se,
                                                       bool wide, uint16_t* out, int64_t out_lines, int64_t out_n,
                                                       int64_t out_line, int64_t piece, int lx) {
  constexpr int P = Pieces<T>::n;
  const int tx = threadIdx.x & (lx - 1), ly = kBlock / lx, ty = threadIdx.x / lx;
  for (int64_t line = static_cast<int64_t>(blockIdx.x) * ly + ty; line < out_lines;
       line += static_cast<int64_t>(gridDim.x) * ly) {
    for (int64_t c = tx; c < out_n / 8; c += lx) {
      const int64_t left = line < lines ? n - c * 8 : 0;
      float v[8];
      load8(x + line * sl + c * 8 * se, se, left > 8 ? 8 : left < 0 ? 0 : static_cast<int>(left), wide, v);
      uint4 p[P];
      pieces8<P>(v, p);
#pragma unroll
      for (int i = 0; i < P; ++i) *reinterpret_cast<uint4*>(out + i * piece + line * out_line + c * 8) = p[i];
    }
  }
}

template <int BITS>
__global__ __launch_bounds__(kBlock) void k_big_values(int64_t lines, int64_t n, const uint8_t* codes,
                                                       const uint8_t* scales, uint16_t* out, int64_t out_lines,
                                                       int64_t out_n, int lx) {
  const int64_t kept = BITS == 4 ? div_up(n, 128) * 16 : div_up(n, 32) * 4;
  const int tx = threadIdx.x & (lx - 1), ly = kBlock / lx, ty = threadIdx.x / lx;
  for (int64_t line = static_cast<int64_t>(blockIdx.x) * ly + ty; line < out_lines;
       line += static_cast<int64_t>(gridDim.x) * ly) {
    for (int64_t c = tx; c < out_n / 8; c += lx) {
      uint4 r = make_uint4(0, 0, 0, 0);
      if (line < lines && c < kept) {
        const float scale = scale_value(scales[line * (kept / 4) + c / 4]);
        r = BITS == 4 ? bf16_of4(reinterpret_cast<const uint32_t*>(codes)[line * kept + c], scale)
                      : bf16_of8(reinterpret_cast<const uint2*>(codes)[line * kept + c], scale);
      }
      *reinterpret_cast<uint4*>(out + line * out_n + c * 8) = r;
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr int64_t kMaxDim = int64_t{1} << 30;
constexpr int64_t kBigLeast = 256;              // m, n and k of a large product
constexpr int64_t kBigLine = int64_t{1} << 22;  // elements of its lines: 256 of them stay below 2^32 bytes

inline bool dims_fit(int64_t a, int64_t b) { return a >= 0 && b >= 0 && a <= kMaxDim && b <= kMaxDim; }
inline int size_of(int dtype) { return dtype == PLX_LB_F32 ? 4 : 2; }
inline bool known(int dtype) { return dtype == PLX_LB_F32 || dtype == PLX_LB_BF16 || dtype == PLX_LB_F16; }

// Rows of this stride can be read 16 bytes at a time.
inline bool rows_on16(const void* p, int64_t stride, int dtype) { return on16(p) && (stride * size_of(dtype)) % 16 == 0; }

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

// The k ranges of a product: enough workgroups for two per CU, each range
// four steps of 64 at least.
int splits_of(int64_t m, int64_t n, int64_t k) {
  const int64_t tiles = div_up(m, kTile) * div_up(n, kTile);
  int64_t s = 2 * cu_count() / (tiles > 0 ? tiles : 1);
  const int64_t most = div_up(k, 256);
  s = s < most ? s : most;
  return static_cast<int>(s < 1 ? 1 : s > 64 ? 64 : s);
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
  bool across_a, across_b, direct;
  int64_t kp;       // k padded to whole steps
  int64_t mp, np;   // padded rows' lengths of "across" operands
  int64_t bytes_a, bytes_b, bytes;
};

// Workgroups that a large product should fill: one per CU.
int big_splits(int64_t m, int64_t n, int64_t steps) {
  const int64_t tiles = div_up(m, kBig) * div_up(n, kBig);
  int64_t s = cu_count() / (tiles > 0 ? tiles : 1);
  s = s < steps / 8 ? s : steps / 8;
  if (s < 2) return 1;
  return static_cast<int>(div_up(steps, div_up(steps, s)));  // (no range is empty)
}

Plan plan_of(int kind, const Shape& s, int dtype, const void* a, int64_t sm, int64_t sk) {
  Plan p{};
  const int pieces = dtype == PLX_LB_F32 ? 3 : dtype == PLX_LB_F16 ? 2 : 1;
  p.big = s.m >= kBigLeast && s.n >= kBigLeast && s.k >= kBigLeast;
  if (!p.big) {
    p.splits = splits_of(s.m, s.n, s.k);
    p.bytes = p.splits > 1 ? int64_t{4} * p.splits * s.m * s.n : 0;
    return p;
  }
  p.across_a = sm == 1 && sk != 1;
  p.across_b = kind == PLX_LB_PRODUCT_GRAD || kind == PLX_LB_WEIGHT_GRAD;
  p.kp = round_up(s.k, 64), p.mp = round_up(s.m, 8), p.np = round_up(s.n, 8);
  const int64_t line = p.across_a ? sk : sm;
  p.direct = dtype == PLX_LB_BF16 && s.k % 64 == 0 && on16(a) && line % 8 == 0 && line <= kBigLine &&
             (p.across_a ? s.m % 8 == 0 : sk == 1);
  p.bytes_a = p.direct ? 0 : round_up(2 * pieces * p.kp * (p.across_a ? p.mp : s.m), 256);
  p.bytes_b = round_up(2 * p.kp * (p.across_b ? p.np : s.n), 256);
  p.splits = big_splits(s.m, s.n, pieces * p.kp / 64);
  p.bytes = p.bytes_a + p.bytes_b + (p.splits > 1 ? int64_t{4} * p.splits * s.m * s.n : 0);
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
  constexpr bool BA = KIND == kWT || KIND == kX;
  BigArgs b{};
  if (p.direct) {
    b.a = static_cast<const char*>(g.a);
    b.lda = 2 * (p.across_a ? g.sk : g.sm);
    b.rows_a = g.M;
  } else {
    uint16_t* out = reinterpret_cast<uint16_t*>(work);
    const int64_t lines = p.across_a ? g.K : g.M, n = p.across_a ? g.M : g.K;
    const int64_t sl = p.across_a ? g.sk : g.sm, se = p.across_a ? g.sm : g.sk;
    const int64_t out_lines = p.across_a ? p.kp : g.M, out_n = p.across_a ? p.mp : p.kp;
    const int64_t out_line = p.across_a ? p.mp : P * p.kp, piece = p.across_a ? p.kp * p.mp : p.kp;
    const int lx = lanes_along(out_n / 8);
    const bool wide = se == 1 && on16(g.a) && (sl * sizeof(T)) % 16 == 0;
    k_big_pieces<T><<<groups_along(out_lines, lx), kBlock, 0, s>>>(lines, n, static_cast<const T*>(g.a), sl, se, wide,
                                                                   out, out_lines, out_n, out_line, piece, lx);
    b.a = work;
    b.lda = 2 * out_line;
    b.rows_a = static_cast<int>(p.across_a ? p.mp : g.M);
  }
  uint16_t* vb = reinterpret_cast<uint16_t*>(work + p.bytes_a);
  const int64_t lines = BA ? g.K : g.N, out_lines = BA ? p.kp : g.N, out_n = BA ? p.np : p.kp;
  const int lx = lanes_along(out_n / 8);
  k_big_values<KIND == kW || KIND == kWT ? 4 : 8><<<groups_along(out_lines, lx), kBlock, 0, s>>>(
      lines, BA ? g.N : g.K, g.codes, g.scales, vb, out_lines, out_n, lx);
  b.b = reinterpret_cast<const char*>(vb);
  b.ldb = 2 * out_n;
  b.rows_b = static_cast<int>(BA ? p.np : g.N);
  b.out = g.out;
  b.part = reinterpret_cast<float*>(work + p.bytes_a + p.bytes_b);
  b.M = g.M, b.N = g.N;
  b.wrap = static_cast<int>(p.kp / 64), b.steps = P * b.wrap;
  b.split = static_cast<int>(div_up(b.steps, p.splits));
  b.tiles_m = static_cast<int>(div_up(g.M, kBig)), b.tiles_n = static_cast<int>(div_up(g.N, kBig));
  const dim3 grid(static_cast<unsigned>(b.tiles_m) * b.tiles_n, static_cast<unsigned>(p.splits));
  if (p.across_a)
    k_big_gemm<true, BA, OT><<<grid, kBigThreads, 0, s>>>(b);
  else
    k_big_gemm<false, BA, OT><<<grid, kBigThreads, 0, s>>>(b);
  if (p.splits > 1) launch_join(static_cast<int64_t>(g.M) * g.N, p.splits, b.part, static_cast<OT*>(g.out), s);
}

// How a product of two in 4 bits runs; `big` takes the scales in its order.
struct Plan4 {
  bool big;
  int steps, splits;
  int64_t bytes_a, bytes_b, bytes;
};
Plan4 plan4_of(int64_t m, int64_t n, int64_t k) {
  Plan4 p{};
  p.big = m >= kBigLeast && n >= kBigLeast && k >= kBigLeast && k <= 8 * kBigLine;
  if (!p.big) return p;
  p.steps = static_cast<int>(div_up(k, 256));
  p.splits = big_splits(m, n, p.steps);
  p.bytes_a = div_up(m, 128) * p.steps * 64 * 16, p.bytes_b = div_up(n, 64) * p.steps * 64 * 8;
  p.bytes = p.bytes_a + p.bytes_b + (p.splits > 1 ? 4 * p.splits * m * n : 0);
  return p;
}

template <typename T, int KIND, typename OT>
void launch_gemm(GemmArgs g, void* workspace, hipStream_t s) {
  const int splits = splits_of(g.M, g.N, g.K);
  g.kper = static_cast<int>(div_up(div_up(g.K, splits), 64) * 64);
  g.tiles_n = static_cast<int>(div_up(g.N, kTile));
  g.part = static_cast<float*>(workspace);
  const int64_t rows = (kMaxGroups / g.tiles_n > 0 ? kMaxGroups / g.tiles_n : 1) * kTile;  // of one launch
  const T* a = static_cast<const T*>(g.a);
  OT* out = static_cast<OT*>(g.out);
  const int64_t all = g.M;
  for (int64_t m = 0; m < all; m += rows) {
    g.M = static_cast<int>(all - m < rows ? all - m : rows);
    g.a = a + m * g.sm;
    g.out = out + m * g.N;
    const dim3 grid(static_cast<unsigned>(div_up(g.M, kTile) * g.tiles_n), static_cast<unsigned>(splits));
    k_mx_gemm<T, KIND, OT><<<grid, 256, 0, s>>>(g);
  }
  if (splits > 1) launch_join(all * g.N, splits, g.part, out, s);  // (then there are few tiles: one launch)
}

template <typename T, int KIND, typename OT>
void launch_product(const GemmArgs& g, const Plan& p, void* workspace, hipStream_t s) {
  if (p.big)
    launch_big<T, KIND, OT>(g, p, static_cast<char*>(workspace), s);
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
      k_mx4_along<T><<<groups_along(lines, lx), kBlock, 0, s>>>(lines, n, p, line_stride,
                                                                rows_on16(x, line_stride, dtype), codes, scales, lx);
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
  const int lx = lanes_along(div_up(n, 8));
  with_type(dtype, [&](auto* t) {
    using T = PLX_TYPE(t);
    const bool wide = rows_on16(out, n, dtype);
    if (bits == 4)
      k_mx_values<4, T><<<groups_along(lines, lx), kBlock, 0, s>>>(lines, n, codes, scales, static_cast<T*>(out), wide,
                                                                   lx);
    else
      k_mx_values<8, T><<<groups_along(lines, lx), kBlock, 0, s>>>(lines, n, codes, scales, static_cast<T*>(out), wide,
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
  if (!h || !y || !codes || !scales) return fail(PLX_ERR_INVALID, "plx_mx8_activate: null pointer");
  if (!on16(codes)) return fail(PLX_ERR_INVALID, "plx_mx8_activate: codes not on 16 bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(dtype, [&](auto* t) {
    using T = PLX_TYPE(t);
    with_fn(fn, [&](auto f) {
      constexpr int FN = decltype(f)::value;
      if (h_elem == 1 && y_elem == 1) {
        const int lx = lanes_along(div_up(n, 32) * 4);
        const bool wide = rows_on16(h, h_line, dtype) && rows_on16(y, y_line, dtype);
        k_act_along<FN, T><<<groups_along(lines, lx), kBlock, 0, s>>>(lines, n, static_cast<const T*>(h), h_line,
                                                                      static_cast<T*>(y), y_line, wide, codes, scales,
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
        const bool wide = rows_on16(dy, y_line, dtype) && rows_on16(dh, h_line, dtype);
        k_grad_along<FN, T><<<groups_along(lines, lx), kBlock, 0, s>>>(lines, n, static_cast<const T*>(dy), y_line,
                                                                       codes, scales, static_cast<T*>(dh), h_line, wide,
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
  if (kind < PLX_LB_PRODUCT || kind > PLX_LB_WEIGHT_GRAD_COLUMNS || !known(dtype) || !dims_fit(tokens, inputs) ||
      !dims_fit(outputs, outputs))
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
  if (!dims_fit(tokens, inputs) || !dims_fit(outputs, outputs)) return fail(PLX_ERR_INVALID, "plx_mx_product: bad size");
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
  g.wide = g.sk == 1 && rows_on16(a, g.sm, dtype);
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
  if (!dims_fit(tokens, inputs) || !dims_fit(outputs, outputs)) return -1;
  return plan4_of(tokens, outputs, inputs).bytes;
}

int plx_mx4_product(int64_t tokens, int64_t inputs, int64_t outputs, const uint8_t* x_codes, const uint8_t* x_scales,
                    const uint8_t* w_codes, const uint8_t* w_scales, int32_t dtype, void* out, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  if (!dims_fit(tokens, inputs) || !dims_fit(outputs, outputs))
    return fail(PLX_ERR_INVALID, "plx_mx4_product: bad size");
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
    Big4Args g{};
    g.a = reinterpret_cast<const char*>(x_codes), g.b = reinterpret_cast<const char*>(w_codes);
    g.sa = reinterpret_cast<const uint4*>(work), g.sb = reinterpret_cast<const uint2*>(work + p.bytes_a);
    g.out = out, g.part = reinterpret_cast<float*>(work + p.bytes_a + p.bytes_b);
    g.M = static_cast<int>(tokens), g.N = static_cast<int>(outputs), g.line = blocks * 16;
    g.steps = p.steps, g.split = static_cast<int>(div_up(p.steps, p.splits));
    g.tiles_m = static_cast<int>(div_up(tokens, kBig)), g.tiles_n = static_cast<int>(div_up(outputs, kBig));
    const int64_t groups = div_up(p.bytes_a / 16 + p.bytes_b / 8, 256);
    k_big_scales<<<static_cast<unsigned>(groups < kMaxGroups ? groups : kMaxGroups), 256, 0, s>>>(
        g.M, g.N, blocks, p.steps, x_scales, w_scales, reinterpret_cast<uint8_t*>(work),
        reinterpret_cast<uint8_t*>(work + p.bytes_a));
    with_type(dtype, [&](auto* t) {
      using T = PLX_TYPE(t);
      const dim3 grid(static_cast<unsigned>(g.tiles_m) * g.tiles_n, static_cast<unsigned>(p.splits));
      k_big4_gemm<T><<<grid, kBigThreads, 0, s>>>(g);
      if (p.splits > 1) launch_join(tokens * outputs, p.splits, g.part, static_cast<T*>(out), s);
    });
    return check_launch("plx_mx4_product");
  }
  const int tiles_n = static_cast<int>(div_up(outputs, kTile));
  const int64_t rows = (kMaxGroups / tiles_n > 0 ? kMaxGroups / tiles_n : 1) * kTile;  // of one launch
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(dtype, [&](auto* t) {
    using T = PLX_TYPE(t);
    for (int64_t m = 0; m < tokens; m += rows) {
      const int64_t now = tokens - m < rows ? tokens - m : rows;
      k_mx4_gemm<T><<<static_cast<unsigned>(div_up(now, kTile) * tiles_n), 256, 0, s>>>(
          static_cast<int>(now), static_cast<int>(outputs), blocks, x_codes + m * blocks * 16, x_scales + m * blocks,
          w_codes, w_scales, static_cast<T*>(out) + m * outputs, tiles_n);
    }
  });
  return check_launch("plx_mx4_product");
}

}  // extern "C"
