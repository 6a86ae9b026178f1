// px_lowbit_gemm.h -- the large products of level pairs in few bits: operands
// as bf16 (or 4-bit) matrices in memory, copied straight into LDS.
#pragma once

#include <type_traits>

#include "px_lowbit.h"

namespace px {

// out[m][n] = sum over k of a(m, k) b(n, k). An operand is kept "along" (rows
// of k next to each other) or "across" (rows of m or n, one for each k).
struct BigArgs {
  const char* a;
  const char* b;
  int64_t lda, ldb;  // bytes of a row
  void* out;         // [M][N]
  float* part;       // [splits][M][N], where splits > 1
  int M, N;
  int rows_a, rows_b;  // m and n that are in memory (M and N, or padded for "across")
  int steps;         // of 64 k, over all of a's pieces
  int wrap;          // steps of b, which starts again after them
  int split;         // steps of one k range
  int tiles_m, tiles_n;
};

constexpr int kBig = 256;                 // rows and columns of a workgroup's tile
constexpr int kBigThreads = 512;
constexpr int kBigBytes = kBig * 128;     // of one operand's step in LDS

typedef __attribute__((address_space(3))) char lds_char;
typedef const __attribute__((address_space(1))) char glb_char;

// The four 16-byte loads of a lane for one operand's step, in LDS order (a
// wave's 64 lanes write 1 KB in a row), so that the swizzle is in the global
// addresses. Along: 256 rows of 8 chunks, chunk c of row r at c ^ (r & 7).
// Across: 64 rows (k) of 32 chunks, pair p of row k at p ^ (k & 3 | k / 8 % 4 * 4).
template <bool ACROSS>
__device__ __forceinline__ void big_offsets(int tid, int first, int rows, int64_t ld, uint32_t off[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int slot = i * kBigThreads + tid;
    if (ACROSS) {
      const int k = slot >> 5, cp = slot & 31;
      const int c = ((cp >> 1) ^ ((k & 3) | ((k >> 3) & 3) << 2)) << 1 | (cp & 1);
      const int last = (rows - first) / 8 - 1;  // (rows is a multiple of 8)
      off[i] = static_cast<uint32_t>(k * ld + (c < last ? c : last) * 16);
    } else {
      const int r = slot >> 3, c = (slot & 7) ^ (r & 7);
      const int last = rows - first - 1;
      off[i] = static_cast<uint32_t>((r < last ? r : last) * ld + c * 16);
    }
  }
}

__device__ __forceinline__ void big_load(const char* base, const uint32_t off[4], lds_char* lds, int wave) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    __builtin_amdgcn_global_load_lds((glb_char*)(base + off[i]),
                                     (__attribute__((address_space(3))) void*)(lds + (i * kBigThreads + wave * 64) * 16),
                                     16, 0, 0);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// LDS addresses of a lane's fragments of F x 16 rows from `row`.
template <bool ACROSS, int F>
struct BigFrags {
  int at[ACROSS ? F : 2];
  __device__ __forceinline__ void init(int row, int l15, int q) {
    if (ACROSS) {
#pragma unroll
      for (int f = 0; f < F; ++f)
        at[f] = (q * 8 + (l15 >> 2)) * 512 + (((row >> 4) + f) ^ ((l15 >> 2) | q << 2)) * 32 + (l15 & 3) * 8;
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = (row + l15) * 128 + ((s * 4 + q) ^ (l15 & 7)) * 16;
    }
  }
  __device__ __forceinline__ bf16x8 get(const lds_char* lds, int f, int s) const {
    if (ACROSS) {
      typedef __attribute__((address_space(3))) s16x4* p4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lds + at[f] + s * 16384));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lds + at[f] + s * 16384 + 2048));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return *reinterpret_cast<const __attribute__((address_space(3))) bf16x8*>(lds + at[s] + f * 2048);
  }
};

// Which tile a workgroup takes: workgroups go round the 8 XCDs, each of which
// takes a run of tiles of its own, in strips of 8 tile rows, so that its L2
// holds the rows and columns that its workgroups share.
__device__ __forceinline__ void big_tile(int wg, int tiles_m, int tiles_n, int* tm, int* tn) {
  const int n = tiles_m * tiles_n;
  const int per = n / 8, rest = n % 8, x = wg & 7, j = wg >> 3;
  const int t = x * per + (x < rest ? x : rest) + j;
  const int strip = 8 * tiles_n, g = t / strip, r = t - g * strip;
  const int high = tiles_m - g * 8 < 8 ? tiles_m - g * 8 : 8;
  *tm = g * 8 + r % high;
  *tn = r / high;
}

// A wave's 128 x 64 results: with b's rows as the matrix instruction's first
// operand a lane holds four consecutive n of one m.
template <typename OT>
__device__ __forceinline__ void big_store(const f32x4 acc[8][4], void* out, float* part, int M, int N, int m0, int n0) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int m = m0 + i * 16;
    if (m >= M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + j * 16;
      const int64_t at = static_cast<int64_t>(m) * N + n;
      if (gridDim.y > 1)
        store4(part + static_cast<int64_t>(blockIdx.y) * M * N + at, N - n, acc[i][j]);
      else
        store4(static_cast<OT*>(out) + at, N - n, acc[i][j]);
    }
  }
}

template <bool AA, bool BA, typename OT>
__global__ __launch_bounds__(kBigThreads, 2) void k_big_gemm(BigArgs g) {
  __shared__ __align__(16) char lds[4 * kBigBytes];
  lds_char* l = (lds_char*)lds;
  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tm, tn;
  big_tile(blockIdx.x, g.tiles_m, g.tiles_n, &tm, &tn);
  const int m0 = tm * kBig, n0 = tn * kBig, wm = (wave >> 2) * 128, wn = (wave & 3) * 64;

  uint32_t oa[4], ob[4];
  big_offsets<AA>(tid, m0, g.rows_a, g.lda, oa);
  big_offsets<BA>(tid, n0, g.rows_b, g.ldb, ob);
  const int64_t sa = AA ? 64 * g.lda : 128, sb = BA ? 64 * g.ldb : 128;
  const char* a = g.a + (AA ? int64_t{2} * m0 : m0 * g.lda);
  const char* b = g.b + (BA ? int64_t{2} * n0 : n0 * g.ldb);
  const int beg = blockIdx.y * g.split, end = beg + g.split < g.steps ? beg + g.split : g.steps;
  int bt = beg % g.wrap;
  a += beg * sa;

  BigFrags<AA, 8> fa;
  BigFrags<BA, 4> fb;
  fa.init(wm, l15, q);
  fb.init(wn, l15, q);

  f32x4 acc[8][4] = {};
  auto load = [&](int buf) {
    big_load(a, oa, l + buf * 2 * kBigBytes, wave);
    big_load(b + bt * sb, ob, l + buf * 2 * kBigBytes + kBigBytes, wave);
    a += sa;
    bt = bt + 1 == g.wrap ? 0 : bt + 1;
  };
  auto compute = [&](int buf) {
    const lds_char* la = l + buf * 2 * kBigBytes;
    const lds_char* lb = la + kBigBytes;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 xb[4], xa[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) xb[i] = fb.get(lb, i, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) xa[i] = fa.get(la, i, s);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb[j], xa[i], acc[i][j], 0, 0, 0);
    }
  };
  load(0);
  int buf = 0;
  for (int t = beg; t < end; ++t) {
    __syncthreads();
    if (t + 1 < end) load(buf ^ 1);
    compute(buf);
    buf ^= 1;
  }

  big_store<OT>(acc, g.out, g.part, g.M, g.N, m0 + wm + l15, n0 + wn + q * 4);
}

// The same with both operands in 4-bit blocks along k: a row's 128 bytes are
// 8 blocks, and a lane's 16 bytes one of them with its scale byte, so that
// the LDS layout and the fragments' addresses are the bf16 kernel's. A wave
// finds the scales of its rows' blocks of a step side by side in `sa` and
// `sb` (k_big_scales), a lane's own in 16 and 8 bytes.
struct Big4Args {
  const char* a;
  const char* b;
  const uint4* sa;  // [ceil(M / 128)][steps][64]
  const uint2* sb;  // [ceil(N / 64)][steps][64]
  void* out;
  float* part;
  int M, N;
  int64_t line;  // bytes of a row, a multiple of 64
  int steps, split, tiles_m, tiles_n;
};

template <int I>
__device__ __forceinline__ uint32_t word(uint4 v) {
  return I == 0 ? v.x : I == 1 ? v.y : I == 2 ? v.z : v.w;
}

template <typename OT>
__global__ __launch_bounds__(kBigThreads, 2) void k_big4_gemm(Big4Args g) {
  __shared__ __align__(16) char lds[4 * kBigBytes];
  lds_char* l = (lds_char*)lds;
  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tm, tn;
  big_tile(blockIdx.x, g.tiles_m, g.tiles_n, &tm, &tn);
  const int m0 = tm * kBig, n0 = tn * kBig, wm = (wave >> 2) * 128, wn = (wave & 3) * 64;

  uint32_t oa[4], ob[4];
  big_offsets<false>(tid, m0, g.M, g.line, oa);
  big_offsets<false>(tid, n0, g.N, g.line, ob);
  const int beg = blockIdx.y * g.split, end = beg + g.split < g.steps ? beg + g.split : g.steps;
  const char* a = g.a + m0 * g.line + beg * 128;
  const char* b = g.b + n0 * g.line + beg * 128;
  // A line of an odd number of 64 bytes ends inside its last step, which then
  // reads its first half twice and multiplies it once.
  const bool odd = (g.line & 64) != 0;
  const uint32_t back = (((tid & 7) ^ ((tid >> 3) & 7)) & 4) ? 64 : 0;
  // (a wave past the last rows reads the last ones' scales)
  const int ga = (m0 + wm) / 128, gb = (n0 + wn) / 64, la = (g.M - 1) / 128, lb = (g.N - 1) / 64;
  const uint4* sa = g.sa + (static_cast<int64_t>(ga < la ? ga : la) * g.steps + beg) * 64 + lane;
  const uint2* sb = g.sb + (static_cast<int64_t>(gb < lb ? gb : lb) * g.steps + beg) * 64 + lane;

  BigFrags<false, 8> fa;
  BigFrags<false, 4> fb;
  fa.init(wm, l15, q);
  fb.init(wn, l15, q);

  f32x4 acc[8][4] = {};
  uint4 xs = make_uint4(0, 0, 0, 0);
  uint2 ws = make_uint2(0, 0);
  auto load = [&](int t, int buf) {
    if (odd && t + 1 == g.steps) {
#pragma unroll
      for (int i = 0; i < 4; ++i) oa[i] -= back, ob[i] -= back;
    }
    big_load(a, oa, l + buf * 2 * kBigBytes, wave);
    big_load(b, ob, l + buf * 2 * kBigBytes + kBigBytes, wave);
    a += 128, b += 128;
    xs = *sa, ws = *sb;
    sa += 64, sb += 64;
  };
  auto half = [&](int buf, auto step, uint4 s_a, uint2 s_b) {
    constexpr int s = decltype(step)::value;
    const lds_char* pa = l + buf * 2 * kBigBytes;
    const lds_char* pb = pa + kBigBytes;
    i32x8 xb[4], xa[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) xb[i] = as_i32x8(fb.get(pb, i, s));
#pragma unroll
    for (int i = 0; i < 8; ++i) xa[i] = as_i32x8(fa.get(pa, i, s));
#define PX_BIG4_MFMA(i, j)                                                                          \
  acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(                                     \
      xb[j], xa[i], acc[i][j], 4, 4, ((j) * 2 + s) & 3, static_cast<int>((j) < 2 ? s_b.x : s_b.y),  \
      ((i) * 2 + s) & 3, static_cast<int>(word<(i) / 2>(s_a)))
#define PX_BIG4_ROW(i) PX_BIG4_MFMA(i, 0), PX_BIG4_MFMA(i, 1), PX_BIG4_MFMA(i, 2), PX_BIG4_MFMA(i, 3)
    PX_BIG4_ROW(0), PX_BIG4_ROW(1), PX_BIG4_ROW(2), PX_BIG4_ROW(3);
    PX_BIG4_ROW(4), PX_BIG4_ROW(5), PX_BIG4_ROW(6), PX_BIG4_ROW(7);
#undef PX_BIG4_ROW
#undef PX_BIG4_MFMA
  };
  load(beg, 0);
  int buf = 0;
  for (int t = beg; t < end; ++t) {
    const uint4 s_a = xs;
    const uint2 s_b = ws;
    __syncthreads();
    if (t + 1 < end) load(t + 1, buf ^ 1);
    half(buf, std::integral_constant<int, 0>{}, s_a, s_b);
    if (!(odd && t + 1 == g.steps)) half(buf, std::integral_constant<int, 1>{}, s_a, s_b);
    buf ^= 1;
  }
  big_store<OT>(acc, g.out, g.part, g.M, g.N, m0 + wm + l15, n0 + wn + q * 4);
}

// Scale bytes [rows][blocks] as k_big4_gemm reads them: of group r / (16 F),
// step and lane (l15, q), byte 2 f + s is row 16 f + l15's block 8 step + 4 s
// + q. Rows and blocks past the end get the scale 1.
template <int F>
__device__ __forceinline__ void big_scales(int64_t at, int rows, int64_t blocks, int steps, const uint8_t* in,
                                           uint8_t* out) {
  const int lane = at & 63;
  const int64_t w = at >> 6;
  const int step = static_cast<int>(w % steps), group = static_cast<int>(w / steps);
  const int64_t b = int64_t{8} * step + (lane >> 4);
  uint32_t r[F / 2];
#pragma unroll
  for (int i = 0; i < F / 2; ++i) r[i] = 0;
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int row = group * 16 * F + f * 16 + (lane & 15);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t v = row < rows && b + 4 * s < blocks ? in[row * blocks + b + 4 * s] : 127u;
      r[f / 2] |= v << (8 * ((f * 2 + s) & 3));
    }
  }
  uint32_t* o = reinterpret_cast<uint32_t*>(out) + at * (F / 2);
#pragma unroll
  for (int i = 0; i < F / 2; ++i) o[i] = r[i];
}

__global__ __launch_bounds__(256) void k_big_scales(int M, int N, int64_t blocks, int steps, const uint8_t* xs,
                                                    const uint8_t* ws, uint8_t* sa, uint8_t* sb) {
  const int64_t na = static_cast<int64_t>((M + 127) / 128) * steps * 64;
  const int64_t nb = static_cast<int64_t>((N + 63) / 64) * steps * 64;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < na + nb;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    if (i < na)
      big_scales<8>(i, M, blocks, steps, xs, sa);
    else
      big_scales<4>(i - na, N, blocks, steps, ws, sb);
  }
}

}  // namespace px
