// px_lowbit_gemm.h -- the large products of level pairs in few bits: operands
// as bf16 (or 4-bit) matrices in memory, copied straight into LDS.
#pragma once

#include <type_traits>

#include "px_lowbit.h"

namespace px {

// out[m][n] = sum over k of u(m, k) w(n, k): w from codes, in lines of k
// ("along": next to each other in memory), u the user's, in lines of k or of m
// ("across"). w is the side of whose rows a wave has more.
struct BigArgs {
  const char* w;
  const char* u;
  int64_t ldw, ldu;    // bytes of a line
  void* out;           // [M][N]
  float* part;         // [splits][M][N], where splits > 1
  int M, N;
  int rows_u;          // m that are in memory (M, or padded for "across")
  int wrap;            // steps of w's lines, 64 k each (256 in 4 bits), which start again with u's next piece
  int units;           // pieces of u that have units of their own (the others have one and follow each other)
  int steps;           // of u's lines in one unit
  float down[2];       // the first unit in the second one, and the second in the third
  const char* sw;      // 4 bits: the scales in the waves' order (k_big_scales)
  const char* su;
  int split;           // steps of one k range, in every unit
  int tiles_m, tiles_n;
};

constexpr int kBig = 256;              // rows and columns of a workgroup's tile
constexpr int kBigThreads = 512;
constexpr int kBigBytes = kBig * 128;     // of one operand's step in LDS

typedef __attribute__((address_space(3))) char lds_char;
typedef const __attribute__((address_space(1))) char glb_char;
typedef short s16x4 __attribute__((ext_vector_type(4)));

// One operand's step in LDS: two halves of 128 rows (of m or n), 16 KB each.
// Along: 128 lines of 8 chunks of 16 bytes, chunk c of line r at c ^ (r & 7).
// Across: 64 lines (k) of 16 chunks, pair p of line k at p ^ (k & 3 | k / 8 % 2
// * 4). A lane's loads are in LDS order (a wave's 64 lanes write 1 KB in a
// row), so the swizzle is in the global addresses: off[2 h + i] of half h.
template <bool ACROSS, bool F4 = false>
__device__ __forceinline__ void big_offsets(int tid, int first, int rows, int64_t ld, uint32_t off[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int slot = (i & 1) * kBigThreads + tid, half = i >> 1;
    if (ACROSS) {
      const int k = slot >> 4, cp = slot & 15;
      const int c = half * 16 + (((cp >> 1) ^ ((k & 3) | ((k >> 3) & 1) << 2)) << 1 | (cp & 1));
      const int last = (rows - first) / 8 - 1;  // (rows is a multiple of 8)
      off[i] = static_cast<uint32_t>(k * ld + (c < last ? c : last) * 16);
    } else {
      const int r = half * 128 + (slot >> 3), c = (slot & 7) ^ (r & 7) ^ (F4 ? (r >> 4) & 1 : 0);
      const int last = rows - first - 1;
      off[i] = static_cast<uint32_t>((r < last ? r : last) * ld + c * 16);
    }
  }
}

__device__ __forceinline__ void big_load(const char* base, const uint32_t* off, lds_char* lds, int wave) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    __builtin_amdgcn_global_load_lds((glb_char*)(base + off[i]),
                                     (__attribute__((address_space(3))) void*)(lds + (i * kBigThreads + wave * 64) * 16),
                                     16, 0, 0);
}

// LDS addresses of a lane's fragments of F x 16 rows from `row` of a half.
template <bool ACROSS, int F>
struct BigFrags {
  int at[ACROSS ? F : 2];
  __device__ __forceinline__ void init(int row, int l15, int q) {
    if (ACROSS) {
#pragma unroll
      for (int f = 0; f < F; ++f)
        at[f] = (q * 8 + (l15 >> 2)) * 256 + (((row >> 4) + f) ^ ((l15 >> 2) | (q & 1) << 2)) * 32 + (l15 & 3) * 8;
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = (row + l15) * 128 + ((s * 4 + q) ^ (l15 & 7)) * 16;
    }
  }
  __device__ __forceinline__ bf16x8 get(const lds_char* lds, int f, int s) const {
    if (ACROSS) {
      typedef __attribute__((address_space(3))) s16x4* p4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lds + at[f] + s * 8192));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lds + at[f] + s * 8192 + 1024));
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

// The same of the scaled 4-bit instruction, 32 rows by 64 k: a lane has row
// l & 31 and one block of a step's eight, 2 s + l / 32.
template <int F>
struct Big4Frags {
  int at[4];
  __device__ __forceinline__ void init(int row, int lane) {
#pragma unroll
    for (int s = 0; s < 4; ++s) at[s] = (row + (lane & 31)) * 128 + ((s * 2 + (lane >> 5)) ^ (lane & 7) ^ ((lane >> 4) & 1)) * 16;
  }
  __device__ __forceinline__ bf16x8 get(const lds_char* lds, int f, int s) const {
    return *reinterpret_cast<const __attribute__((address_space(3))) bf16x8*>(lds + at[s] + f * 4096);
  }
};

// The barrier between a wave's loads from LDS and its matrix instructions (the
// reads are back before it, so that others may overwrite what they read) and
// the one after those.
__device__ __forceinline__ void big_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// A wave's results, from its first row and column on: with w's rows as the
// matrix instruction's first operand a lane holds runs of four consecutive n
// of one m: one in a fragment of 16 x 16, in one of 32 x 32 four, 8 columns
// apart, lanes l and l + 32 having neighbouring runs of the same row. Rows are
// written 64 bytes and more at a time (32 left lines of 16-bit results that were
// written twice: 183 MB for 134). Tiles that are inside take the straight way.
template <typename T>
__device__ __forceinline__ void big_store(const f32x4 (&acc)[2][2][4][2], T* out, int M, int N, int m, int n,
                                          bool whole) {
#pragma unroll
  for (int hu = 0; hu < 2; ++hu)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = m + hu * 128 + j * 16;
      T* p = out + static_cast<int64_t>(row) * N + n;
      if (sizeof(T) == 2) {
        // Two fragments' runs, 32 columns: of lanes 16 apart the first gets 8
        // columns of the first fragment, the second 8 of the second one, so
        // that a row is written 64 bytes at a time.
        const int q = (threadIdx.x >> 4) & 3, to = (q & 1) * 16 + (q >> 1) * 8 - q * 4;
#pragma unroll
        for (int hw = 0; hw < 2; ++hw)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[hw][hu][i][j][k]),
                                                              __float_as_uint(acc[hw][hu][i + 1][j][k]), false, false);
              v[k] = __uint_as_float(t[0]), v[4 + k] = __uint_as_float(t[1]);
            }
            const int col = hw * 128 + i * 16 + to;
            if (whole)
              store8(p + col, 8, v);
            else if (row < M)
              store8(p + col, N - n - col, v);
          }
        continue;
      }
#pragma unroll
      for (int hw = 0; hw < 2; ++hw)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = hw * 128 + i * 16;
          if (whole)
            store4(p + col, 4, acc[hw][hu][i][j]);
          else if (row < M)
            store4(p + col, N - n - col, acc[hw][hu][i][j]);
        }
    }
}
template <typename T>
__device__ __forceinline__ void big_store(const f32x16 (&acc)[2][2][2][1], T* out, int M, int N, int m, int n,
                                          bool whole) {
  // Neighbouring runs of lanes 32 apart, then those of lanes 16 apart: a lane
  // gets 8 columns of rows l % 16 and l % 16 + 16, and a fragment's 32 columns
  // of a row are written at once.
  const int lane = threadIdx.x & 63, q = lane >> 4;
  const int row0 = m - (lane & 31) + (lane & 15), to = (q & 1) * 16 + (q >> 1) * 8 - (lane >> 5) * 4;
#pragma unroll
  for (int hu = 0; hu < 2; ++hu)
#pragma unroll
    for (int hw = 0; hw < 2; ++hw)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v[2][8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t r[2][2];  // runs 2 p and 2 p + 1 after the first exchange
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[hw][hu][i][0][8 * p + k]),
                                                            __float_as_uint(acc[hw][hu][i][0][8 * p + 4 + k]), false,
                                                            false);
            r[p][0] = t[0], r[p][1] = t[1];
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const auto t = __builtin_amdgcn_permlane16_swap(r[0][h], r[1][h], false, false);
            v[0][4 * h + k] = __uint_as_float(t[0]), v[1][4 * h + k] = __uint_as_float(t[1]);
          }
        }
        const int col = hw * 128 + i * 32 + to;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int row = row0 + hu * 128 + b * 16;
          T* p = out + static_cast<int64_t>(row) * N + n + col;
          if (whole)
            store8(p, 8, v[b]);
          else if (row < M)
            store8(p, N - n - col, v[b]);
        }
      }
}

// 256 x 256 of the output by 8 waves. A wave has 64 rows in each half of its w
// and 32 in each half of u, so four quarters of 64 x 32, one a phase: LDS
// reads and global loads, barrier, 16 matrix instructions, barrier. The second
// four waves are one barrier behind the first, so that on each SIMD one wave
// multiplies while the other one loads. A half of a buffer is loaded for the
// step after next as soon as both have read it, nearly two steps before it is
// needed. bf16 8192 cubed 702 us on average, 1570 TFLOP/s; 8192 x 4096 x 4096
// 214 (184 at least), matrix cores 77 % busy (two buffers and one barrier a step:
// 58 %, 270 us). F4: both operands in 4-bit blocks along k, 8 of them in a line's 128
// bytes: a lane's 16 bytes are one block, and the LDS layout is the bf16 one.
// The scales of a step come in the waves' order (k_big_scales) and by way of
// LDS too, a lane's own in 16 and 8 bytes (8192 cubed 242 us; read by each lane
// for itself, every load under way would be waited for first).
template <bool UA, bool F4, typename OT>
__global__ __launch_bounds__(kBigThreads, 2) void k_big_gemm(BigArgs g) {
  __shared__ __align__(16) char lds[4 * kBigBytes + (F4 ? 2 * 4096 : 0)];
  lds_char* l = (lds_char*)lds;
  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), ww = wave >> 2, wu = wave & 3;
  int tm, tn;
  big_tile(blockIdx.x, g.tiles_m, g.tiles_n, &tm, &tn);
  const int m0 = tm * kBig, n0 = tn * kBig;

  uint32_t ow[4], ou[4];
  big_offsets<false, F4>(tid, n0, g.N, g.ldw, ow);
  big_offsets<UA, F4>(tid, m0, g.rows_u, g.ldu, ou);
  const int64_t su = UA ? 64 * g.ldu : 128;
  const int beg = blockIdx.y * g.split, end = beg + g.split < g.steps ? beg + g.split : g.steps;
  const int count = F4 ? end - beg : (end - beg) * g.units;
  const char* w = g.w + n0 * g.ldw;
  const char* u = g.u + (UA ? int64_t{2} * m0 : m0 * g.ldu) + beg * su;
  // Where w's steps start again, after which one, and u's way to its next piece.
  const bool alone = F4 || g.units == 1;
  const int again = alone ? 0 : beg, last = (alone ? g.wrap : end) - 1;
  const int64_t next_piece = alone ? su : (g.steps - last + again) * su;
  int wt = alone ? beg % g.wrap : beg;
  // 4 bits: a line of an odd number of 64 bytes ends inside its last step,
  // which then reads its first half twice and multiplies it once.
  const bool odd = F4 && (g.ldw & 64) != 0;
  const uint32_t back = (((tid & 7) ^ ((tid >> 3) & 7) ^ ((tid >> 7) & 1)) & 4) ? 64 : 0;
  // 4 KB of scales a step, by the first four waves: w's, then u's.
  const char* gs = nullptr;
  u32x4 ws = {};
  u32x2 us = {};
  if (F4)
    gs = (wave < 2 ? g.sw + (static_cast<int64_t>(tn) * g.steps + beg) * 2048
                   : g.su + (static_cast<int64_t>(tm) * g.steps + beg) * 2048) +
         (wave & 1) * 1024 + lane * 16;

  // Fragments: 16 rows by 32 k, or 32 rows by 64 k of 4 bits; of either a
  // quarter's 64 x 32 take FW x FU, in S steps of k.
  constexpr int FW = F4 ? 2 : 4, FU = F4 ? 1 : 2, S = F4 ? 4 : 2;
  typedef typename std::conditional<F4, f32x16, f32x4>::type sums;
  typename std::conditional<F4, Big4Frags<FW>, BigFrags<false, FW>>::type fw;
  typename std::conditional<F4, Big4Frags<FU>, BigFrags<UA, FU>>::type fu;
  if constexpr (F4) {
    fw.init(ww * 64, lane);
    fu.init(wu * 32, lane);
  } else {
    fw.init(ww * 64, l15, q);
    fu.init(wu * 32, l15, q);
  }
  sums acc[2][2][FW][FU] = {};
  bf16x8 rw[FW][S], ru[2][FU][S];

  // A step's four loads, of w's and u's first halves, u's and w's second ones;
  // the last of them moves on to the next step.
  auto load_w0u0 = [&](int buf) {
    if (odd && wt + 1 == g.wrap) {
#pragma unroll
      for (int i = 0; i < 4; ++i) ow[i] -= back, ou[i] -= back;
    }
    big_load(w + static_cast<int64_t>(wt) * 128, ow, l + buf * 2 * kBigBytes, wave);
    big_load(u, ou, l + buf * 2 * kBigBytes + kBigBytes, wave);
  };
  auto load_u1 = [&](int buf) { big_load(u, ou + 2, l + buf * 2 * kBigBytes + kBigBytes + kBigBytes / 2, wave); };
  auto load_w1 = [&](int buf) {
    big_load(w + static_cast<int64_t>(wt) * 128, ow + 2, l + buf * 2 * kBigBytes + kBigBytes / 2, wave);
    if (F4 && wave < 4) {
      __builtin_amdgcn_global_load_lds(
          (glb_char*)gs, (__attribute__((address_space(3))) void*)(l + 4 * kBigBytes + buf * 4096 + wave * 1024), 16, 0, 0);
      gs += 2048;
    }
    const bool over = wt == last;
    u += over ? next_piece : su;
    wt = over ? again : wt + 1;
  };
  auto read_w = [&](int buf, int h) {
    const lds_char* p = l + buf * 2 * kBigBytes + h * (kBigBytes / 2);
#pragma unroll
    for (int i = 0; i < FW; ++i)
#pragma unroll
      for (int s = 0; s < S; ++s) rw[i][s] = fw.get(p, i, s);
  };
  auto read_u = [&](int buf, auto half) {
    constexpr int h = decltype(half)::value;
    const lds_char* p = l + buf * 2 * kBigBytes + kBigBytes + h * (kBigBytes / 2);
#pragma unroll
    for (int i = 0; i < FU; ++i)
#pragma unroll
      for (int s = 0; s < S; ++s) ru[h][i][s] = fu.get(p, i, s);
  };
  auto multiply = [&](auto half_w, auto half_u, bool both) {
    constexpr int hw = decltype(half_w)::value, hu = decltype(half_u)::value;
    __builtin_amdgcn_s_setprio(1);
    if constexpr (F4) {
#define PX_F4(i, s)                                                                                            \
  acc[hw][hu][i][0] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(                                         \
      as_i32x8(rw[i][s]), as_i32x8(ru[hu][0][s]), acc[hw][hu][i][0], 4, 4, s,                                  \
      static_cast<int>(ws[hw * 2 + (i)]), s, static_cast<int>(us[hu]))
      PX_F4(0, 0), PX_F4(1, 0), PX_F4(0, 1), PX_F4(1, 1);
      if (both) PX_F4(0, 2), PX_F4(1, 2), PX_F4(0, 3), PX_F4(1, 3);
#undef PX_F4
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            acc[hw][hu][i][j] =
                __builtin_amdgcn_mfma_f32_16x16x32_bf16(rw[i][s], ru[hu][j][s], acc[hw][hu][i][j], 0, 0, 0);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  constexpr std::integral_constant<int, 0> k0{};
  constexpr std::integral_constant<int, 1> k1{};

  // All but the newest step's loads are back.
  auto wait_older = [&]() {
    if (F4 && wave < 4)
      asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
    else
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
  };
  load_w0u0(0);
  load_u1(0);
  load_w1(0);
  if (count > 1) {
    load_w0u0(1);
    load_u1(1);
    load_w1(1);
    wait_older();
  } else {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  big_barrier();
  if (ww) big_barrier();
  auto step = [&](int t) {
    const int buf = t & 1;
    const bool more = t + 2 < count, both = !(odd && beg + t + 1 == g.steps);
    read_u(buf, k0);
    read_w(buf, 0);
    if (F4) {
      const lds_char* p = l + 4 * kBigBytes + buf * 4096;
      // (Written out, and waited for in place: the compiler would wait for
      // every load under way before it.)
      asm volatile(
          "ds_read_b128 %0, %2\n\tds_read_b64 %1, %3 offset:2048\n\ts_waitcnt lgkmcnt(0)"
          : "=&v"(ws), "=&v"(us)
          : "v"(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p + ww * 1024 + lane * 16))),
            "v"(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p + wu * 512 + lane * 8)))
          : "memory");
    }
    big_barrier();
    multiply(k0, k0, both);
    big_barrier();
    read_u(buf, k1);
    if (more) load_w0u0(buf);
    big_barrier();
    multiply(k0, k1, both);
    big_barrier();
    read_w(buf, 1);
    if (more) load_u1(buf);
    big_barrier();
    multiply(k1, k1, both);
    big_barrier();
    if (more) {
      load_w1(buf);
      wait_older();
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    big_barrier();
    multiply(k1, k0, both);
    big_barrier();
  };
  // At the end of a piece the sums change to the next one's unit.
  int left = end - beg, piece = 0;
  for (int t = 0; t < count; ++t) {
    step(t);
    if (!F4 && --left == 0 && t + 1 < count) {
      const float by = g.down[piece++];
      left = end - beg;
#pragma unroll
      for (int hw = 0; hw < 2; ++hw)
#pragma unroll
        for (int hu = 0; hu < 2; ++hu)
#pragma unroll
          for (int i = 0; i < FW; ++i)
#pragma unroll
            for (int j = 0; j < FU; ++j) acc[hw][hu][i][j] *= by;
    }
  }
  if (!ww) big_barrier();

  const int m = m0 + wu * 32 + (F4 ? lane & 31 : l15), n = n0 + ww * 64 + (F4 ? (lane >> 5) * 4 : q * 4);
  const bool whole = m0 + kBig <= g.M && n0 + kBig <= g.N;
  if (gridDim.y > 1)
    big_store(acc, g.part + static_cast<int64_t>(blockIdx.y) * g.M * g.N, g.M, g.N, m, n, false);
  else if (whole)
    big_store(acc, static_cast<OT*>(g.out), g.M, g.N, m, n, true);
  else
    big_store(acc, static_cast<OT*>(g.out), g.M, g.N, m, n, false);
}

// Scale bytes [rows][blocks] as the waves of k_big_gemm read them: W waves
// share a tile's 256 rows, each with F fragments of 32 rows in each half. Of
// tile, step, wave and lane, byte 4 (F h + f) + s is the scale of row
// 128 h + 32 (F wave + f) + lane % 32 in block 8 step + 2 s + lane / 32. Rows
// past the end and blocks that hold no values (from `used` on) get the scale 1. A workgroup takes 8 steps of a tile
// through LDS (two of 8192 x 8192 values 8 us).
typedef uint32_t u32_any __attribute__((aligned(1)));  // (scale bytes start anywhere)
constexpr int kScaleRow = 68;  // bytes of 8 steps of a row in LDS, and 4 that move the rows over the banks
template <int F>
__device__ __forceinline__ void big_scales(int tile, int step0, int steps, int rows, int64_t blocks, int64_t used,
                                           const uint8_t* in, uint8_t* out, uint8_t* lds) {
  constexpr int W = 4 / F;
  const int tid = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int at = i * 256 + tid, r = at >> 4, c = (at & 15) * 4;
    const int row = tile * 256 + r;
    uint32_t v = 0x7F7F7F7Fu;
    const int64_t left = used - (int64_t{8} * step0 + c);
    if (row < rows && left > 0) {
      const uint32_t keep = left < 4 ? (1u << (8 * left)) - 1u : ~0u;
      v = (*reinterpret_cast<const u32_any*>(in + row * blocks + int64_t{8} * step0 + c) & keep) | (v & ~keep);
    }
    *reinterpret_cast<uint32_t*>(lds + r * kScaleRow + c) = v;
  }
  __syncthreads();
  for (int at = tid; at < 8 * W * 64; at += 256) {
    const int step = at / (W * 64), wave = at / 64 % W, lane = at & 63;
    if (step0 + step >= steps) break;
    uint32_t* o = reinterpret_cast<uint32_t*>(out) + ((static_cast<int64_t>(tile) * steps + step0) * W * 64 + at) * 2 * F;
#pragma unroll
    for (int f = 0; f < 2 * F; ++f) {
      const int row = f / F * 128 + (wave * F + f % F) * 32 + (lane & 31);
      const uint8_t* p = lds + row * kScaleRow + step * 8 + (lane >> 5);
      o[f] = p[0] | p[2] << 8 | p[4] << 16 | static_cast<uint32_t>(p[6]) << 24;
    }
  }
}

__global__ __launch_bounds__(256) void k_big_scales(int N, int M, int64_t blocks, int64_t used, int steps,
                                                    const uint8_t* ws, const uint8_t* us, uint8_t* sw, uint8_t* su) {
  __shared__ uint8_t lds[256 * kScaleRow];
  const int runs = (steps + 7) / 8, tile = blockIdx.x / runs, step0 = blockIdx.x % runs * 8, tiles_n = (N + 255) / 256;
  if (tile < tiles_n)
    big_scales<2>(tile, step0, steps, N, blocks, used, ws, sw, lds);
  else
    big_scales<1>(tile - tiles_n, step0, steps, M, blocks, used, us, su, lds);
}

// Codes as bf16 lines of k for k_big_gemm, kp values each.
struct BigValues {
  int64_t lines, n, blocks;  // of the codes
  const uint8_t* codes;
  const uint8_t* scales;
  uint16_t* out;
  int64_t kp;
  int tiles_n;  // turned
  int lx;       // not turned: lanes beside each other along a line
};

// The first `left` of 8 codes from the at-th eight on, as bf16 (in 4 bits the
// codes behind a line's end are zeros).
template <int BITS>
__device__ __forceinline__ uint4 bf16_unit(const uint8_t* codes, const uint8_t* scales, int64_t at, int64_t left = 8) {
  const float scale = scale_value(scales[at / 4]);
  return BITS == 4 ? bf16_of4(reinterpret_cast<const uint32_t*>(codes)[at], scale)
                   : bf16_of8(first_codes8(reinterpret_cast<const uint2*>(codes)[at], left), scale);
}

// Lines of k: line by line, zeros behind their ends.
template <int BITS>
__device__ __forceinline__ void big_values(const BigValues& g, int64_t group, int64_t groups) {
  const int tx = threadIdx.x & (g.lx - 1), ly = 256 / g.lx, ty = threadIdx.x / g.lx;
  for (int64_t line = group * ly + ty; line < g.lines; line += groups * ly)
    for (int64_t c = tx; c < g.kp / 8; c += g.lx) {
      uint4 r = make_uint4(0, 0, 0, 0);
      if (c * 8 < g.n) r = bf16_unit<BITS>(g.codes, g.scales, line * g.blocks * 4 + c, g.n - c * 8);
      *reinterpret_cast<uint4*>(g.out + line * g.kp + c * 8) = r;
    }
}

// Lines across, each of one k: 64 k by 128 n go through LDS in k_big_gemm's
// layout and come back transposed. k past the lines are zeros.
template <int BITS>
__device__ __forceinline__ void big_turned(const BigValues& g, int64_t group, char* lds) {
  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, q = lane >> 4, wave = tid >> 6;
  const int64_t k0 = group / g.tiles_n * 64, n0 = group % g.tiles_n * 128;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int u = i * 256 + tid, line = u >> 4, c = u & 15;
    const int64_t pos = n0 + c * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (k0 + line < g.lines && pos < g.blocks * 32)
      v = bf16_unit<BITS>(g.codes, g.scales, (k0 + line) * g.blocks * 4 + pos / 8);
    *reinterpret_cast<uint4*>(lds + line * 256 + ((c >> 1) ^ ((line & 3) | ((line >> 3) & 1) << 2)) * 32 + (c & 1) * 16) = v;
  }
  __syncthreads();
  BigFrags<true, 2> f;
  f.init(wave * 32, l15, q);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t row = n0 + wave * 32 + i * 16 + l15;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bf16x8 v = f.get((const lds_char*)lds, i, s);
      if (row < g.n) *reinterpret_cast<bf16x8*>(g.out + row * g.kp + k0 + s * 32 + q * 8) = v;
    }
  }
}

// The user's operand as bf16 pieces in padded lines: piece p of line l at
// out + (P - 1 - p) * piece + l * out_line. k goes over the least pieces first:
// added to the sums of the largest ones they would be rounded off one by one.
struct BigPieces {
  const void* x;
  int64_t lines, n, sl, se;  // elements of line l at l * sl + i * se
  uint16_t* out;
  int64_t out_lines, out_n, out_line, piece;
  int lx;
};
template <typename T>
__device__ __forceinline__ void big_pieces(const BigPieces& g, int64_t group, int64_t groups) {
  constexpr int P = Pieces<T>::n;
  const T* x = static_cast<const T*>(g.x);
  const int tx = threadIdx.x & (g.lx - 1), ly = 256 / g.lx, ty = threadIdx.x / g.lx;
  for (int64_t line = group * ly + ty; line < g.out_lines; line += groups * ly)
    for (int64_t c = tx; c < g.out_n / 8; c += g.lx) {
      const int64_t left = line < g.lines ? g.n - c * 8 : 0;
      float v[8];
      load8(x + line * g.sl + c * 8 * g.se, g.se, left > 8 ? 8 : left < 0 ? 0 : static_cast<int>(left), v);
      uint4 p[P];
      pieces8<P>(v, p);
#pragma unroll
      for (int i = 0; i < P; ++i)
        *reinterpret_cast<uint4*>(g.out + (P - 1 - i) * g.piece + line * g.out_line + c * 8) = p[i];
    }
}

// Both operands of a large product in one launch, at the rate of memory (4096
// x 8192 codes of 8 bits turned 20 us, 101 MB): the first `groups`
// workgroups make w, the others u (none where it is taken as it is).
template <typename T, int BITS, bool TURNED>
__global__ __launch_bounds__(256) void k_big_operands(BigValues w, BigPieces u, unsigned groups) {
  __shared__ __align__(16) char lds[TURNED ? 64 * 256 : 16];
  if (blockIdx.x >= groups)
    big_pieces<T>(u, blockIdx.x - groups, gridDim.x - groups);
  else if (TURNED)
    big_turned<BITS>(w, blockIdx.x, lds);
  else
    big_values<BITS>(w, blockIdx.x, groups);
}

}  // namespace px
