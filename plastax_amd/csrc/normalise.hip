// normalise.hip -- layer norm of what goes from one level pair to the next,
// and its gradients. No counterpart in the reference.
//
// Over a token's units: n = (x - mean) r, r = 1 / sqrt(var + eps),
// y = n w + b. With u = g w: dx = r (u - mean(u) - n mean(u n)); dw and db are
// the sums of g n and g over the tokens, by workgroup and then over the
// workgroups, always in the same order.
//
// Bound by memory: a row stays in registers, so that x (and g) are read once
// and y (dx) written once. 16384 x 4096 bf16: 54 us forwards, 5.0 TB/s; the
// gradients 79, 5.1 TB/s, and 4 for the join of dw and db. A row has as many
// waves as hold it with a chunk of 16 bytes a lane, up to 16 waves, then up to
// 4 chunks; several rows share a workgroup. Levels that fill 64 2^k lanes in part
// leave the others idle: 47072 x 1425 bf16 (179 chunks, 256 lanes) 58 us and 108,
// 4.6 and 3.7 TB/s.

#include "px_dense.h"

using plx_detail::check_launch;
using plx_detail::cu_count;
using plx_detail::fail;

namespace {

using namespace px;

constexpr int kRows = 4;  // rows that a group of waves takes at a time, forwards

struct NormArgs {
  int64_t tokens, x_line, g_line;
  int units;
  float eps;
  const void* x;
  const void* g;
  const void* weight;
  const void* bias;
  void* y;       // or dx
  float* kept;   // [tokens][2]: mean, r
  float* part;   // [workgroups][2][units]
};

// N sums over the WAVES waves that share rows. One barrier: the next sums take
// another `part`.
template <int WAVES, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*part)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if (WAVES == 1) return;
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) part[wave][i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = part[wave / WAVES * WAVES + (threadIdx.x & (WAVES - 1))][i];
#pragma unroll
    for (int d = 1; d < WAVES; d *= 2) v[i] += __shfl_xor(v[i], d, 64);
  }
}

template <int WAVES>
__device__ __forceinline__ float row_sum(float v, float (*part)[1]) {
  float sums[1] = {v};
  row_sums<WAVES>(sums, part);
  return sums[0];
}

// sum / units, inv = 1 / units: a product with the rounding of inv taken out
// again, so that a row of one value has it for its mean.
__device__ __forceinline__ float mean_of(float sum, float units, float inv) {
  const float m = sum * inv;
  return __builtin_fmaf(__builtin_fmaf(-m, units, sum), inv, m);
}

// R rows' chunks at `at`, one branch for all of them.
template <int R, typename T>
__device__ __forceinline__ void load_rows(const T* const (&row)[R], int at, int units,
                                          typename Pack<T, kChunk<T>>::type (&v)[R]) {
  constexpr int W = kChunk<T>;
  if (at + W <= units) {
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = *reinterpret_cast<const typename Pack<T, W>::load*>(row[r] + at);
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = load_pack<W>(row[r] + at, units - at);
  }
}

// ROWS groups of WAVES waves, NC chunks of 16 bytes a lane. A group takes R
// rows at a time, for which it waits once, and goes on to gridDim.x * ROWS * R
// rows further: a lane's weights stay in registers. The variance is the mean of
// the squares of x - mean, from registers.
template <typename T, typename P, int ROWS, int WAVES, int NC, int R>
__global__ __launch_bounds__(ROWS* WAVES * 64) void k_normalise(NormArgs a) {
  constexpr int W = kChunk<T>, NT = WAVES * 64;
  __shared__ float part[2][ROWS * WAVES][R];
  const int lane = threadIdx.x % NT;
  const float units = static_cast<float>(a.units), inv = 1.0f / units;
  float w[NC][W], b[NC][W];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int at = (k * NT + lane) * W;
    const typename Pack<P, W>::type p = load_pack<W>(static_cast<const P*>(a.weight) + at, a.units - at);
#pragma unroll
    for (int i = 0; i < W; ++i) w[k][i] = to_f32(p[i]), b[k][i] = 0.0f;
    if (a.bias) {
      const typename Pack<P, W>::type q = load_pack<W>(static_cast<const P*>(a.bias) + at, a.units - at);
#pragma unroll
      for (int i = 0; i < W; ++i) b[k][i] = to_f32(q[i]);
    }
  }
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * ROWS * R; first < a.tokens;
       first += static_cast<int64_t>(gridDim.x) * ROWS * R) {
    const int64_t token = first + threadIdx.x / NT * R;
    const T* row[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      row[r] = static_cast<const T*>(a.x) + (token + r < a.tokens ? token + r : first) * a.x_line;
    typename Pack<T, W>::type x[NC][R];
#pragma unroll
    for (int k = 0; k < NC; ++k) load_rows<R>(row, (k * NT + lane) * W, a.units, x[k]);
    float mean[R] = {}, r1[R] = {};
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < W; ++i) mean[r] += to_f32(x[k][r][i]);
    row_sums<WAVES>(mean, part[0]);
#pragma unroll
    for (int r = 0; r < R; ++r) mean[r] = mean_of(mean[r], units, inv);
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int left = a.units - (k * NT + lane) * W;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float d = i < left ? to_f32(x[k][r][i]) - mean[r] : 0.0f;
          r1[r] = __builtin_fmaf(d, d, r1[r]);
        }
    }
    row_sums<WAVES>(r1, part[1]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      r1[r] = 1.0f / sqrtf(r1[r] * inv + a.eps);
      if (token + r >= a.tokens) continue;
      if (lane == 0) reinterpret_cast<float2*>(a.kept)[token + r] = make_float2(mean[r], r1[r]);
      T* out = static_cast<T*>(a.y) + (token + r) * a.units;
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const int at = (k * NT + lane) * W;
        float y[W];
#pragma unroll
        for (int i = 0; i < W; ++i)
          y[i] = __builtin_fmaf((to_f32(x[k][r][i]) - mean[r]) * r1[r], w[k][i], b[k][i]);
        if (at < a.units) store_pack<W>(out + at, a.units - at, y);
      }
    }
  }
}

// Levels that no registers hold: the row is read three times.
template <typename T, typename P>
__global__ __launch_bounds__(1024) void k_normalise_stream(NormArgs a) {
  constexpr int W = kChunk<T>, WAVES = 16, STEP = 1024 * W;
  __shared__ float part[2][WAVES][1];
  const int64_t token = blockIdx.x;
  const T* row = static_cast<const T*>(a.x) + token * a.x_line;
  float sum = 0.0f, square = 0.0f;
  for (int at = threadIdx.x * W; at < a.units; at += STEP) {
    const typename Pack<T, W>::type x = load_pack<W>(row + at, a.units - at);
#pragma unroll
    for (int i = 0; i < W; ++i) sum += to_f32(x[i]);
  }
  const float units = static_cast<float>(a.units), inv = 1.0f / units;
  const float mean = mean_of(row_sum<WAVES>(sum, part[0]), units, inv);
  for (int at = threadIdx.x * W; at < a.units; at += STEP) {
    const typename Pack<T, W>::type x = load_pack<W>(row + at, a.units - at);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float d = at + i < a.units ? to_f32(x[i]) - mean : 0.0f;
      square = __builtin_fmaf(d, d, square);
    }
  }
  const float var = row_sum<WAVES>(square, part[1]) * inv;
  const float r = 1.0f / sqrtf(var + a.eps);
  if (threadIdx.x == 0) reinterpret_cast<float2*>(a.kept)[token] = make_float2(mean, r);
  T* out = static_cast<T*>(a.y) + token * a.units;
  for (int at = threadIdx.x * W; at < a.units; at += STEP) {
    const typename Pack<T, W>::type x = load_pack<W>(row + at, a.units - at);
    const typename Pack<P, W>::type w = load_pack<W>(static_cast<const P*>(a.weight) + at, a.units - at);
    float y[W];
#pragma unroll
    for (int i = 0; i < W; ++i) y[i] = (to_f32(x[i]) - mean) * r * to_f32(w[i]);
    if (a.bias) {
      const typename Pack<P, W>::type b = load_pack<W>(static_cast<const P*>(a.bias) + at, a.units - at);
#pragma unroll
      for (int i = 0; i < W; ++i) y[i] += to_f32(b[i]);
    }
    store_pack<W>(out + at, a.units - at, y);
  }
}

// The gradients, a row at a time: a lane keeps its sums of g n and g in
// registers; they are joined over the groups in LDS and written as the
// workgroup's part. (16384 x 4096 bf16 79 us with two workgroups a CU, which fit
// while a lane has at most 64 registers; 61 are used. With one a CU it was 87, and
// 94 with two rows at a time or the next one's loads ahead, for which those
// registers are not there.)
template <typename T, typename P, int ROWS, int WAVES, int NC>
__global__ __launch_bounds__(ROWS* WAVES * 64) void k_normalise_grad(NormArgs a) {
  constexpr int W = kChunk<T>, NT = WAVES * 64;
  __shared__ float part[2][ROWS * WAVES][2];
  __shared__ float joined[ROWS > 1 ? NT * W : 1];
  const int lane = threadIdx.x % NT, group = threadIdx.x / NT;
  const float inv = 1.0f / static_cast<float>(a.units);
  float w[NC][W], dw[NC][W], db[NC][W];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int at = (k * NT + lane) * W;
    const typename Pack<P, W>::type p = load_pack<W>(static_cast<const P*>(a.weight) + at, a.units - at);
#pragma unroll
    for (int i = 0; i < W; ++i) w[k][i] = to_f32(p[i]), dw[k][i] = 0.0f, db[k][i] = 0.0f;
  }
  int slot = 0;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * ROWS; first < a.tokens;
       first += static_cast<int64_t>(gridDim.x) * ROWS) {
    const int64_t token = first + group, from = token < a.tokens ? token : first;
    const bool there = token < a.tokens;
    const T* const xr[1] = {static_cast<const T*>(a.x) + from * a.x_line};
    const T* const gr[1] = {static_cast<const T*>(a.g) + from * a.g_line};
    const float2 kept = reinterpret_cast<const float2*>(a.kept)[from];
    typename Pack<T, W>::type x[NC][1], g[NC][1];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      load_rows<1>(xr, (k * NT + lane) * W, a.units, x[k]);
      load_rows<1>(gr, (k * NT + lane) * W, a.units, g[k]);
    }
    float sums[2] = {0.0f, 0.0f};
    // Past the row's end n is 0, as g and w are: (0 - mean) r may be past float32, and 0 times that is a NaN in the sums.
    // (Where a lane has several chunks the whole ones go without the selects, for their registers: 4096 x 16384 bf16 90
    // us, with them 96. Of one chunk a lane they cost nothing.)
    const auto add = [&](int k, int i, int left) {
      const float n = i < left ? (to_f32(x[k][0][i]) - kept.x) * kept.y : 0.0f;
      const float d = to_f32(g[k][0][i]), u = d * w[k][i];
      dw[k][i] = __builtin_fmaf(d, n, dw[k][i]);
      db[k][i] += d;
      sums[0] += u;
      sums[1] = __builtin_fmaf(u, n, sums[1]);
    };
    if (there) {
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const int left = a.units - (k * NT + lane) * W;
        if (NC > 1 && left >= W) {
#pragma unroll
          for (int i = 0; i < W; ++i) add(k, i, W);
        } else {
#pragma unroll
          for (int i = 0; i < W; ++i) add(k, i, left);
        }
      }
    }
    row_sums<WAVES>(sums, part[slot]);
    slot ^= 1;
    if (!there) continue;
    const float mean = sums[0] * inv, mean_n = sums[1] * inv;
    T* out = static_cast<T*>(a.y) + token * a.units;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int at = (k * NT + lane) * W;
      float d[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float n = (to_f32(x[k][0][i]) - kept.x) * kept.y;
        d[i] = kept.y * (to_f32(g[k][0][i]) * w[k][i] - mean - n * mean_n);
      }
      if (at < a.units) store_pack<W>(out + at, a.units - at, d);
    }
  }
  float* mine = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.units;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int at = (k * NT + lane) * W;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* v = h ? db[k] : dw[k];
      for (int o = 1; o < ROWS; ++o) {
        __syncthreads();
        if (group == o) {
#pragma unroll
          for (int i = 0; i < W; ++i) joined[i * NT + lane] = v[i];
        }
        __syncthreads();
        if (group == 0) {
#pragma unroll
          for (int i = 0; i < W; ++i) v[i] += joined[i * NT + lane];
        }
      }
      if (group == 0 && at < a.units) store_pack<W>(mine + h * a.units + at, a.units - at, v);
    }
  }
}

// Levels that no registers hold: first each row's two means, then dx and the
// parts of dw and db by columns of units (blockIdx.y), rows in turn.
template <typename T, typename P>
__global__ __launch_bounds__(1024) void k_normalise_means(NormArgs a, float* means) {
  constexpr int W = kChunk<T>, WAVES = 16;
  __shared__ float part[WAVES][2];
  const int64_t token = blockIdx.x;
  const T* xr = static_cast<const T*>(a.x) + token * a.x_line;
  const T* gr = static_cast<const T*>(a.g) + token * a.g_line;
  const float2 kept = reinterpret_cast<const float2*>(a.kept)[token];
  float s = 0.0f, sn = 0.0f;
  for (int at = threadIdx.x * W; at < a.units; at += 1024 * W) {
    const typename Pack<T, W>::type x = load_pack<W>(xr + at, a.units - at), d = load_pack<W>(gr + at, a.units - at);
    const typename Pack<P, W>::type w = load_pack<W>(static_cast<const P*>(a.weight) + at, a.units - at);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float u = to_f32(d[i]) * to_f32(w[i]);
      s += u;
      sn += at + i < a.units ? u * ((to_f32(x[i]) - kept.x) * kept.y) : 0.0f;
    }
  }
  float sums[2] = {s, sn};
  row_sums<WAVES>(sums, part);
  const float inv = 1.0f / static_cast<float>(a.units);
  if (threadIdx.x == 0) reinterpret_cast<float2*>(means)[token] = make_float2(sums[0] * inv, sums[1] * inv);
}
template <typename T, typename P>
__global__ __launch_bounds__(256) void k_normalise_columns(NormArgs a, const float* means) {
  const int unit = blockIdx.y * 256 + threadIdx.x;
  if (unit >= a.units) return;
  const float w = to_f32(static_cast<const P*>(a.weight)[unit]);
  float dw = 0.0f, db = 0.0f;
  for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
    const float2 kept = reinterpret_cast<const float2*>(a.kept)[token];
    const float2 mean = reinterpret_cast<const float2*>(means)[token];
    const float g = to_f32(static_cast<const T*>(a.g)[token * a.g_line + unit]);
    const float n = (to_f32(static_cast<const T*>(a.x)[token * a.x_line + unit]) - kept.x) * kept.y;
    dw += g * n;
    db += g;
    static_cast<T*>(a.y)[token * a.units + unit] = from_f32<T>(kept.y * (g * w - mean.x - n * mean.y));
  }
  float* mine = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.units;
  mine[unit] = dw;
  mine[a.units + unit] = db;
}

// out [2][units] = the sums of the workgroups' parts: 64 columns a workgroup,
// the parts over its 16 waves.
__global__ __launch_bounds__(1024) void k_normalise_join(int parts, int64_t n, const float* part, float* out) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  float s = 0.0f;
  if (at < n) {
    const int per = (parts + 15) / 16, last = (wave + 1) * per < parts ? (wave + 1) * per : parts;
#pragma unroll 8
    for (int p = wave * per; p < last; ++p) s += part[p * n + at];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave > 0 || at >= n) return;
  for (int w = 1; w < 16; ++w) s += sums[w][lane];
  out[at] = s;
}

// How a level's rows are taken: as many waves as give each lane a chunk of 16
// bytes (of wide levels more, up to 16 values); workgroups of 4 waves and more
// forwards and of 16 backwards, those of the gradients at most two a CU where they hold
// several rows (their barriers are for all of them), else one: every workgroup
// has a part of dw and db to write.
struct NormPlan {
  int waves, chunks, rows, groups;  // chunks 0: the forms that hold no rows
  int64_t bytes, means;
};
NormPlan norm_plan(int64_t tokens, int64_t units, int dtype) {
  const int64_t chunks = div_up(units, dtype == PLX_LB_F32 ? 4 : 8);
  NormPlan p{};
  p.waves = chunks <= 64 ? 1 : chunks <= 128 ? 2 : chunks <= 256 ? 4 : chunks <= 512 ? 8 : 16;
  p.chunks = chunks <= 1024 ? 1 : chunks <= 2048 ? 2 : chunks <= 4096 && dtype == PLX_LB_F32 ? 4 : 0;
  p.rows = p.chunks ? 16 / p.waves : 1;
  // (Figures of rules here: one input again and again, partly in the caches.)
  // Two workgroups a CU, whose loads and sums overlap, where each has rows enough to make up for a second part to
  // join, and registers for both (16384 x 4096 bf16 68 us, one a CU 81; 2000 x 4096 19, one 16; 16384 units, one row
  // a workgroup, 4096 bf16 80, one 68).
  const int64_t groups = div_up(tokens, p.rows), cus = cu_count();
  const int64_t most = cus * (p.rows > 1 && groups > 4 * cus ? 2 : 1);
  p.groups = static_cast<int>(groups < most ? groups : most);
  p.bytes = int64_t{8} * p.groups * units;
  p.means = p.bytes;
  if (!p.chunks) p.bytes += 8 * tokens;
  return p;
}

template <typename T, typename F>
void with_rows(const NormPlan& p, F f) {
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I4 = std::integral_constant<int, 4>;
  using I8 = std::integral_constant<int, 8>;
  using I16 = std::integral_constant<int, 16>;
  if (p.waves == 1)
    f(I1{}, I1{});
  else if (p.waves == 2)
    f(I2{}, I1{});
  else if (p.waves == 4)
    f(I4{}, I1{});
  else if (p.waves == 8)
    f(I8{}, I1{});
  else if (p.chunks == 1)
    f(I16{}, I1{});
  else if (p.chunks == 2)
    f(I16{}, I2{});
  else if constexpr (sizeof(T) == 4)
    f(I16{}, I4{});
}

template <typename T, typename P>
void launch_normalise(const NormArgs& all, const NormPlan& p, hipStream_t s) {
  if (p.chunks) {
    with_rows<T>(p, [&](auto waves, auto chunks) {
      constexpr int WAVES = decltype(waves)::value, NC = decltype(chunks)::value, ROWS = WAVES < 4 ? 4 / WAVES : 1;
      const int64_t most = int64_t{cu_count()} * (32 / (ROWS * WAVES));  // all waves that a CU holds
      // (Several rows at a time where all waves have more than two: 16384 x 4096 bf16 45 us, one at a time 51;
      // 1200 x 4096 7.2, one 6.4; two or so, as 4096 x 1000 float32 7.5 and 8.2, 16384 x 512 bf16 8.0 and 7.5.)
      if (all.tokens > 2 * most * ROWS) {
        constexpr int R = kRows / NC;
        const int64_t groups = div_up(all.tokens, ROWS * R);
        k_normalise<T, P, ROWS, WAVES, NC, R>
            <<<static_cast<unsigned>(groups < most ? groups : most), ROWS * WAVES * 64, 0, s>>>(all);
      } else {
        k_normalise<T, P, ROWS, WAVES, NC, 1>
            <<<static_cast<unsigned>(div_up(all.tokens, ROWS)), ROWS * WAVES * 64, 0, s>>>(all);
      }
    });
    return;
  }
  constexpr int64_t most = int64_t{1} << 20;  // workgroups of a launch: at most 2^30 lanes
  for (int64_t first = 0; first < all.tokens; first += most) {
    NormArgs a = all;
    a.tokens = all.tokens - first < most ? all.tokens - first : most;
    a.x = static_cast<const T*>(all.x) + first * all.x_line;
    a.y = static_cast<T*>(all.y) + first * all.units;
    a.kept = all.kept + 2 * first;
    k_normalise_stream<T, P><<<static_cast<unsigned>(a.tokens), 1024, 0, s>>>(a);
  }
}

template <typename T, typename P>
void launch_grad(const NormArgs& a, const NormPlan& p, hipStream_t s) {
  if (!p.chunks) {
    float* means = reinterpret_cast<float*>(reinterpret_cast<char*>(a.part) + p.means);
    constexpr int64_t most = int64_t{1} << 20;
    for (int64_t first = 0; first < a.tokens; first += most) {
      NormArgs b = a;
      b.x = static_cast<const T*>(a.x) + first * a.x_line;
      b.g = static_cast<const T*>(a.g) + first * a.g_line;
      b.kept = a.kept + 2 * first;
      const int64_t now = a.tokens - first < most ? a.tokens - first : most;
      k_normalise_means<T, P><<<static_cast<unsigned>(now), 1024, 0, s>>>(b, means + 2 * first);
    }
    const dim3 grid(static_cast<unsigned>(p.groups), static_cast<unsigned>(div_up(a.units, 256)));
    k_normalise_columns<T, P><<<grid, 256, 0, s>>>(a, means);
    return;
  }
  with_rows<T>(p, [&](auto waves, auto chunks) {
    constexpr int WAVES = decltype(waves)::value, ROWS = 16 / WAVES;
    k_normalise_grad<T, P, ROWS, WAVES, decltype(chunks)::value>
        <<<static_cast<unsigned>(p.groups), ROWS * WAVES * 64, 0, s>>>(a);
  });
}

// F(T, P) by the types of the batch and of the parameters.
template <typename F>
void with_types(int dtype, int params, F f) {
  with_type(dtype, [&](auto* e) {
    if (params == PLX_LB_F32)
      f(e, static_cast<float*>(nullptr));
    else
      f(e, e);
  });
}

int check_norm(const char* who, int64_t tokens, int64_t units, int dtype, int params, float eps) {
  if (!batch_fits(tokens, units)) return fail(PLX_ERR_INVALID, who);
  if (!known_type(dtype) || (params != dtype && params != PLX_LB_F32)) return fail(PLX_ERR_UNSUPPORTED, who);
  if (!(eps >= 0.0f && eps < INFINITY)) return fail(PLX_ERR_INVALID, who);
  return PLX_OK;
}

}  // namespace

extern "C" {

int plx_normalise(int64_t tokens, int64_t units, int32_t dtype, const void* x, int64_t line, int32_t params,
                  const void* weight, const void* bias, float eps, void* y, float* kept, void* stream) {
  const char* who = "plx_normalise: bad size, type, eps or null pointer";
  if (const int rc = check_norm(who, tokens, units, dtype, params, eps)) return rc;
  if (tokens == 0 || units == 0) return PLX_OK;
  if (!x || !weight || !y || !kept) return fail(PLX_ERR_INVALID, who);
  NormArgs a{};
  a.tokens = tokens, a.x_line = line, a.units = static_cast<int>(units), a.eps = eps;
  a.x = x, a.weight = weight, a.bias = bias, a.y = y, a.kept = kept;
  const NormPlan p = norm_plan(tokens, units, dtype);
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_types(dtype, params, [&](auto* t, auto* q) {
    launch_normalise<PLX_DENSE_TYPE(t), PLX_DENSE_TYPE(q)>(a, p, s);
  });
  return check_launch("plx_normalise");
}

int64_t plx_normalise_workspace(int64_t tokens, int64_t units, int32_t dtype) {
  if (!batch_fits(tokens, units) || !known_type(dtype)) return -1;
  return tokens == 0 || units == 0 ? 0 : norm_plan(tokens, units, dtype).bytes;
}

int plx_normalise_grad(int64_t tokens, int64_t units, int32_t dtype, const void* g, int64_t g_line, const void* x,
                       int64_t x_line, int32_t params, const void* weight, const float* kept, void* dx,
                       float* dparams, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "plx_normalise_grad: bad size, type or null pointer";
  if (const int rc = check_norm(who, tokens, units, dtype, params, 0.0f)) return rc;
  if (units == 0) return PLX_OK;
  if (!dparams) return fail(PLX_ERR_INVALID, who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t n = 2 * units;
  if (tokens == 0) {
    k_normalise_join<<<static_cast<unsigned>(div_up(n, 64)), 1024, 0, s>>>(0, n, nullptr, dparams);
    return check_launch("plx_normalise_grad");
  }
  const NormPlan p = norm_plan(tokens, units, dtype);
  if (!g || !x || !weight || !kept || !dx) return fail(PLX_ERR_INVALID, who);
  if (!workspace || !on_16(workspace) || workspace_bytes < p.bytes)
    return fail(PLX_ERR_INVALID, "plx_normalise_grad: plx_normalise_workspace() bytes on 16 bytes needed");
  NormArgs a{};
  a.tokens = tokens, a.x_line = x_line, a.g_line = g_line, a.units = static_cast<int>(units);
  a.x = x, a.g = g, a.weight = weight, a.y = dx, a.kept = const_cast<float*>(kept);
  a.part = static_cast<float*>(workspace);
  with_types(dtype, params, [&](auto* t, auto* q) { launch_grad<PLX_DENSE_TYPE(t), PLX_DENSE_TYPE(q)>(a, p, s); });
  k_normalise_join<<<static_cast<unsigned>(div_up(n, 64)), 1024, 0, s>>>(p.groups, n, a.part, dparams);
  return check_launch("plx_normalise_grad");
}

}  // extern "C"
