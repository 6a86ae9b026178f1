// recur.hip -- a level carried along sequences by a gated linear recurrence,
// its gradients, and one token at a time. No counterpart in the reference,
// whose PIPELINE nets carry state from step to step only.
//
// a = sigmoid(z), h[t] = a[t] h[t-1] + (1 - a[t]) x[t] for each unit, from the
// sequence's state. Backwards c[t] = g[t] + a[t+1] c[t+1] (at a sequence's
// last row plus its last state's gradient), dx = (1 - a) c,
// dz = a (1 - a) (h[t-1] - x) c, and a c of its first row is the state's.
//
// Rows with h -> A h + H compose, so a row range can be summed up before what
// comes in is known. A workgroup walks its part of the rows in steps of kStep,
// a lane two units of a few rows, the step's waves behind each other: each
// wave sums up its rows, the sums meet in LDS, and each wave walks its rows
// again from what comes in. Where units alone do not fill the CUs the rows are
// cut into parts, which a launch before sums up (the rows are read twice).

#include "px_dense.h"

using plx_detail::check_launch;
using plx_detail::cu_count;
using plx_detail::fail;

namespace {

using namespace px;

constexpr int kWaves = 16, kRows = 8, kStep = kWaves * kRows;  // rows of a step
constexpr int kBack = 4, kKeep = PLX_RECUR_KEEP;              // and of one of the gradients' (registers)
static_assert(kKeep == kWaves * kBack && kStep % kKeep == 0, "a step begins where its state is kept");
constexpr int kSlab = 128;                                     // units of a workgroup
constexpr int64_t kMaxSequences = int64_t{1} << 30;

struct RecurArgs {
  int64_t tokens, sequences, line, g_line, part;  // part: rows of a part, a multiple of kStep
  int units, wide;
  const void* xz;
  const void* starts;  // null: one sequence
  const int* of;       // [tokens]: the row's sequence, -1 outside of all (null: one sequence)
  const float* state;  // null: zeros
  void* h;
  float* last;
  float* kept;  // [ceil(tokens / kKeep)][units]: what comes into its rows
  float* sums;  // [parts][3][units]
  // backwards
  const void* g;
  const float* g_last;  // null: zeros
  void* dxz;
  float* dstate;
};

__device__ __forceinline__ int64_t start_of(const RecurArgs& a, int64_t s) {
  const int64_t t = load_id(a.starts, a.wide, s);
  return t < 0 ? 0 : t < a.tokens ? t : a.tokens;
}

// of[t]: the last sequence that starts at t or before, if t is before its end.
__global__ __launch_bounds__(256) void k_recur_rows(RecurArgs a, int* of) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t >= a.tokens) return;
  int64_t lo = -1, hi = a.sequences;  // start_of(lo) <= t < start_of(hi), as far as they are sequences
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (start_of(a, mid) <= t)
      lo = mid;
    else
      hi = mid;
  }
  of[t] = lo >= 0 && t < start_of(a, lo + 1) ? static_cast<int>(lo) : -1;
}

// The sequences of rows first - 1 to first + N, the same in all lanes.
template <int N>
__device__ __forceinline__ void rows_of(const RecurArgs& a, int64_t first, int of[N + 2]) {
#pragma unroll
  for (int i = 0; i < N + 2; ++i) {
    const int64_t t = first - 1 + i;
    const bool there = t >= 0 && t < a.tokens;
    of[i] = !there ? -1 : a.of ? __builtin_amdgcn_readfirstlane(a.of[t]) : 0;
  }
}

// a = sigmoid(z) and b = 1 - a, both to a few steps: by exp(-|z|), with the
// rounding error of its exponent carried on.
__device__ __forceinline__ void gate(float z, float& a, float& b) {
  const float y = fabsf(z);
  const float hi = y * -1.44269502162933349609375f;
  float lo = __builtin_fmaf(y, -1.44269502162933349609375f, -hi);
  lo = __builtin_fmaf(y, -1.925963033500011e-8f, lo);
  float t = __builtin_amdgcn_exp2f(hi);
  t = t > 0.0f ? __builtin_fmaf(t * lo, 0.693147182464599609375f, t) : t;
  float r = __builtin_amdgcn_rcpf(1.0f + t);
  r = __builtin_fmaf(__builtin_fmaf(-(1.0f + t), r, 1.0f), r, r);
  const float s = t * r;
  a = z < 0.0f ? s : r;
  b = z < 0.0f ? r : s;
}

struct Pair {
  float v[2];
};
__device__ __forceinline__ Pair load_pair(const float* p, int n) {
  Pair r;
  r.v[0] = n > 0 ? p[0] : 0.0f, r.v[1] = n > 1 ? p[1] : 0.0f;
  return r;
}
__device__ __forceinline__ void store_pair(float* p, int n, const float v[2]) {
  if (n > 0) p[0] = v[0];
  if (n > 1) p[1] = v[1];
}

__device__ __forceinline__ Pair load_state(const RecurArgs& a, const float* states, int s, int col, int n) {
  if (!states) return {{0.0f, 0.0f}};
  return load_pair(states + static_cast<int64_t>(s) * a.units + col, n);
}

// A row range as a map of what comes in, two units: v -> A v + H, or H alone
// where a sequence's border lies in it (`cut`, the same in all lanes; with
// A = 0 in its place an infinity or a NaN would go on into the next sequence).
struct Span {
  float A[2], H[2];
  bool cut;
};
__device__ __forceinline__ Span span_none() { return {{1.0f, 1.0f}, {0.0f, 0.0f}, false}; }
__device__ __forceinline__ void span_then(Span& s, const Span& next) {  // s, then next
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s.H[i] = next.cut ? next.H[i] : __builtin_fmaf(next.A[i], s.H[i], next.H[i]);
    s.A[i] *= next.A[i];
  }
  s.cut |= next.cut;
}
// The spans of a step's waves.
struct Spans {
  float4 v[kWaves][64];
  int cut[kWaves];
  __device__ __forceinline__ void put(int wave, int lane, const Span& s) {
    v[wave][lane] = make_float4(s.A[0], s.A[1], s.H[0], s.H[1]);
    if (lane == 0) cut[wave] = s.cut;
  }
  __device__ __forceinline__ Span get(int wave, int lane) const {
    const float4 f = v[wave][lane];
    return {{f.x, f.y}, {f.z, f.w}, __builtin_amdgcn_readfirstlane(cut[wave]) != 0};
  }
  __device__ __forceinline__ void pass(int wave, int lane, Pair& in) const {
    const Span s = get(wave, lane);
#pragma unroll
    for (int j = 0; j < 2; ++j) in.v[j] = s.cut ? s.H[j] : __builtin_fmaf(s.A[j], in.v[j], s.H[j]);
  }
};

// A part's span in memory: A, H, and cut (as a float) for each unit.
__device__ __forceinline__ void store_span(const RecurArgs& a, int64_t part, int col, int n, const Span& s) {
  float* out = a.sums + part * 3 * a.units + col;
  const float cut[2] = {s.cut ? 1.0f : 0.0f, s.cut ? 1.0f : 0.0f};
  store_pair(out, n, s.A);
  store_pair(out + a.units, n, s.H);
  store_pair(out + 2 * a.units, n, cut);
}

// The parts before (or, backwards, behind) part p summed up to what comes into
// it: over the waves, then over LDS.
template <bool BACK>
__device__ __forceinline__ Pair into_part(const RecurArgs& a, int64_t p, int64_t parts, int col, int n, Spans& spans) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t count = BACK ? parts - 1 - p : p, per = div_up(count, kWaves);
  Span s = span_none();
  for (int64_t i = wave * per; i < (wave + 1) * per && i < count; ++i) {
    const float* q = a.sums + (BACK ? parts - 1 - i : i) * 3 * a.units;
    const Pair A = load_pair(q + col, n), H = load_pair(q + a.units + col, n);
    // (the first unit's: a slab's first column is there)
    const bool cut = __builtin_amdgcn_readfirstlane(__float_as_int(q[2 * a.units + blockIdx.x * kSlab])) != 0;
    span_then(s, {{A.v[0], A.v[1]}, {H.v[0], H.v[1]}, cut});
  }
  spans.put(wave, lane, s);
  __syncthreads();
  Pair in = {{0.0f, 0.0f}};
#pragma unroll 4
  for (int w = 0; w < kWaves; ++w) spans.pass(w, lane, in);
  __syncthreads();
  return in;
}

// One row forwards: A and H as its map, from its z and x; `first` has the
// sequence's state put in.
__device__ __forceinline__ void row_forward(const RecurArgs& a, int q, bool first, int col, int n, float A[2],
                                            float H[2]) {
  if (q < 0) {
    H[0] = H[1] = 0.0f;
  } else if (first) {
    const Pair in = load_state(a, a.state, q, col, n);
#pragma unroll
    for (int j = 0; j < 2; ++j) H[j] = __builtin_fmaf(A[j], in.v[j], H[j]);
  }
}

// Forwards: each part (but the last) as a span; a wave's rows lie behind each
// other.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void k_recur_parts(RecurArgs a) {
  __shared__ Spans spans;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = blockIdx.x * kSlab + lane * 2, n = a.units - col;
  const int64_t part = blockIdx.y, per = a.part / kWaves, begin = part * a.part + wave * per;
  Span s = span_none();
  const T* xz = static_cast<const T*>(a.xz) + col;
  for (int64_t t = begin; t < begin + per; t += kRows) {
    int of[kRows + 2];
    rows_of<kRows>(a, t, of);
    typename Pack<T, 2>::type x[kRows], z[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const bool there = t + i < a.tokens;
      const T* row = xz + (there ? t + i : 0) * a.line;
      x[i] = load_pack<2>(row, there ? n : 0), z[i] = load_pack<2>(row + a.units, there ? n : 0);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      Span row;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float b;
        gate(to_f32(z[i][j]), row.A[j], b);
        row.H[j] = b * to_f32(x[i][j]);
      }
      const int q = of[i + 1];
      row.cut = q < 0 || of[i] != q;
      row_forward(a, q, row.cut, col, n, row.A, row.H);
      span_then(s, row);
    }
  }
  spans.put(wave, lane, s);
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < kWaves; ++w) span_then(s, spans.get(w, lane));
  store_span(a, part, col, n, s);
}

// Sequences without rows: out = in (null: zeros), 64 of them at a time by the
// waves of a slab's workgroups.
__device__ __forceinline__ void pass_empty(const RecurArgs& a, const float* in, float* out, int col, int n) {
  const int lane = threadIdx.x & 63;
  if (!a.starts && a.tokens > 0) return;
  for (int64_t first = (static_cast<int64_t>(blockIdx.y) * kWaves + (threadIdx.x >> 6)) * 64; first < a.sequences;
       first += static_cast<int64_t>(gridDim.y) * kWaves * 64) {
    const int64_t s = first + lane;
    const bool empty = s < a.sequences && (!a.starts || start_of(a, s) >= start_of(a, s + 1));
    for (uint64_t mask = __ballot(empty); mask; mask &= mask - 1) {
      const int64_t at = (first + __builtin_ctzll(mask)) * a.units + col;
      const Pair v = in ? load_pair(in + at, n) : Pair{{0.0f, 0.0f}};
      store_pair(out + at, n, v.v);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(64 * kWaves) void k_recur(RecurArgs a) {
  __shared__ Spans spans[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = blockIdx.x * kSlab + lane * 2, n = a.units - col;
  const int64_t part = blockIdx.y, begin = part * a.part;
  const int64_t end = begin + a.part < a.tokens ? begin + a.part : a.tokens;
  const T* xz = static_cast<const T*>(a.xz) + col;
  T* out = static_cast<T*>(a.h) + col;
  Pair in = {{0.0f, 0.0f}};
  if (part > 0) in = into_part<false>(a, part, gridDim.y, col, n, spans[0]);
  int slot = 0;
  for (int64_t step = begin; step < end; step += kStep) {
    const int64_t t = step + wave * kRows;
    int of[kRows + 2];
    rows_of<kRows>(a, t, of);
    typename Pack<T, 2>::type x[kRows], z[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const bool there = t + i < a.tokens;
      const T* row = xz + (there ? t + i : 0) * a.line;
      x[i] = load_pack<2>(row, there ? n : 0), z[i] = load_pack<2>(row + a.units, there ? n : 0);
    }
    float A[kRows][2], H[kRows][2];
    Span s = span_none();
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float b;
        gate(to_f32(z[i][j]), A[i][j], b);
        H[i][j] = b * to_f32(x[i][j]);
      }
      const int q = of[i + 1];
      const bool cut = q < 0 || of[i] != q;
      row_forward(a, q, cut, col, n, A[i], H[i]);
      span_then(s, {{A[i][0], A[i][1]}, {H[i][0], H[i][1]}, cut});
    }
    spans[slot].put(wave, lane, s);
    __syncthreads();
    Pair h = in;
#pragma unroll 4
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) h = in;
      spans[slot].pass(w, lane, in);
    }
    slot ^= 1;
    if (t % kKeep == 0 && t < end) store_pair(a.kept + t / kKeep * a.units + col, n, h.v);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (t + i >= end) break;
      const int q = of[i + 1];
      const bool cut = q < 0 || of[i] != q;
#pragma unroll
      for (int j = 0; j < 2; ++j) h.v[j] = cut ? H[i][j] : __builtin_fmaf(A[i][j], h.v[j], H[i][j]);
      store_pack<2>(out + (t + i) * a.units, n, h.v);
      if (q >= 0 && of[i + 2] != q) store_pair(a.last + static_cast<int64_t>(q) * a.units + col, n, h.v);
    }
  }
  pass_empty(a, a.state, a.last, col, n);
}

// Backwards, a row passes on what comes in from behind as u -> a (g + u); a
// sequence's last row puts its last state's gradient in, its first row's goes
// to its state and no further.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void k_recur_grad_parts(RecurArgs a) {
  __shared__ Spans spans;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = blockIdx.x * kSlab + lane * 2, n = a.units - col;
  const int64_t part = blockIdx.y + 1, per = a.part / kWaves, begin = part * a.part + wave * per;
  Span s = span_none();
  const T* zs = static_cast<const T*>(a.xz) + a.units + col;
  const T* gs = static_cast<const T*>(a.g) + col;
  for (int64_t t = begin + per - kRows; t >= begin; t -= kRows) {
    int of[kRows + 2];
    rows_of<kRows>(a, t, of);
    typename Pack<T, 2>::type z[kRows], g[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const bool there = t + i < a.tokens;
      z[i] = load_pack<2>(zs + (there ? t + i : 0) * a.line, there ? n : 0);
      g[i] = load_pack<2>(gs + (there ? t + i : 0) * a.g_line, there ? n : 0);
    }
#pragma unroll
    for (int i = kRows - 1; i >= 0; --i) {
      const int q = of[i + 1];
      const bool on = q >= 0 && of[i] == q, last = of[i + 2] != q;
      const Pair more = on && last ? load_state(a, a.g_last, q, col, n) : Pair{{0.0f, 0.0f}};
      Span row;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float b;
        gate(to_f32(z[i][j]), row.A[j], b);
        row.H[j] = on ? row.A[j] * (to_f32(g[i][j]) + more.v[j]) : 0.0f;
      }
      row.cut = !on || last;
      span_then(s, row);
    }
  }
  spans.put(wave, lane, s);
  __syncthreads();
  if (wave < kWaves - 1) return;
  for (int w = kWaves - 2; w >= 0; --w) span_then(s, spans.get(w, lane));
  store_span(a, part, col, n, s);
}

// The gradients, steps from the last to the first. h is walked again from what
// came into the step, so that it is neither kept nor rounded.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void k_recur_grad(RecurArgs a) {
  __shared__ Spans spans[2], backs[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = blockIdx.x * kSlab + lane * 2, n = a.units - col;
  const int64_t part = blockIdx.y, begin = part * a.part;
  const int64_t end = begin + a.part < a.tokens ? begin + a.part : a.tokens;
  const T* xz = static_cast<const T*>(a.xz) + col;
  const T* gs = static_cast<const T*>(a.g) + col;
  T* out = static_cast<T*>(a.dxz) + col;
  Pair back = {{0.0f, 0.0f}};
  if (part + 1 < gridDim.y) back = into_part<true>(a, part, gridDim.y, col, n, spans[0]);
  int slot = 0;
  for (int64_t step = begin + (div_up(end - begin, kKeep) - 1) * kKeep; step >= begin; step -= kKeep) {
    const int64_t t = step + wave * kBack;
    int of[kBack + 2];
    rows_of<kBack>(a, t, of);
    typename Pack<T, 2>::type x[kBack], z[kBack], g[kBack];
#pragma unroll
    for (int i = 0; i < kBack; ++i) {
      const bool there = t + i < a.tokens;
      const T* row = xz + (there ? t + i : 0) * a.line;
      x[i] = load_pack<2>(row, there ? n : 0), z[i] = load_pack<2>(row + a.units, there ? n : 0);
      g[i] = load_pack<2>(gs + (there ? t + i : 0) * a.g_line, there ? n : 0);
    }
    Pair h = load_pair(a.kept + step / kKeep * a.units + col, n);
    float A[kBack][2], B[kBack][2], d[kBack][2];  // d: g, with the last state's gradient at a last row
    Span s = span_none(), u = span_none();
#pragma unroll
    for (int i = 0; i < kBack; ++i) {
      const int q = of[i + 1];
      Span row;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        gate(to_f32(z[i][j]), A[i][j], B[i][j]);
        row.A[j] = A[i][j], row.H[j] = B[i][j] * to_f32(x[i][j]);
      }
      row.cut = q < 0 || of[i] != q;
      row_forward(a, q, row.cut, col, n, row.A, row.H);
      span_then(s, row);
    }
#pragma unroll
    for (int i = kBack - 1; i >= 0; --i) {
      const int q = of[i + 1];
      const bool on = q >= 0 && of[i] == q, last = of[i + 2] != q;
      const Pair more = q >= 0 && last ? load_state(a, a.g_last, q, col, n) : Pair{{0.0f, 0.0f}};
      Span row;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        d[i][j] = to_f32(g[i][j]) + more.v[j];
        row.A[j] = A[i][j], row.H[j] = on ? A[i][j] * d[i][j] : 0.0f;
      }
      row.cut = !on || last;
      span_then(u, row);
    }
    spans[slot].put(wave, lane, s);
    backs[slot].put(wave, lane, u);
    __syncthreads();
    Pair c = back;
    for (int w = 0; w < wave; ++w) spans[slot].pass(w, lane, h);
#pragma unroll 4
    for (int w = kWaves - 1; w >= 0; --w) {
      if (w == wave) c = back;
      backs[slot].pass(w, lane, back);
    }
    slot ^= 1;
    float before[kBack][2];  // h of the row before
#pragma unroll
    for (int i = 0; i < kBack; ++i) {
      const int q = of[i + 1];
      if (of[i] != q) h = q >= 0 ? load_state(a, a.state, q, col, n) : Pair{{0.0f, 0.0f}};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        before[i][j] = h.v[j];
        h.v[j] = __builtin_fmaf(A[i][j], h.v[j], B[i][j] * to_f32(x[i][j]));
      }
    }
#pragma unroll
    for (int i = kBack - 1; i >= 0; --i) {
      if (t + i >= end) continue;
      const int q = of[i + 1];
      float dx[2] = {0.0f, 0.0f}, dz[2] = {0.0f, 0.0f};
      if (q >= 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float v = of[i + 2] != q ? d[i][j] : d[i][j] + c.v[j];
          dx[j] = B[i][j] * v;
          dz[j] = dx[j] * A[i][j] * (before[i][j] - to_f32(x[i][j]));
          c.v[j] = A[i][j] * v;
        }
        if (of[i] != q) store_pair(a.dstate + static_cast<int64_t>(q) * a.units + col, n, c.v);
      }
      T* row = out + (t + i) * 2 * a.units;
      store_pack<2>(row, n, dx);
      store_pack<2>(row + a.units, n, dz);
    }
  }
  pass_empty(a, a.g_last, a.dstate, col, n);
}

// One row a sequence, the state in place; a lane takes 4 units.
template <typename T>
__global__ __launch_bounds__(256) void k_recur_step(int64_t sequences, int units, const T* xz, int64_t line,
                                                    float* state, int64_t state_line, T* h) {
  const int64_t chunks = div_up(units, 4), total = sequences * chunks;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t s = i / chunks;
    const int at = static_cast<int>(i - s * chunks) * 4, n = units - at;
    const typename Pack<T, 4>::type x = load_pack<4>(xz + s * line + at, n), z = load_pack<4>(xz + s * line + units + at, n);
    const typename Pack<float, 4>::type v = load_pack<4>(state + s * state_line + at, n);
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      gate(to_f32(z[j]), a, b);
      y[j] = __builtin_fmaf(a, v[j], b * to_f32(x[j]));
    }
    store_pack<4>(state + s * state_line + at, n, y);
    store_pack<4>(h + s * units + at, n, y);
  }
}

// How the rows are cut: two workgroups a CU, parts of whole steps, few enough
// that what comes into one is soon summed up.
struct RecurPlan {
  int64_t slabs, parts, part, steps, of, bytes;
};
constexpr int64_t kMaxParts = 128;
RecurPlan recur_plan(int64_t tokens, int64_t units, bool ragged) {
  RecurPlan p{};
  p.slabs = div_up(units, kSlab);
  p.steps = div_up(tokens, kStep);
  int64_t parts = 2 * cu_count() / p.slabs;
  parts = parts < kMaxParts ? parts : kMaxParts;
  parts = parts < p.steps ? parts : p.steps;
  parts = parts > 1 ? parts : 1;
  p.part = div_up(p.steps, parts) * kStep;
  p.part = p.part > 0 ? p.part : kStep;
  p.parts = tokens > 0 ? div_up(tokens, p.part) : 1;
  p.of = p.parts > 1 ? div_up(12 * p.parts * units, 16) * 16 : 0;
  p.bytes = p.of + (ragged ? 4 * tokens : 0);
  return p;
}

bool recur_fits(int64_t tokens, int64_t units, int64_t sequences, int wide) {
  return batch_fits(tokens, units) && units <= kMaxLevel / 2 && sequences >= 0 && sequences <= kMaxSequences &&
         (wide == 0 || wide == 1);
}
int64_t recur_bytes(int64_t tokens, int64_t units, int64_t sequences, bool ragged) {
  if (units == 0 || (tokens == 0 && sequences == 0)) return 0;
  return recur_plan(tokens, units, ragged).bytes;
}

// The plan into the arguments, and the rows' sequences.
void recur_setup(RecurArgs& a, const RecurPlan& p, void* workspace, hipStream_t s) {
  a.part = p.part;
  a.sums = static_cast<float*>(workspace);
  if (!a.starts || a.tokens == 0) return;
  int* of = reinterpret_cast<int*>(static_cast<char*>(workspace) + p.of);
  a.of = of;
  k_recur_rows<<<static_cast<unsigned>(div_up(a.tokens, 256)), 256, 0, s>>>(a, of);
}

}  // namespace

extern "C" {

int64_t plx_recur_workspace(int64_t tokens, int64_t units, int64_t sequences, int32_t ragged) {
  if (!recur_fits(tokens, units, sequences, 0)) return -1;
  return recur_bytes(tokens, units, sequences, ragged != 0);
}

int plx_recur(int64_t tokens, int64_t units, int64_t sequences, int32_t dtype, const void* xz, int64_t line,
              const void* starts, int32_t wide, const float* state, void* h, float* last, float* kept,
              void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "plx_recur: bad size or null pointer";
  if (!recur_fits(tokens, units, sequences, wide)) return fail(PLX_ERR_INVALID, who);
  if (!known_type(dtype)) return fail(PLX_ERR_UNSUPPORTED, "plx_recur: unknown element type");
  if (!starts && sequences != 1) return fail(PLX_ERR_INVALID, who);
  if (units == 0 || (tokens == 0 && sequences == 0)) return PLX_OK;
  if ((tokens > 0 && (!xz || !h || !kept)) || (sequences > 0 && !last)) return fail(PLX_ERR_INVALID, who);
  const RecurPlan p = recur_plan(tokens, units, starts != nullptr);
  if (p.bytes > 0 && (!workspace || !on_16(workspace) || workspace_bytes < p.bytes))
    return fail(PLX_ERR_INVALID, "plx_recur: plx_recur_workspace() bytes on 16 bytes needed");
  hipStream_t s = static_cast<hipStream_t>(stream);
  RecurArgs a{};
  a.tokens = tokens, a.sequences = sequences, a.line = line, a.units = static_cast<int>(units), a.wide = wide;
  a.xz = xz, a.starts = starts, a.state = state, a.h = h, a.last = last, a.kept = kept;
  recur_setup(a, p, workspace, s);
  with_type(dtype, [&](auto* e) {
    using T = PLX_DENSE_TYPE(e);
    const unsigned slabs = static_cast<unsigned>(p.slabs), parts = static_cast<unsigned>(p.parts);
    if (parts > 1) k_recur_parts<T><<<dim3(slabs, parts - 1), 64 * kWaves, 0, s>>>(a);
    k_recur<T><<<dim3(slabs, parts), 64 * kWaves, 0, s>>>(a);
  });
  return check_launch("plx_recur");
}

int plx_recur_grad(int64_t tokens, int64_t units, int64_t sequences, int32_t dtype, const void* g, int64_t g_line,
                   const void* xz, int64_t line, const void* starts, int32_t wide, const float* state,
                   const float* g_last, const float* kept, void* dxz, float* dstate, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  const char* who = "plx_recur_grad: bad size or null pointer";
  if (!recur_fits(tokens, units, sequences, wide)) return fail(PLX_ERR_INVALID, who);
  if (!known_type(dtype)) return fail(PLX_ERR_UNSUPPORTED, "plx_recur_grad: unknown element type");
  if (!starts && sequences != 1) return fail(PLX_ERR_INVALID, who);
  if (units == 0 || (tokens == 0 && sequences == 0)) return PLX_OK;
  if ((tokens > 0 && (!xz || !g || !kept || !dxz)) || (sequences > 0 && !dstate)) return fail(PLX_ERR_INVALID, who);
  const RecurPlan p = recur_plan(tokens, units, starts != nullptr);
  if (p.bytes > 0 && (!workspace || !on_16(workspace) || workspace_bytes < p.bytes))
    return fail(PLX_ERR_INVALID, "plx_recur_grad: plx_recur_workspace() bytes on 16 bytes needed");
  hipStream_t s = static_cast<hipStream_t>(stream);
  RecurArgs a{};
  a.tokens = tokens, a.sequences = sequences, a.line = line, a.g_line = g_line, a.units = static_cast<int>(units);
  a.wide = wide, a.xz = xz, a.starts = starts, a.state = state, a.kept = const_cast<float*>(kept);
  a.g = g, a.g_last = g_last, a.dxz = dxz, a.dstate = dstate;
  recur_setup(a, p, workspace, s);
  with_type(dtype, [&](auto* e) {
    using T = PLX_DENSE_TYPE(e);
    const unsigned slabs = static_cast<unsigned>(p.slabs), parts = static_cast<unsigned>(p.parts);
    if (parts > 1) k_recur_grad_parts<T><<<dim3(slabs, parts - 1), 64 * kWaves, 0, s>>>(a);
    k_recur_grad<T><<<dim3(slabs, parts), 64 * kWaves, 0, s>>>(a);
  });
  return check_launch("plx_recur_grad");
}

int plx_recur_step(int64_t sequences, int64_t units, int32_t dtype, const void* xz, int64_t line, float* state,
                   int64_t state_line, void* h, void* stream) {
  if (!recur_fits(sequences, units, sequences, 0)) return fail(PLX_ERR_INVALID, "plx_recur_step: bad size");
  if (!known_type(dtype)) return fail(PLX_ERR_UNSUPPORTED, "plx_recur_step: unknown element type");
  if (sequences == 0 || units == 0) return PLX_OK;
  if (!xz || !state || !h) return fail(PLX_ERR_INVALID, "plx_recur_step: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t groups = div_up(sequences * div_up(units, 4), 256), most = int64_t{1} << 22;
  with_type(dtype, [&](auto* e) {
    using T = PLX_DENSE_TYPE(e);
    k_recur_step<T><<<static_cast<unsigned>(groups < most ? groups : most), 256, 0, s>>>(
        sequences, static_cast<int>(units), static_cast<const T*>(xz), line, state, state_line, static_cast<T*>(h));
  });
  return check_launch("plx_recur_step");
}

}  // extern "C"
