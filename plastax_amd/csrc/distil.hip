// distil.hip -- a level of outputs learned from a teacher that named a few of
// them: the loss of each token and its gradient. No counterpart in the
// reference, whose losses read whole target columns.
//
// With q = softmax(x / T) over a token's outputs and p = softmax(t / T) over
// its named ones, loss = T^2 sum p (log p - log q) and
// d loss / dx = T (q - p), p 0 where nothing is named.
//
// Bound by memory: a row is read once into registers, its largest logit, its
// sum and its gradient are made from there, and the gradient is written once:
// 8192 x 131072 bf16 858 us, 5.0 TB/s.

#include "px_dense.h"

using plx_detail::check_launch;
using plx_detail::cu_count;
using plx_detail::fail;

namespace {

using namespace px;

constexpr float kLog2e = 1.44269504088896341f;
constexpr double kLn2 = 0.693147180559945309;

struct DistilArgs {
  int64_t tokens, outputs, line;
  const void* x;
  const void* ids;
  const void* top;
  const float* g;
  float* loss;
  void* dx;
  int named, wide, top_type;
  int whole;  // the gradient's rows begin on 64 bytes: its stores go past the caches (in rows that do not they
              // would leave parts of lines: 2048 x 32003 bf16 60 us, past the caches 65)
  float t;    // the temperature
};

__device__ __forceinline__ float load_top(const DistilArgs& a, int64_t i) {
  if (a.top_type == PLX_LB_F32) return static_cast<const float*>(a.top)[i];
  if (a.top_type == PLX_LB_BF16) return to_f32(static_cast<const __bf16*>(a.top)[i]);
  return to_f32(static_cast<const _Float16*>(a.top)[i]);
}

// log2 of v > 0: its exponent, and the logarithm of a value from 0.5 to 1, so
// that large sums lose nothing.
__device__ __forceinline__ double log2_of(float v) {
  if (!(v < INFINITY)) return v;  // (an infinity or a NaN)
  return static_cast<double>(__builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(v))) +
         static_cast<double>(__builtin_amdgcn_frexp_expf(v));
}

// A place of the teacher's: its weight p, the output (-1: none), its logit and
// the teacher's.
struct Named {
  double p;
  int id;
  float x, top;
};
struct Teacher {
  double largest, log_sum;  // of the teacher's logits; of exp((t - largest) / T)
  bool any;
};

// One wave's: a token's places. In 64 bits, with log p kept apart, for the loss
// is a difference of logarithms (64 of 131072 outputs: nothing beside the row).
template <typename T>
__device__ __forceinline__ Teacher name_outputs(const DistilArgs& a, int64_t token, const T* row, Named* named) {
  const int lane = threadIdx.x & 63;
  const double inv_t = 1.0 / a.t;
  float m = -INFINITY;
  bool any = false;
  for (int i = lane; i < a.named; i += 64) {
    const int64_t id = load_id(a.ids, a.wide, token * a.named + i);
    const float t = load_top(a, token * a.named + i);
    const bool there = id >= 0 && id < a.outputs && t != -INFINITY;
    named[i] = {0.0, there ? static_cast<int>(id) : -1, there ? to_f32(row[id]) : 0.0f, t};
    any |= there;
    if (there) m = fmaxf(m, t);
  }
  m = wave_max(m);
  double sum = 0.0;
  for (int i = lane; i < a.named; i += 64) {
    const double p = named[i].id >= 0 ? exp((static_cast<double>(named[i].top) - m) * inv_t) : 0.0;
    named[i].p = p;
    sum += p;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64);
  const double inv = 1.0 / sum;
  for (int i = lane; i < a.named; i += 64) named[i].p *= inv;  // (only read where an output is named)
  return {m, log(sum), __any(any) != 0};
}

// What a row's values are taken from before the exponential: a logit's is
// 2^(x c - shift), one operation, with the rounding of shift = m c in all of a
// row's exponents alike: half a unit at most while |m c| < 2^24, and taken out
// of the loss again. From there on, where it would grow until the powers
// overflow or vanish, a logit's is 2^((x - m) c), whose exponents are rounded
// relative to themselves.
struct Shift {
  float c, m, shift;
  bool far;
};
__device__ __forceinline__ Shift shift_of(float m, float t) {
  Shift s;
  s.c = kLog2e / t, s.m = m, s.shift = m * s.c;
  s.far = !(fabsf(s.shift) < 16777216.0f);  // (a NaN is far)
  return s;
}
template <bool FAR>
__device__ __forceinline__ float power(float x, const Shift& s) {
  return __builtin_amdgcn_exp2f(FAR ? (x - s.m) * s.c : __builtin_fmaf(x, s.c, -s.shift));
}

// One wave's: the token's loss, from the sum of its outputs' powers (and what
// the shift's rounding put into all of them).
__device__ __forceinline__ void write_loss(const DistilArgs& a, int64_t token, const Shift& s, float sum,
                                           const Teacher& t, const Named* named) {
  const int lane = threadIdx.x & 63;
  const double inv_t = 1.0 / a.t;
  const double log_q = kLn2 * (log2_of(sum) - (s.far ? 0.0 : static_cast<double>(s.m) * s.c - s.shift));
  double loss = 0.0;
  for (int i = lane; i < a.named; i += 64) {
    const Named v = named[i];
    const double d = ((v.top - t.largest) - (static_cast<double>(v.x) - s.m)) * inv_t - t.log_sum + log_q;
    if (v.id >= 0 && v.p != 0.0) loss += v.p * d;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) loss += __shfl_xor(loss, d, 64);
  if (lane == 0) a.loss[token] = t.any ? static_cast<float>(loss * a.t * a.t) : 0.0f;
}

// The gradient at the named outputs, after the others' (the same output named
// twice is written twice with the same value).
template <int NT, typename T>
__device__ __forceinline__ void write_named(const DistilArgs& a, T* out, const Shift& s, float scale, float r,
                                            const Named* named) {
  for (int i = threadIdx.x % NT; i < a.named; i += NT) {
    const Named v = named[i];
    if (v.id < 0) continue;
    double p = 0.0;
    for (int j = 0; j < a.named; ++j) p += named[j].id == v.id ? named[j].p : 0.0;
    const float q = s.far ? power<true>(v.x, s) : power<false>(v.x, s);
    out[v.id] = from_f32<T>(static_cast<float>(static_cast<double>(q) * r - p * scale));
  }
}

// The waves' values joined, the same in every lane.
template <int WAVES, typename F>
__device__ __forceinline__ float over_waves(float v, float* part, F f) {
  if (WAVES == 1) return v;
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[threadIdx.x & (WAVES - 1)];
#pragma unroll
  for (int d = 1; d < WAVES; d *= 2) v = f(v, __shfl_xor(v, d, 64));
  return v;
}

// A row's chunks of 16 bytes without a branch in their loads: chunks past the
// last whole one are read as the row's last 16 bytes, of which the values
// behind the last whole chunk are its rest. (Rows of less than a chunk are
// read value by value.)
template <typename T, int NT, int NC>
struct RowChunks {
  static constexpr int W = kChunk<T>;
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  words v[NC];
  int lane;
  __device__ __forceinline__ int at(int k) const { return (k * NT + lane) * W; }
  __device__ __forceinline__ void load(const T* row, int outputs) {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      if (NC == 1 && NT == 64 && outputs < W)
        v[k] = __builtin_bit_cast(words, load_pack<W>(row + at(k), outputs - at(k), -INFINITY));
      else
        v[k] = __builtin_bit_cast(words, __builtin_nontemporal_load(chunk<const typename Pack<T, W>::load>(
                                             row, at(k) + W <= outputs ? at(k) : outputs - W)));
    }
  }
  // The chunk at a value of a row (by the row's address, the same in all lanes,
  // and a lane's 32 bits).
  template <typename V, typename R>
  __device__ __forceinline__ static V* chunk(R* row, int at) {
    typedef typename std::conditional<std::is_const<V>::value, const char, char>::type byte;
    return reinterpret_cast<V*>(reinterpret_cast<byte*>(row) + static_cast<unsigned>(at * static_cast<int>(sizeof(T))));
  }
  __device__ __forceinline__ float get(int k, int i) const {
    return to_f32(__builtin_bit_cast(typename Pack<T, W>::type, v[k])[i]);
  }
  // As new to the compiler, which would keep every value as float32 from one
  // pass over them to the next, and every chunk's place.
  __device__ __forceinline__ void again() {
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int k = 0; k < NC; ++k) asm volatile("" : "+v"(v[k]));
  }
  __device__ __forceinline__ float largest() const {
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i) m = fmaxf(m, get(k, i));
    return m;
  }
  // f(k, first): values from `first` to W of the lane's chunk k are the row's.
  template <typename F>
  __device__ __forceinline__ void each(int outputs, F f) const {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      if (at(k) + W <= outputs)
        f(k, 0);
      else if (at(k) < outputs)
        f(k, outputs < W ? 0 : at(k) + W - outputs);
    }
  }
  template <bool FAR>
  __device__ __forceinline__ float sum(int outputs, const Shift& s) const {
    float all = 0.0f;
    each(outputs, [&](int k, int first) {
      float part = 0.0f;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float e = power<FAR>(get(k, i), s);
        part += i < first || (NC == 1 && i >= outputs) ? 0.0f : e;
      }
      all += part;
    });
    return all;
  }
  template <bool FAR>
  __device__ __forceinline__ void gradient(T* out, int outputs, int whole, const Shift& s, float r) const {
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (at(k) < outputs) gradient<FAR>(out, outputs, whole, s, r, k);
  }
  template <bool FAR>
  __device__ __forceinline__ void gradient(T* out, int outputs, int whole, const Shift& s, float r, int k) const {
    float d[W];
#pragma unroll
    for (int i = 0; i < W; ++i) d[i] = power<FAR>(get(k, i), s) * r;
    if (at(k) + W <= outputs) {
      typename Pack<T, W>::load y;
#pragma unroll
      for (int i = 0; i < W; ++i) y[i] = from_f32<T>(d[i]);
      typename Pack<T, W>::load* p = chunk<typename Pack<T, W>::load>(out, at(k));
      if (whole) {
        __builtin_nontemporal_store(y, p);
      } else {
        asm volatile("");  // (or the two become one store, through the caches)
        *p = y;
        asm volatile("");
      }
    } else if (outputs < W) {
      store_pack<W>(out, outputs, d);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i >= at(k) + W - outputs) out[outputs - W + i] = from_f32<T>(d[i]);
    }
  }
  __device__ __forceinline__ void zeros(T* out, int outputs) const {
    const float d[W] = {};
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (at(k) < outputs) store_pack<W>(out + at(k), outputs - at(k), d);
  }
};

// A workgroup a token. The row stays in registers, NC chunks a lane: it is read
// once and its gradient written once. The first wave looks at the teacher's
// places before it loads the row (registers).
template <typename T, int WAVES, int NC, bool GRAD>
__global__ __launch_bounds__(WAVES * 64) void k_distil_row(DistilArgs a) {
  constexpr int NT = WAVES * 64;
  extern __shared__ Named named[];
  __shared__ float part[2][WAVES];
  __shared__ int some;
  const int64_t token = blockIdx.x;
  const int outputs = static_cast<int>(a.outputs);
  const bool first = WAVES == 1 || threadIdx.x < 64;
  const T* row = static_cast<const T*>(a.x) + token * a.line;
  Teacher teacher{};
  if (first) teacher = name_outputs(a, token, row, named);
  if (WAVES > 1 && threadIdx.x == 0) some = teacher.any;
  RowChunks<T, NT, NC> chunks;
  chunks.lane = threadIdx.x;
  if (outputs > 0) chunks.load(row, outputs);
  const float m = over_waves<WAVES>(wave_max(outputs > 0 ? chunks.largest() : -INFINITY), part[0],
                                    [](float a, float b) { return fmaxf(a, b); });
  const Shift s = shift_of(m, a.t);
  chunks.again();
  float sum = wave_sum(s.far ? chunks.template sum<true>(outputs, s) : chunks.template sum<false>(outputs, s));
  sum = over_waves<WAVES>(sum, part[1], [](float a, float b) { return a + b; });
  if (GRAD) {
    T* out = static_cast<T*>(a.dx) + token * a.outputs;
    const float scale = a.g[token] * a.t, r = scale / sum;
    chunks.again();
    if (!(WAVES > 1 ? some != 0 : teacher.any))
      chunks.zeros(out, outputs);
    else if (s.far)
      chunks.template gradient<true>(out, outputs, a.whole, s, r);
    else
      chunks.template gradient<false>(out, outputs, a.whole, s, r);
    if (WAVES > 1)
      __syncthreads();
    else  // (a wave's stores are made in their order, and its lanes see each other's: for the compiler)
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    write_named<NT>(a, out, s, scale, r, named);
  }
  if (first) write_loss(a, token, s, sum, teacher, named);
}

// Rows that no registers hold: a lane's largest logit and its sum go along the
// row together, and the gradient reads the row again.
template <typename T, bool GRAD>
__global__ __launch_bounds__(1024) void k_distil_stream(DistilArgs a) {
  constexpr int W = kChunk<T>, WAVES = 16, NT = 1024;
  extern __shared__ Named named[];
  __shared__ float part[2][WAVES];
  __shared__ int some;
  const int64_t token = blockIdx.x;
  const T* row = static_cast<const T*>(a.x) + token * a.line;
  Teacher teacher{};
  if (threadIdx.x < 64) teacher = name_outputs(a, token, row, named);
  if (threadIdx.x == 0) some = teacher.any;
  const float c = kLog2e / a.t;
  float m = -INFINITY, sum = 0.0f;
  for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.outputs; at += NT * W) {
    const typename Pack<T, W>::type v = load_pack<W>(row + at, a.outputs - at, -INFINITY);
    float top = m, more = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) top = fmaxf(top, to_f32(v[i]));
    const float from = top == -INFINITY ? 0.0f : top;  // (a lane without a logit above -inf has the sum 0)
#pragma unroll
    for (int i = 0; i < W; ++i) more += __builtin_amdgcn_exp2f((to_f32(v[i]) - from) * c);
    sum = sum * (m == top ? 1.0f : __builtin_amdgcn_exp2f((m - top) * c)) + more;
    m = top;
  }
  const float own = m;
  m = over_waves<WAVES>(wave_max(m), part[0], [](float a, float b) { return fmaxf(a, b); });
  sum = wave_sum(sum * (own == m ? 1.0f : __builtin_amdgcn_exp2f((own - m) * c)));
  sum = over_waves<WAVES>(sum, part[1], [](float a, float b) { return a + b; });
  Shift s = shift_of(m, a.t);
  s.far = true;  // (as the sum was made)
  if (GRAD) {
    T* out = static_cast<T*>(a.dx) + token * a.outputs;
    const float scale = a.g[token] * a.t, r = scale / sum;
    const bool any = some != 0;
    for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.outputs; at += NT * W) {
      const typename Pack<T, W>::type v = load_pack<W, true>(row + at, a.outputs - at);
      float d[W];
#pragma unroll
      for (int i = 0; i < W; ++i) d[i] = any ? power<true>(to_f32(v[i]), s) * r : 0.0f;
      store_pack<W, true>(out + at, a.outputs - at, d);
    }
    __syncthreads();
    write_named<NT>(a, out, s, scale, r, named);
  }
  if (threadIdx.x < 64) write_loss(a, token, s, sum, teacher, named);
}

template <typename T, int WAVES, int NC, bool GRAD>
void launch_row(const DistilArgs& a, hipStream_t s) {
  k_distil_row<T, WAVES, NC, GRAD>
      <<<static_cast<unsigned>(a.tokens), WAVES * 64, a.named * sizeof(Named), s>>>(a);
}

// Few waves with many chunks where there are tokens enough for every CU (a
// token's places are looked at by one wave, for which the others wait: 2048 x
// 3800 float32 15 us, with 16 waves 30), else many with few (200 x 3800 6.3 us,
// with 2 waves 7.0; 1 x 3800 5.5 and 6.3). A row stays in registers as long as
// it fits there (2048 x 60000 float32 184 us, as a stream 216; 32 x 60000 10.9
// and 13.9).
template <typename T, bool GRAD>
void launch_distil(const DistilArgs& a, hipStream_t s) {
  const int64_t chunks = div_up(a.outputs, kChunk<T>);
  const bool few = a.tokens < 2 * cu_count();
  if (chunks <= 64)
    launch_row<T, 1, 1, GRAD>(a, s);
  else if (chunks <= 256 && few)
    launch_row<T, 4, 1, GRAD>(a, s);
  else if (chunks <= 128)
    launch_row<T, 1, 2, GRAD>(a, s);
  else if (chunks <= 256)
    launch_row<T, 1, 4, GRAD>(a, s);
  else if (chunks <= 1024 && few)
    launch_row<T, 16, 1, GRAD>(a, s);
  else if (chunks <= 512)
    launch_row<T, 2, 4, GRAD>(a, s);
  else if (chunks <= 1024)
    launch_row<T, 2, 8, GRAD>(a, s);
  else if (chunks <= 2048)
    launch_row<T, 4, 8, GRAD>(a, s);
  else if (chunks <= 4096)
    launch_row<T, 8, 8, GRAD>(a, s);
  else if (chunks <= 8192)
    launch_row<T, 16, 8, GRAD>(a, s);
  else if (chunks <= 16384)
    launch_row<T, 16, 16, GRAD>(a, s);
  else
    k_distil_stream<T, GRAD><<<static_cast<unsigned>(a.tokens), 1024, a.named * sizeof(Named), s>>>(a);
}

int run_distil(const char* who, bool grad, const DistilArgs& all, int dtype, void* stream) {
  if (!batch_fits(all.tokens, all.outputs) || all.named < 0 || all.named > PLX_MAX_NAMED || all.wide < 0 || all.wide > 1)
    return fail(PLX_ERR_INVALID, who);
  if (!known_type(dtype) || !known_type(all.top_type)) return fail(PLX_ERR_UNSUPPORTED, who);
  if (!(all.t >= 0x1p-120f && all.t <= 0x1p120f)) return fail(PLX_ERR_INVALID, who);  // (1 / T is normal too)
  if (all.tokens == 0) return PLX_OK;
  if (!all.loss || (all.outputs > 0 && !all.x) || (all.named > 0 && (!all.ids || !all.top)) ||
      (grad && (!all.g || (all.outputs > 0 && !all.dx))))
    return fail(PLX_ERR_INVALID, who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  constexpr int64_t most = int64_t{1} << 20;  // tokens of a launch: at most 2^30 lanes
  with_type(dtype, [&](auto* e) {
    using T = PLX_DENSE_TYPE(e);
    for (int64_t first = 0; first < all.tokens; first += most) {
      DistilArgs a = all;
      a.tokens = all.tokens - first < most ? all.tokens - first : most;
      a.x = static_cast<const T*>(all.x) + first * all.line;
      a.ids = static_cast<const char*>(all.ids) + first * all.named * (all.wide ? 8 : 4);
      a.top = static_cast<const char*>(all.top) + first * all.named * (all.top_type == PLX_LB_F32 ? 4 : 2);
      a.loss = all.loss + first;
      if (grad) {
        a.g = all.g + first;
        a.dx = static_cast<T*>(all.dx) + first * all.outputs;
        a.whole = ((reinterpret_cast<uintptr_t>(a.dx) | (a.outputs * sizeof(T))) & 63) == 0;
        launch_distil<T, true>(a, s);
      } else {
        launch_distil<T, false>(a, s);
      }
    }
  });
  return check_launch(who);
}

}  // namespace

extern "C" {

int plx_distil(int64_t tokens, int64_t outputs, int32_t named, int32_t dtype, const void* logits, int64_t line,
               const void* ids, int32_t wide, int32_t top_type, const void* top, float temperature, float* loss,
               void* stream) {
  DistilArgs a{};
  a.tokens = tokens, a.outputs = outputs, a.line = line, a.x = logits, a.ids = ids, a.top = top, a.loss = loss;
  a.named = named, a.wide = wide, a.top_type = top_type, a.t = temperature;
  return run_distil("plx_distil: bad size, type, temperature or null pointer", false, a, dtype, stream);
}

int plx_distil_grad(int64_t tokens, int64_t outputs, int32_t named, const float* g, int32_t dtype, const void* logits,
                    int64_t line, const void* ids, int32_t wide, int32_t top_type, const void* top, float temperature,
                    float* loss, void* dlogits, void* stream) {
  DistilArgs a{};
  a.tokens = tokens, a.outputs = outputs, a.line = line, a.x = logits, a.ids = ids, a.top = top, a.loss = loss;
  a.g = g, a.dx = dlogits;
  a.named = named, a.wide = wide, a.top_type = top_type, a.t = temperature;
  return run_distil("plx_distil_grad: bad size, type, temperature or null pointer", true, a, dtype, stream);
}

}  // extern "C"
