// distil.hip -- a level of outputs learned from a teacher that named a few of
// them: the loss of each token and its gradient. No counterpart in the
// reference, whose losses read whole target columns.
//
// With q = softmax(x / T) over a token's outputs and p = softmax(t / T) over
// its named ones, loss = T^2 sum p (log p - log q) and
// d loss / dx = T (q - p), p 0 where nothing is named.

#include "px_dense.h"

using plx_detail::check_launch;
using plx_detail::fail;

namespace {

using namespace px;

constexpr int kNamed = PLX_MAX_NAMED;  // named outputs of a token at most: what they need is in LDS

struct DistilArgs {
  int64_t tokens, outputs, line;
  const void* x;
  const void* ids;
  const void* top;
  const float* g;
  float* loss;
  void* dx;
  int named, wide, top_type;
  float t;  // the temperature
};

// What a workgroup's waves share.
template <int WAVES>
struct DistilShared {
  float top[WAVES], sum[WAVES];
  float x[kNamed];
  double p[kNamed], log_p[kNamed];
  int id[kNamed];  // -1: names nothing
  int any;
};

__device__ __forceinline__ float load_top(const DistilArgs& a, int64_t i) {
  if (a.top_type == PLX_LB_F32) return static_cast<const float*>(a.top)[i];
  if (a.top_type == PLX_LB_BF16) return to_f32(static_cast<const __bf16*>(a.top)[i]);
  return to_f32(static_cast<const _Float16*>(a.top)[i]);
}

// The waves' values joined, the same in every lane.
template <int WAVES, typename F>
__device__ __forceinline__ float over_waves(const float* part, F f) {
  float v = part[threadIdx.x & (WAVES - 1)];
#pragma unroll
  for (int d = 1; d < WAVES; d *= 2) v = f(v, __shfl_xor(v, d, 64));
  return v;
}

// The first wave's: the token's named outputs, their weights p, log p and
// logits. In 64 bits, for the loss is a difference of logarithms (64 of 131072
// outputs: nothing beside the row).
template <int WAVES, typename T>
__device__ __forceinline__ void name_outputs(const DistilArgs& a, int64_t token, const T* row,
                                             DistilShared<WAVES>& sh) {
  const int lane = threadIdx.x;
  double m = -INFINITY;
  bool any = false;
  for (int i = lane; i < a.named; i += 64) {
    const int64_t id = load_id(a.ids, a.wide, token * a.named + i);
    const float t = load_top(a, token * a.named + i);
    const bool there = id >= 0 && id < a.outputs && t != -INFINITY;
    sh.id[i] = there ? static_cast<int>(id) : -1;
    sh.x[i] = there ? to_f32(row[id]) : 0.0f;
    sh.log_p[i] = t;
    any |= there;
    if (there) m = fmax(m, static_cast<double>(t));
  }
  any = __any(any);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) m = fmax(m, __shfl_xor(m, d, 64));
  double sum = 0.0;
  for (int i = lane; i < a.named; i += 64) {
    const double l = (sh.log_p[i] - m) / a.t, e = sh.id[i] >= 0 ? exp(l) : 0.0;
    sh.log_p[i] = l;
    sh.p[i] = e;
    sum += e;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64);
  const double log_sum = log(sum);
  for (int i = lane; i < a.named; i += 64) {
    sh.p[i] /= sum;  // (only read where an output is named)
    sh.log_p[i] -= log_sum;
  }
  if (lane == 0) sh.any = any;
}

// The first wave's: the token's loss, from the row's largest logit and the sum
// of exp((x - m) / T).
template <int WAVES>
__device__ __forceinline__ void write_loss(const DistilArgs& a, int64_t token, float m, float sum,
                                           const DistilShared<WAVES>& sh) {
  const int lane = threadIdx.x;
  const double log_sum = log(static_cast<double>(sum));
  double loss = 0.0;
  for (int i = lane; i < a.named; i += 64) {
    const double p = sh.p[i];
    if (sh.id[i] >= 0 && !(p == 0.0))
      loss += p * (sh.log_p[i] - (static_cast<double>(sh.x[i]) - m) / a.t + log_sum);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) loss += __shfl_xor(loss, d, 64);
  if (lane == 0) a.loss[token] = sh.any ? static_cast<float>(loss * a.t * a.t) : 0.0f;
}

// The gradient at the named outputs, after the others' (the same output named
// twice is written twice with the same value).
template <int WAVES, typename T>
__device__ __forceinline__ void write_named(const DistilArgs& a, T* out, float m, float c, float scale, float sum,
                                            const DistilShared<WAVES>& sh) {
  for (int i = threadIdx.x; i < a.named; i += WAVES * 64) {
    const int id = sh.id[i];
    if (id < 0) continue;
    double p = 0.0;
    for (int j = 0; j < a.named; ++j) p += sh.id[j] == id ? sh.p[j] : 0.0;
    const double q = static_cast<double>(__builtin_amdgcn_exp2f((sh.x[i] - m) * c)) / sum;
    out[id] = from_f32<T>(static_cast<float>((q - p) * scale));
  }
}

// A workgroup per token. The row stays in registers, NC chunks of 16 bytes a
// lane: it is read once and its gradient written once.
template <typename T, int WAVES, int NC, bool GRAD>
__global__ __launch_bounds__(WAVES * 64) void k_distil_row(DistilArgs a) {
  constexpr int W = kChunk<T>, NT = WAVES * 64;
  __shared__ DistilShared<WAVES> sh;
  const int64_t token = blockIdx.x;
  const T* row = static_cast<const T*>(a.x) + token * a.line;
  typename Pack<T, W>::type v[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int64_t at = (static_cast<int64_t>(k) * NT + threadIdx.x) * W;
    v[k] = load_pack<W, true>(row + at, a.outputs - at, -INFINITY);
  }
  if (threadIdx.x < 64) name_outputs<WAVES>(a, token, row, sh);
  const float c = 1.44269504088896341f / a.t;
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int i = 0; i < W; ++i) m = fmaxf(m, to_f32(v[k][i]));
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) sh.top[threadIdx.x >> 6] = m;
  __syncthreads();
  m = over_waves<WAVES>(sh.top, [](float a, float b) { return fmaxf(a, b); });
  // (x - m first: logits of the type's lowest value, and rows of nothing else,
  // stay finite)
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    if ((static_cast<int64_t>(k) * NT + threadIdx.x) * W >= a.outputs) break;
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float x = to_f32(v[k][i]);
      part += __builtin_amdgcn_exp2f((x - m) * c);
    }
    sum += part;
  }
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) sh.sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = over_waves<WAVES>(sh.sum, [](float a, float b) { return a + b; });
  if (threadIdx.x < 64) write_loss<WAVES>(a, token, m, sum, sh);
  if (!GRAD) return;
  T* out = static_cast<T*>(a.dx) + token * a.outputs;
  const bool any = sh.any;
  const float scale = a.g[token] * a.t, r = scale / sum;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int64_t at = (static_cast<int64_t>(k) * NT + threadIdx.x) * W;
    if (at >= a.outputs) break;
    float d[W];
#pragma unroll
    for (int i = 0; i < W; ++i)
      d[i] = any ? __builtin_amdgcn_exp2f((to_f32(v[k][i]) - m) * c) * r : 0.0f;
    store_pack<W, true>(out + at, a.outputs - at, d);
  }
  __syncthreads();
  write_named<WAVES>(a, out, m, c, scale, sum, sh);
}

// Rows that no registers hold: a lane's largest logit and its sum go along the
// row together, and the gradient reads the row again.
template <typename T, bool GRAD>
__global__ __launch_bounds__(1024) void k_distil_stream(DistilArgs a) {
  constexpr int W = kChunk<T>, WAVES = 16, NT = 1024;
  __shared__ DistilShared<WAVES> sh;
  const int64_t token = blockIdx.x;
  const T* row = static_cast<const T*>(a.x) + token * a.line;
  if (threadIdx.x < 64) name_outputs<WAVES>(a, token, row, sh);
  const float c = 1.44269504088896341f / a.t;
  float m = -INFINITY, sum = 0.0f;
  for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.outputs; at += NT * W) {
    const typename Pack<T, W>::type v = load_pack<W>(row + at, a.outputs - at, -INFINITY);
    float top = m, part = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) top = fmaxf(top, to_f32(v[i]));
    const float from = top == -INFINITY ? 0.0f : top;  // (a lane without a logit above -inf has the sum 0)
#pragma unroll
    for (int i = 0; i < W; ++i) part += __builtin_amdgcn_exp2f((to_f32(v[i]) - from) * c);
    sum = sum * (m == top ? 1.0f : __builtin_amdgcn_exp2f((m - top) * c)) + part;
    m = top;
  }
  const float own = m;
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) sh.top[threadIdx.x >> 6] = m;
  __syncthreads();
  m = over_waves<WAVES>(sh.top, [](float a, float b) { return fmaxf(a, b); });
  sum = wave_sum(sum * (own == m ? 1.0f : __builtin_amdgcn_exp2f((own - m) * c)));
  if ((threadIdx.x & 63) == 0) sh.sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = over_waves<WAVES>(sh.sum, [](float a, float b) { return a + b; });
  if (threadIdx.x < 64) write_loss<WAVES>(a, token, m, sum, sh);
  if (!GRAD) return;
  T* out = static_cast<T*>(a.dx) + token * a.outputs;
  const bool any = sh.any;
  const float scale = a.g[token] * a.t, r = scale / sum;
  for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.outputs; at += NT * W) {
    const typename Pack<T, W>::type v = load_pack<W, true>(row + at, a.outputs - at);
    float d[W];
#pragma unroll
    for (int i = 0; i < W; ++i) d[i] = any ? __builtin_amdgcn_exp2f((to_f32(v[i]) - m) * c) * r : 0.0f;
    store_pack<W, true>(out + at, a.outputs - at, d);
  }
  __syncthreads();
  write_named<WAVES>(a, out, m, c, scale, sum, sh);
}

template <typename T, bool GRAD>
void launch_distil(const DistilArgs& a, hipStream_t s) {
  const unsigned rows = static_cast<unsigned>(a.tokens);
  const int64_t chunks = div_up(a.outputs, kChunk<T>);
  if (chunks <= 64)
    k_distil_row<T, 1, 1, GRAD><<<rows, 64, 0, s>>>(a);
  else if (chunks <= 256)
    k_distil_row<T, 4, 1, GRAD><<<rows, 256, 0, s>>>(a);
  else if (chunks <= 512)
    k_distil_row<T, 4, 2, GRAD><<<rows, 256, 0, s>>>(a);
  else if (chunks <= 1024)
    k_distil_row<T, 4, 4, GRAD><<<rows, 256, 0, s>>>(a);
  else if (chunks <= 2048)
    k_distil_row<T, 8, 4, GRAD><<<rows, 512, 0, s>>>(a);
  else if (chunks <= 4096)
    k_distil_row<T, 16, 4, GRAD><<<rows, 1024, 0, s>>>(a);
  else if (chunks <= 8192)
    k_distil_row<T, 16, 8, GRAD><<<rows, 1024, 0, s>>>(a);
  else
    k_distil_stream<T, GRAD><<<rows, 1024, 0, s>>>(a);
}

int run_distil(const char* who, bool grad, const DistilArgs& all, int dtype, void* stream) {
  if (!batch_fits(all.tokens, all.outputs) || all.named < 0 || all.named > kNamed || all.wide < 0 || all.wide > 1)
    return fail(PLX_ERR_INVALID, who);
  if (!known_type(dtype) || !known_type(all.top_type)) return fail(PLX_ERR_UNSUPPORTED, who);
  if (!(all.t > 0.0f && all.t < INFINITY)) return fail(PLX_ERR_INVALID, who);
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
