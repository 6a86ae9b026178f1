// px_dense.h -- pieces shared by the operators around dense level pairs:
// chunks of 16 bytes of a row, sums over a wave and over a workgroup, ids of 4
// or 8 bytes, and the host's dispatch by element type.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/plastax_hip.h"
#include "px_common.h"
#include "px_lowbit.h"

namespace px {

__host__ __device__ constexpr int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// N consecutive values as they are in memory, and as a load that needs no more
// than the values' own alignment.
template <typename T, int N>
struct Pack {
  typedef T type __attribute__((ext_vector_type(N)));
  typedef T load __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
// Values of T in 16 bytes.
template <typename T>
constexpr int kChunk = 16 / static_cast<int>(sizeof(T));

// p[i], i < n; `rest` from there on. PASS: what a pass reads once.
template <int N, bool PASS = false, typename T>
__device__ __forceinline__ typename Pack<T, N>::type load_pack(const T* p, int64_t n, float rest = 0.0f) {
  if (n >= N) {
    if (PASS) return __builtin_nontemporal_load(reinterpret_cast<const typename Pack<T, N>::load*>(p));
    return *reinterpret_cast<const typename Pack<T, N>::load*>(p);
  }
  typename Pack<T, N>::type r;
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = i < n ? p[i] : from_f32<T>(rest);
  return r;
}
// p[i] = v[i], i < n. PASS: results that nothing in the pass reads.
template <int N, bool PASS = false, typename T>
__device__ __forceinline__ void store_pack(T* p, int64_t n, const float* v) {
  if (n >= N) {
    typename Pack<T, N>::load r;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = from_f32<T>(v[i]);
    if (PASS)
      __builtin_nontemporal_store(r, reinterpret_cast<typename Pack<T, N>::load*>(p));
    else
      *reinterpret_cast<typename Pack<T, N>::load*>(p) = r;
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) p[i] = from_f32<T>(v[i]);
}

// Whole numbers of 4 or 8 bytes.
__device__ __forceinline__ int64_t load_id(const void* p, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// Over a wave's lanes, the same in all of them: within rows of 16 lanes, then
// over the rows, by the vector unit's own lane shifts (a shuffle goes through
// LDS); always in the same order.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ float from_lane(float v, float other) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(__float_as_int(other), __float_as_int(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float last_lane(float v) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += from_lane<0x111>(v, 0.0f);  // from 1, 2, 4, 8 lanes below in the row
  v += from_lane<0x112>(v, 0.0f);
  v += from_lane<0x114>(v, 0.0f);
  v += from_lane<0x118>(v, 0.0f);
  v += from_lane<0x142, 0xA>(v, 0.0f);  // rows 0 and 2 to 1 and 3
  v += from_lane<0x143, 0xC>(v, 0.0f);  // both to rows 2 and 3
  return last_lane(v);
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, from_lane<0x111>(v, v));
  v = fmaxf(v, from_lane<0x112>(v, v));
  v = fmaxf(v, from_lane<0x114>(v, v));
  v = fmaxf(v, from_lane<0x118>(v, v));
  v = fmaxf(v, from_lane<0x142, 0xA>(v, v));
  v = fmaxf(v, from_lane<0x143, 0xC>(v, v));
  return last_lane(v);
}

template <typename F>
void with_type(int dtype, F f) {
  if (dtype == PLX_LB_F32)
    f(static_cast<float*>(nullptr));
  else if (dtype == PLX_LB_BF16)
    f(static_cast<__bf16*>(nullptr));
  else
    f(static_cast<_Float16*>(nullptr));
}
#define PLX_DENSE_TYPE(p) typename std::remove_pointer<decltype(p)>::type

inline bool known_type(int dtype) { return dtype == PLX_LB_F32 || dtype == PLX_LB_BF16 || dtype == PLX_LB_F16; }
inline bool on_16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
constexpr int64_t kMaxRows = int64_t{1} << 30, kMaxLevel = int64_t{1} << 24;  // tokens; units of a level, ids
inline bool batch_fits(int64_t tokens, int64_t units) {
  return tokens >= 0 && units >= 0 && tokens <= kMaxRows && units <= kMaxLevel;
}

}  // namespace px
