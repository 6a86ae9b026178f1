// recur.hip -- a level carried along sequences by a gated linear recurrence,
// its gradients, and one token at a time. No counterpart in the reference,
// whose PIPELINE nets carry state from step to step only.
//
// a = sigmoid(z), h[t] = a[t] h[t-1] + (1 - a[t]) x[t] for each unit, from the
// sequence's state. Backwards c[t] = g[t] + a[t+1] c[t+1] (at a sequence's
// last row plus its last state's gradient), dx = (1 - a) c,
// dz = a (1 - a) (h[t-1] - x) c, and a c of its first row is the state's.
//
// Rows as maps h -> A h + H compose, so rows can be summed up before what comes
// in is known. A workgroup takes a tile, a few rows a wave of kSlab units, into
// its registers, two units a lane; its waves' sums meet in LDS, the
// tiles' in memory, and each wave walks its rows again from what comes in: xz
// is read once. Tiles are taken in the order of a counter (a slab's), and wait
// for earlier ones of their own slab only (lane_of's words), which are under
// way: every wait ends, in whatever order the slabs' workgroups begin. (It is
// bounded too, for a caller who has two calls share a workspace: NaN then.) A
// tile waits for the sums of the tiles before it in its group of 8, for those of
// the groups before in the row of 8 groups, and for what comes into the row: a
// long sequence is a chain of rows of 64 tiles (a link takes some 3 us), and
// every sum has one order.
//
// 65536 x 1024 bf16: 117 us forwards for 403 MB, 3.4 TB/s, and 216 backwards for
// 671 MB, 3.1: a workgroup's way through a tile (its turn, its loads, the
// exchange in LDS, what it waits for, its stores) takes some 12 us, and the two
// that a CU holds do not cover each other's all the time. Smaller tiles with
// the next one's loads on their way took 185 and 368, four workgroups of half
// the rows 136 forwards.

#include "px_dense.h"
#include "px_recur.h"

using plx_detail::check_launch;
using plx_detail::fail;

namespace {

using namespace px;

constexpr int kWaves = 8;                 // of a tile
constexpr int kForth = 16, kBack = 8;     // rows of a wave forwards, and of the gradients' (registers)
static_assert(kWaves >= 8, "a wave for each of a group's tiles before the last, and one");
constexpr int kKeep = kWaves * kBack;     // rows of the gradients' tile: what comes into it is kept
static_assert(kKeep == PLX_RECUR_KEEP && kKeep % kForth == 0, "a wave begins where its h is kept");
constexpr int kTicket = 64;  // (a counter takes an atomic addition each 20 ns: one for all slabs took longer than the rows)
constexpr int kGroup = 8;  // tiles of a group, groups of a row
constexpr int64_t kMaxSequences = int64_t{1} << 30;

struct RecurArgs {
  int64_t tokens, sequences, line, g_line, tiles;
  int units, wide, slabs;
  const void* xz;
  const void* starts;  // null: one sequence
  const int* of;       // [tokens]: the row's sequence, -1 outside of all (null: one sequence)
  const float* state;  // null: zeros
  void* h;
  float* last;
  float* kept;  // [ceil(tokens / kKeep)][units]: what comes into its rows
  // backwards
  const void* g;
  const float* g_last;  // null: zeros
  void* dxz;
  float* dstate;
  // zeros at first, in the order in which tiles are taken
  unsigned* tickets;  // one a slab, kTicket apart
  uint64_t* spans;    // [tiles][units]: the tile summed up
  uint64_t* groups;   // [groups][units]: the group
  uint64_t* carries;  // [rows of groups][units]: what comes out of the row
};

__device__ __forceinline__ int64_t start_of(const RecurArgs& a, int64_t s) {
  const int64_t t = load_id(a.starts, a.wide, s);
  return t < 0 ? 0 : t < a.tokens ? t : a.tokens;
}

// of[t]: the last sequence that starts at t or before, if t is before its end;
// and the `words` of the tiles' sums, zeros.
__global__ __launch_bounds__(256) void k_recur_setup(RecurArgs a, int* of, uint64_t* zeros, int64_t words) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, all = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t t = i; t < words; t += all) zeros[t] = 0;
  if (!of) return;
  for (int64_t t = i; t < a.tokens; t += all) {
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
}

// The sequences of N rows from first - 1 on, the same in all lanes.
template <int N>
__device__ __forceinline__ void rows_of(const RecurArgs& a, int64_t first, int (&of)[N]) {
  const int lane = threadIdx.x & 63;
  const int64_t t = first - 1 + lane;
  const bool there = t >= 0 && t < a.tokens;
  int mine = there ? 0 : -1;
  if (a.of && there && lane < N) mine = a.of[t];
#pragma unroll
  for (int i = 0; i < N; ++i) of[i] = __builtin_amdgcn_readlane(mine, i);
}

// a = sigmoid(z) and b = 1 - a: the lesser is t / (1 + t), t = exp(-|z|) with
// the rounding error of its exponent carried on, and the other one minus it, so
// that what a row passes on and takes in make one. (log2(e) is in two parts, its
// float32 value and that of what it leaves; an exponent's error e makes t 2^e,
// t + t e ln 2 to first order.)
__device__ __forceinline__ void gate(float z, float& a, float& b) {
  const float y = __builtin_elementwise_minimum(fabsf(z), 128.0f);  // (a NaN stays)
  const float hi = y * -1.44269502162933349609375f;
  float lo = __builtin_fmaf(y, -1.44269502162933349609375f, -hi);
  lo = __builtin_fmaf(y, -1.925963033500011e-8f, lo);
  float t = __builtin_amdgcn_exp2f(hi);
  t = __builtin_fmaf(t * lo, 0.693147182464599609375f, t);
  const float s = t * __builtin_amdgcn_rcpf(1.0f + t), l = 1.0f - s;
  a = z < 0.0f ? s : l;
  b = z < 0.0f ? l : s;
}

struct Pair {
  float v[2];
};
// A lane's two units of a row.
template <int FORM, typename T>
__device__ __forceinline__ typename Pack<T, 2>::type load_two(const T* row, const Lane& l) {
  if (FORM == kOne) return typename Pack<T, 2>::type{row[0], row[0]};
  typename Pack<T, 2>::type v = *reinterpret_cast<const typename Pack<T, 2>::load*>(row + l.at);
  if (FORM == kOdd) v[0] = l.n == 1 ? v[1] : v[0];
  return v;
}
template <int FORM, typename T>
__device__ __forceinline__ void store_two(T* row, const Lane& l, const float v[2]) {
  if (FORM != kOne && l.n > 1)
    *reinterpret_cast<typename Pack<T, 2>::load*>(row + l.col) = {from_f32<T>(v[0]), from_f32<T>(v[1])};
  if (FORM != kEven && l.n == 1) row[l.col] = from_f32<T>(v[0]);
}
template <int FORM>
__device__ __forceinline__ Pair load_pair(const float* row, const Lane& l) {
  const typename Pack<float, 2>::type v = load_two<FORM>(row, l);
  return {{v[0], v[1]}};
}

template <int FORM>
__device__ __forceinline__ Pair load_state(const RecurArgs& a, const float* states, int s, const Lane& l) {
  if (!states) return {{0.0f, 0.0f}};
  return load_pair<FORM>(states + static_cast<int64_t>(s) * a.units, l);
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
// Spans in LDS, and which of them are cut.
template <int N>
struct Spans {
  float4 v[N][64];
  int cut[N];
  __device__ __forceinline__ void put(int i, int lane, const Span& s) {
    v[i][lane] = make_float4(s.A[0], s.A[1], s.H[0], s.H[1]);
    if (lane == 0) cut[i] = s.cut;
  }
  // The first `count`, one after another (what lies before the last cut counts
  // for nothing).
  __device__ __forceinline__ Span fold(int count, int lane) const {
    const uint64_t cuts = __ballot(lane < count && cut[lane < N ? lane : 0] != 0);
    Span s = span_none();
    int i = 0;
    if (cuts) {
      i = 63 - __builtin_clzll(cuts);
      const float4 f = v[i++][lane];
      s = {{0.0f, 0.0f}, {f.z, f.w}, true};
    }
    for (; i < count; ++i) {
      const float4 f = v[i][lane];
      s.H[0] = __builtin_fmaf(f.x, s.H[0], f.z), s.H[1] = __builtin_fmaf(f.y, s.H[1], f.w);
      s.A[0] *= f.x, s.A[1] *= f.y;
    }
    return s;
  }
};
__device__ __forceinline__ void span_into(const Span& s, Pair& in) {
#pragma unroll
  for (int j = 0; j < 2; ++j) in.v[j] = s.cut ? s.H[j] : __builtin_fmaf(s.A[j], in.v[j], s.H[j]);
}

// A unit's span as a word that is not 0: H above, A (never below 0) with its
// sign set, or all ones for a cut. The word is its own flag: words go to memory
// and from there past the caches that the chip's parts have to themselves.
constexpr uint32_t kReady = 0x80000000u, kCut = 0xFFFFFFFFu;
__device__ __forceinline__ void put_word(uint64_t* p, float h, uint32_t low) {
  __hip_atomic_store(p, static_cast<uint64_t>(__float_as_uint(h)) << 32 | low, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint32_t span_low(float A, bool cut) {
  if (cut) return kCut;
  return A != A ? 0xFFC00000u : __float_as_uint(A) | kReady;
}
// A lane's two words, when all lanes' are there. (Some 2^20 polls of half a
// microsecond and more, and then NaN.)
__device__ __forceinline__ void wait_words(const uint64_t* row, const Lane& l, uint64_t w[2]) {
#pragma unroll 1
  for (int tries = 0; tries < 1 << 20; ++tries) {
    w[0] = __hip_atomic_load(row + l.word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    w[1] = __hip_atomic_load(row + l.next, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__all((w[0] & w[1] & kReady) != 0)) return;
    __builtin_amdgcn_s_sleep(1);
  }
  w[0] = w[1] = uint64_t{0x7FC00000u} << 32 | 0xFFC00000u;
}

__device__ __forceinline__ Span wait_span(const uint64_t* row, const Lane& l) {
  uint64_t w[2];
  wait_words(row, l, w);
  Span s;
  s.cut = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(w[0])) == kCut;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    s.A[j] = __uint_as_float(static_cast<uint32_t>(w[j]) & ~kReady);
    s.H[j] = __uint_as_float(static_cast<uint32_t>(w[j] >> 32));
  }
  return s;
}
__device__ __forceinline__ void put_span(uint64_t* row, const Lane& l, const Span& s) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (j < l.n) put_word(row + (l.col + j), s.H[j], span_low(s.A[j], s.cut));
}

// What the waves of a workgroup share.
struct Shared {
  Spans<kWaves> waves;           // of the tile's waves
  Spans<kGroup> tiles, groups;   // of the tiles before it in its group, the groups before in the row
  float2 into[64];               // what comes into the row of groups
  unsigned number;
};
// What comes into the tile that is walked as the `at`-th. Its span goes out (by
// the last wave, `own` the wave's, `s` of the waves before it), and its group's
// if it is the last of it; the other waves wait for the tiles and groups
// before it, the last one for what comes into the row.
__device__ __forceinline__ Pair into_tile(const RecurArgs& a, int64_t at, const Lane& l, int wave, const Span& s,
                                          const Span& own, Shared& sh) {
  const int lane = threadIdx.x & 63;
  const int tile = static_cast<int>(at % kGroup), group = static_cast<int>(at / kGroup % kGroup);
  const int64_t row = at / (kGroup * kGroup);
  const bool last = wave == kWaves - 1, more = at + 1 < a.tiles;
  Span whole = s;
  if (last) {
    span_then(whole, own);
    if (more && tile < kGroup - 1) put_span(a.spans + at * a.units, l, whole);
  } else if (wave < tile) {
    sh.tiles.put(wave, lane, wait_span(a.spans + (at - tile + wave) * a.units, l));
  }
  if (more && tile == kGroup - 1 && group < kGroup - 1) {  // (the group's sum waits for no other group's)
    __syncthreads();
    if (last) {
      Span all = sh.tiles.fold(tile, lane);
      span_then(all, whole);
      put_span(a.groups + at / kGroup * a.units, l, all);
    }
  }
  if (last) {
    Pair in = {{0.0f, 0.0f}};
    if (row > 0) {
      uint64_t w[2];
      wait_words(a.carries + (row - 1) * a.units, l, w);
#pragma unroll
      for (int j = 0; j < 2; ++j) in.v[j] = __uint_as_float(static_cast<uint32_t>(w[j] >> 32));
    }
    sh.into[lane] = make_float2(in.v[0], in.v[1]);
  } else if (wave < group) {
    sh.groups.put(wave, lane, wait_span(a.groups + (at / kGroup - group + wave) * a.units, l));
  }
  __syncthreads();
  Pair in = {{sh.into[lane].x, sh.into[lane].y}};
  span_into(sh.groups.fold(group, lane), in);
  span_into(sh.tiles.fold(tile, lane), in);
  if (last && more && tile == kGroup - 1 && group == kGroup - 1) {
    Pair out = in;
    span_into(whole, out);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (j < l.n) put_word(a.carries + row * a.units + (l.col + j), out.v[j], kReady);
  }
  return in;
}

// Whether no sequence begins or ends in a wave's rows, and all are of one: then
// they are walked without looking.
template <int N>
__device__ __forceinline__ bool unbroken(const int (&of)[N]) {
  bool same = of[0] >= 0;
#pragma unroll
  for (int i = 0; i < N - 1; ++i) same &= of[i] == of[i + 1];
  return same;
}

// A wave's rows forwards, from their A and H: rows at which a sequence starts
// get its state put into H.
template <int FORM, int N>
__device__ __forceinline__ Span sum_up(const RecurArgs& a, const int (&of)[N + 2], const Lane& l,
                                       const float (&A)[N][2], float (&H)[N][2]) {
  Span s = span_none();
  if (unbroken(of)) {
#pragma unroll
    for (int i = 0; i < N; ++i) span_then(s, {{A[i][0], A[i][1]}, {H[i][0], H[i][1]}, false});
    return s;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int q = of[i + 1];
    const bool cut = q < 0 || of[i] != q;
    if (q < 0) {
      H[i][0] = H[i][1] = 0.0f;
    } else if (cut) {
      const Pair in = load_state<FORM>(a, a.state, q, l);
#pragma unroll
      for (int j = 0; j < 2; ++j) H[i][j] = __builtin_fmaf(A[i][j], in.v[j], H[i][j]);
    }
    span_then(s, {{A[i][0], A[i][1]}, {H[i][0], H[i][1]}, cut});
  }
  return s;
}

// Sequences without rows: out = in (null: zeros), 64 of them at a time by the
// waves of a slab's workgroups.
template <int FORM>
__device__ __forceinline__ void pass_empty(const RecurArgs& a, int64_t tile, const float* in, float* out,
                                           const Lane& l) {
  if (!a.starts && a.tokens > 0) return;
  const int64_t all = a.tiles > 0 ? a.tiles : 1;
  for (int64_t first = (tile * kWaves + (threadIdx.x >> 6)) * 64; first < a.sequences; first += all * kWaves * 64) {
    const int64_t s = first + (threadIdx.x & 63);
    const bool empty = s < a.sequences && (!a.starts || start_of(a, s) >= start_of(a, s + 1));
    for (uint64_t mask = __ballot(empty); mask; mask &= mask - 1) {
      const int at = static_cast<int>(first + __builtin_ctzll(mask));
      store_two<FORM>(out + static_cast<int64_t>(at) * a.units, l, load_state<FORM>(a, in, at, l).v);
    }
  }
}

// The workgroup's slab of units, each as often as there are tiles: 8 workgroups
// in a row, one on each of the chip's parts, take the same one. (A slab of a
// row is 256 bytes, a channel of a part's cache; with slab after slab a part
// had the same few of them all the time, 143 us in place of 122.)
__device__ __forceinline__ unsigned slab_of(const RecurArgs& a) {
  const unsigned slabs = a.slabs, i = blockIdx.x, whole = gridDim.x / (8 * slabs) * (8 * slabs);
  return i < whole ? i / 8 % slabs : (i - whole) % slabs;
}
// The workgroup's tile in the order in which a slab's are taken.
__device__ __forceinline__ int take(const RecurArgs& a, unsigned slab, unsigned* shared) {
  if (a.tiles <= 1) return 0;
  if (threadIdx.x == 0)
    *shared = __hip_atomic_fetch_add(a.tickets + slab * kTicket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*shared);
}

template <typename T, int FORM>
__global__ __launch_bounds__(64 * kWaves, 4) void k_recur(RecurArgs a) {
  __shared__ Shared sh;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned slab = slab_of(a);
  const int64_t tile = take(a, slab, &sh.number), t = (tile * kWaves + wave) * kForth;
  const Lane l = lane_of<FORM>(slab * kSlab, lane, a.units);
  int of[kForth + 2];
  float A[kForth][2], H[kForth][2];
  if (a.tokens > 0) {
    typename Pack<T, 2>::type x[kForth], z[kForth];
    const int64_t first = t < a.tokens ? t : 0, rows = a.tokens - t;
    const T* xz = static_cast<const T*>(a.xz) + first * a.line;
#pragma unroll
    for (int i = 0; i < kForth; ++i) {
      const T* row = xz + (i < rows ? i * a.line : 0);
      x[i] = load_two<FORM>(row, l), z[i] = load_two<FORM>(row + a.units, l);
    }
#pragma unroll
    for (int i = 0; i < kForth; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float b;
        gate(to_f32(z[i][j]), A[i][j], b);
        H[i][j] = b * to_f32(x[i][j]);
      }
    }
  }
  rows_of(a, t, of);
  const Span own = sum_up<FORM, kForth>(a, of, l, A, H);
  sh.waves.put(wave, lane, own);
  __syncthreads();
  const Span s = sh.waves.fold(wave, lane);  // the waves before
  Pair h = into_tile(a, tile, l, wave, s, own, sh);
  span_into(s, h);
  if (t % kKeep == 0 && t < a.tokens) store_two<FORM>(a.kept + t / kKeep * a.units, l, h.v);
  T* out = static_cast<T*>(a.h) + t * a.units;
  if (unbroken(of)) {
#pragma unroll
    for (int i = 0; i < kForth; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) h.v[j] = __builtin_fmaf(A[i][j], h.v[j], H[i][j]);
      store_two<FORM>(out + i * a.units, l, h.v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kForth; ++i) {
      if (t + i >= a.tokens) continue;
      const int q = of[i + 1];
      const bool cut = q < 0 || of[i] != q;
#pragma unroll
      for (int j = 0; j < 2; ++j) h.v[j] = cut ? H[i][j] : __builtin_fmaf(A[i][j], h.v[j], H[i][j]);
      store_two<FORM>(out + i * a.units, l, h.v);
      if (q >= 0 && of[i + 2] != q) store_two<FORM>(a.last + static_cast<int64_t>(q) * a.units, l, h.v);
    }
  }
  pass_empty<FORM>(a, tile, a.state, a.last, l);
}

// The gradients, tiles from the last to the first. Backwards, a row passes on
// what comes in from behind as u -> a (g + u); a sequence's last row puts its
// last state's gradient in, its first row's goes to its state and no further.
// h is walked again from what came into the tile, so that it is neither kept
// nor rounded.
template <typename T, int FORM>
__global__ __launch_bounds__(64 * kWaves, 4) void k_recur_grad(RecurArgs a) {
  __shared__ Shared sh;
  __shared__ Spans<kWaves> forth;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned slab = slab_of(a);
  const int64_t at = take(a, slab, &sh.number), tile = a.tiles > 0 ? a.tiles - 1 - at : 0, t = (tile * kWaves + wave) * kBack;
  const Lane l = lane_of<FORM>(slab * kSlab, lane, a.units);
  int of[kBack + 2];
  typename Pack<T, 2>::type x[kBack], g[kBack];
  float A[kBack][2], B[kBack][2];  // the gates
  Pair h = {{0.0f, 0.0f}};
  if (a.tokens > 0) {
    typename Pack<T, 2>::type z[kBack];
    const int64_t first = t < a.tokens ? t : 0, rows = a.tokens - t;
    const T* xz = static_cast<const T*>(a.xz) + first * a.line;
    const T* gs = static_cast<const T*>(a.g) + first * a.g_line;
#pragma unroll
    for (int i = 0; i < kBack; ++i) {
      const T* row = xz + (i < rows ? i * a.line : 0);
      x[i] = load_two<FORM>(row, l), z[i] = load_two<FORM>(row + a.units, l);
      g[i] = load_two<FORM>(gs + (i < rows ? i * a.g_line : 0), l);
    }
    h = load_pair<FORM>(a.kept + tile * a.units, l);
#pragma unroll
    for (int i = 0; i < kBack; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) gate(to_f32(z[i][j]), A[i][j], B[i][j]);
    }
  }
  rows_of(a, t, of);
  const bool whole = unbroken(of);
  Span u = span_none();
  {
    float H[kBack][2];
#pragma unroll
    for (int i = 0; i < kBack; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) H[i][j] = B[i][j] * to_f32(x[i][j]);
    forth.put(wave, lane, sum_up<FORM, kBack>(a, of, l, A, H));
  }
#pragma unroll
  for (int i = kBack - 1; i >= 0; --i) {
    const int q = of[i + 1];
    const bool on = whole || (q >= 0 && of[i] == q), last = !whole && of[i + 2] != q;
    Pair more = {{0.0f, 0.0f}};
    if (on && last) more = load_state<FORM>(a, a.g_last, q, l);
    Span row;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      row.A[j] = A[i][j];
      row.H[j] = on ? A[i][j] * (to_f32(g[i][j]) + more.v[j]) : 0.0f;
    }
    row.cut = !on || last;
    span_then(u, row);
  }
  const int back = kWaves - 1 - wave;  // waves backwards
  sh.waves.put(back, lane, u);
  __syncthreads();
  const Span s = sh.waves.fold(back, lane);  // the waves behind
  Pair c = into_tile(a, at, l, back, s, u, sh);
  span_into(s, c);
  span_into(forth.fold(wave, lane), h);
  float before[kBack][2];  // h of the row before
#pragma unroll
  for (int i = 0; i < kBack; ++i) {
    const int q = of[i + 1];
    if (!whole && of[i] != q) h = q >= 0 ? load_state<FORM>(a, a.state, q, l) : Pair{{0.0f, 0.0f}};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      before[i][j] = h.v[j];
      h.v[j] = __builtin_fmaf(A[i][j], h.v[j], B[i][j] * to_f32(x[i][j]));
    }
  }
  T* out = static_cast<T*>(a.dxz) + t * 2 * a.units;
#pragma unroll
  for (int i = kBack - 1; i >= 0; --i) {
    if (t + i >= a.tokens) continue;
    const int q = of[i + 1];
    float dx[2] = {0.0f, 0.0f}, dz[2] = {0.0f, 0.0f};
    if (whole || q >= 0) {
      if (!whole && of[i + 2] != q) c = load_state<FORM>(a, a.g_last, q, l);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float v = to_f32(g[i][j]) + c.v[j];
        dx[j] = B[i][j] * v;
        c.v[j] = A[i][j] * v;
        dz[j] = B[i][j] * c.v[j] * (before[i][j] - to_f32(x[i][j]));
      }
      if (!whole && of[i] != q) store_two<FORM>(a.dstate + static_cast<int64_t>(q) * a.units, l, c.v);
    }
    T* row = out + i * 2 * a.units;
    store_two<FORM>(row, l, dx);
    store_two<FORM>(row + a.units, l, dz);
  }
  pass_empty<FORM>(a, at, a.g_last, a.dstate, l);
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

struct RecurPlan {
  int64_t tiles, slabs, spans, groups, carries, words, bytes;  // words of 8 bytes, then the rows' sequences
};
RecurPlan recur_plan(int64_t tokens, int64_t units, bool ragged, int rows) {
  RecurPlan p{};
  p.tiles = div_up(tokens, kWaves * rows), p.slabs = div_up(units, kSlab);
  if (p.tiles > 1) {  // (the tickets come first)
    p.spans = p.slabs * kTicket / 2;
    p.groups = p.spans + p.tiles * units;
    p.carries = p.groups + p.tiles / kGroup * units;
    p.words = p.carries + p.tiles / (kGroup * kGroup) * units;
  }
  p.bytes = 8 * p.words + (ragged ? 4 * tokens : 0);
  return p;
}

constexpr int64_t kMaxWork = int64_t{1} << 22;  // workgroups of a launch: at most 2^31 lanes
bool recur_fits(int64_t tokens, int64_t units, int64_t sequences, int wide) {
  return batch_fits(tokens, units) && units <= kMaxLevel / 2 && sequences >= 0 && sequences <= kMaxSequences &&
         (wide == 0 || wide == 1) && div_up(tokens, kKeep) * div_up(units, kSlab) <= kMaxWork;
}

// The plan into the arguments, the rows' sequences and the words' zeros.
void recur_setup(RecurArgs& a, const RecurPlan& p, void* workspace, hipStream_t s) {
  uint64_t* words = static_cast<uint64_t*>(workspace);
  a.tiles = p.tiles, a.slabs = static_cast<int>(p.slabs);
  a.tickets = reinterpret_cast<unsigned*>(words), a.spans = words + p.spans;
  a.groups = words + p.groups, a.carries = words + p.carries;
  int* of = a.starts && a.tokens > 0 ? reinterpret_cast<int*>(words + p.words) : nullptr;
  a.of = of;
  const int64_t rows = of ? a.tokens : 0, lanes = p.words > rows ? p.words : rows;
  if (lanes == 0) return;
  const int64_t groups = div_up(lanes, 256), most = int64_t{1} << 16;
  k_recur_setup<<<static_cast<unsigned>(groups < most ? groups : most), 256, 0, s>>>(a, of, words, p.words);
}
unsigned recur_groups(const RecurPlan& p) { return static_cast<unsigned>((p.tiles > 0 ? p.tiles : 1) * p.slabs); }

}  // namespace

extern "C" {

int64_t plx_recur_workspace(int64_t tokens, int64_t units, int64_t sequences, int32_t ragged) {
  if (!recur_fits(tokens, units, sequences, 0)) return -1;
  if (units == 0 || (tokens == 0 && sequences == 0)) return 0;
  return recur_plan(tokens, units, ragged != 0, kBack).bytes;  // (the gradients' is the larger)
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
  const RecurPlan p = recur_plan(tokens, units, starts != nullptr, kForth);
  if (p.bytes > 0 && (!workspace || !on_16(workspace) || workspace_bytes < p.bytes))
    return fail(PLX_ERR_INVALID, "plx_recur: plx_recur_workspace() bytes on 16 bytes needed");
  hipStream_t s = static_cast<hipStream_t>(stream);
  RecurArgs a{};
  a.tokens = tokens, a.sequences = sequences, a.line = line, a.units = static_cast<int>(units), a.wide = wide;
  a.xz = xz, a.starts = starts, a.state = state, a.h = h, a.last = last, a.kept = kept;
  recur_setup(a, p, workspace, s);
  with_type(dtype, [&](auto* e) {
    using T = PLX_DENSE_TYPE(e);
    if (units == 1)
      k_recur<T, kOne><<<recur_groups(p), 64 * kWaves, 0, s>>>(a);
    else if (units % 2)
      k_recur<T, kOdd><<<recur_groups(p), 64 * kWaves, 0, s>>>(a);
    else
      k_recur<T, kEven><<<recur_groups(p), 64 * kWaves, 0, s>>>(a);
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
  const RecurPlan p = recur_plan(tokens, units, starts != nullptr, kBack);
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
    if (units == 1)
      k_recur_grad<T, kOne><<<recur_groups(p), 64 * kWaves, 0, s>>>(a);
    else if (units % 2)
      k_recur_grad<T, kOdd><<<recur_groups(p), 64 * kWaves, 0, s>>>(a);
    else
      k_recur_grad<T, kEven><<<recur_groups(p), 64 * kWaves, 0, s>>>(a);
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
