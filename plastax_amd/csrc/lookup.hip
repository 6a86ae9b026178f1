// lookup.hip -- an input level of which one unit is on for each token: rows of
// its level pair looked up by id, and the pair's gradient, the sums of the
// tokens' gradients by id. No counterpart in the reference.
//
// The gradient sorts the tokens by id, stably, so that every sum has a fixed
// order (float32, no atomics on floats): three launches,
//   k_group      ids to classes (id mod classes), a workgroup each: it reads
//                all ids, counts those of lower classes, which gives its place
//                in the list, and sorts its own by counting (bound by the
//                caches that all of them read through: 65536 ids 26 us);
//   k_row_sums   every row of up to kPart tokens (zeros where it has none),
//                and the parts of longer ones: kPart places of the list each;
//   k_join_sums  the longer rows from their parts, in order.
//
// 65536 tokens, 131072 rows of 1024 units, bf16: looked up in 48 us (a row read
// again is often in a cache); the gradient in 26, 131 and 12, of which the
// second writes 537 MB and reads 134, 5.1 TB/s. With few tokens a launch's
// chain of loads is what it takes: 4 to 11 us each. The sort reads tokens *
// classes ids, whatever the units: 65536 tokens of 16 units are 28 us, nearly all
// of it the sort's. One workgroup orders all tokens of a class, and one joins the
// parts of 256 columns of a row: 65536 tokens of 131072 rows of 1024 units take
// 145 us with ids that all differ, 160 where one in ten, 254 where half and 357
// where all of them are one id (300 rows: 62, 75, 152 and 233).

#include "px_dense.h"

using plx_detail::check_launch;
using plx_detail::fail;

namespace {

using namespace px;

constexpr int kPart = 16;      // places of the list that one part sums
constexpr int kLocal = 4096;   // rows of a class at most (their counters are in LDS)
constexpr int kGroupWaves = 16;
constexpr int kFound = 512;    // tokens that a wave keeps in LDS, of a range of at most 2^kRange
constexpr int kRange = 20;

struct LookArgs {
  int64_t tokens, line;
  int rows, units, wide, classes, shift;
  float scale;
  const void* ids;
  const void* x;  // the table, or the tokens' gradients
  void* out;      // the rows looked up, or the table's gradient
  int2* info;     // [rows]: the row's first place in the list, its tokens
  int* list;      // [tokens] tokens by id
  int2* stage;    // [tokens] a class's tokens in order, with their rows' numbers in it
  int* total;     // the list's length
  float* part;    // [parts][2][units]
};

// y[t] = scale table[id]. A lane takes 16 bytes; lx lanes a token. Bound by
// memory (the rows come from all over the table).
template <typename T>
__global__ __launch_bounds__(256) void k_look_up(LookArgs a, int lx) {
  constexpr int W = kChunk<T>;
  const int tx = threadIdx.x & (lx - 1);
  const int per = 256 / lx;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / lx; t < a.tokens;
       t += static_cast<int64_t>(gridDim.x) * per) {
    const int64_t id = load_id(a.ids, a.wide, t);
    const bool there = id >= 0 && id < a.rows;
    const T* row = static_cast<const T*>(a.x) + (there ? id : 0) * a.line;
    T* out = static_cast<T*>(a.out) + t * a.units;
    for (int64_t at = static_cast<int64_t>(tx) * W; at < a.units; at += lx * W) {
      const typename Pack<T, W>::type v = load_pack<W>(row + at, there ? a.units - at : 0);
      float y[W];
#pragma unroll
      for (int i = 0; i < W; ++i) y[i] = there ? to_f32(v[i]) * a.scale : 0.0f;
      store_pack<W, true>(out + at, a.units - at, y);
    }
  }
}

__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, 64);
  return v;
}
__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// Ids 64 apart as 32 bits, enough of them on their way at once; from `end` on
// and out of 32 bits they are all ones, which is no row.
constexpr int kAhead = 16;
template <typename I>
__device__ __forceinline__ void load_ids(const LookArgs& a, int64_t t, int64_t end, uint32_t id[kAhead]) {
  I v[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int64_t at = t + 64 * i;
    v[i] = static_cast<const I*>(a.ids)[at < end ? at : end - 1];
  }
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const bool there = t + 64 * i < end && (sizeof(I) == 4 || static_cast<uint64_t>(v[i]) >> 32 == 0);
    id[i] = there ? static_cast<uint32_t>(v[i]) : ~0u;
  }
}

template <typename I>  // the ids' type
__global__ __launch_bounds__(64 * kGroupWaves) void k_group(LookArgs a) {
  constexpr int NT = 64 * kGroupWaves;
  __shared__ int cursor[kLocal];
  __shared__ uint32_t found[kGroupWaves][kFound];  // a wave's tokens of the class, in order: row, place in its range
  __shared__ int less[kGroupWaves], own[kGroupWaves], sums[kGroupWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mine = blockIdx.x;
  const int local = (a.rows + a.classes - 1) / a.classes;
  for (int i = threadIdx.x; i < local; i += NT) cursor[i] = 0;
  // A wave's tokens lie behind each other.
  const int64_t per = div_up(a.tokens, NT) * 64, begin = wave * per;
  const int64_t end = begin + per < a.tokens ? begin + per : a.tokens;
  __syncthreads();
  int below = 0, hits = 0;
  // The wave's tokens of the class, in order: where(place, row, token).
  auto search = [&](auto where) {
    int at = 0;
    for (int64_t first = begin; first < end; first += 64 * kAhead) {
      uint32_t id[kAhead];
      load_ids<I>(a, first + lane, end, id);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const uint32_t c = id[i] < static_cast<uint32_t>(a.rows) ? id[i] & (a.classes - 1) : ~0u;
        below += c < static_cast<uint32_t>(mine);
        const uint64_t mask = __ballot(c == static_cast<uint32_t>(mine));
        if (mask) {
          if (c == static_cast<uint32_t>(mine))
            where(at + lanes_below(mask), static_cast<int>(id[i] >> a.shift), static_cast<int>(first - begin) + 64 * i + lane);
          at += __popcll(mask);
        }
      }
    }
    return at;
  };
  hits = search([&](int place, int row, int token) {
    if (place < kFound) found[wave][place] = static_cast<uint32_t>(row) << kRange | token;
    atomicAdd(&cursor[row], 1);
  });
  below = wave_sum_int(below);
  if (lane == 0) less[wave] = below, own[wave] = hits;
  __syncthreads();
  int base = 0, n = 0, at = 0;
#pragma unroll
  for (int w = 0; w < kGroupWaves; ++w) {
    base += less[w];
    at += w < wave ? own[w] : 0;
    n += own[w];
  }
  if (mine == a.classes - 1 && threadIdx.x == 0) *a.total = base + n;
  int2* stage = a.stage + base;
  const int token0 = static_cast<int>(begin);
  if (hits <= kFound && per <= 1 << kRange) {
    for (int i = lane; i < hits; i += 64) {
      const uint32_t v = found[wave][i];
      stage[at + i] = make_int2(token0 + static_cast<int>(v & ((1u << kRange) - 1)), static_cast<int>(v >> kRange));
    }
  } else {  // (once more: they did not fit)
    search([&](int place, int row, int token) { stage[at + place] = make_int2(token0 + token, row); });
  }
  __syncthreads();
  // The rows' places: an exclusive scan of the counts, kLocal / NT a lane.
  constexpr int EACH = kLocal / NT;
  int count[EACH], sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int r = threadIdx.x * EACH + i;
    count[i] = r < local ? cursor[r] : 0;
    sum += count[i];
  }
  int scan = sum;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int v = __shfl_up(scan, d, 64);
    scan += lane >= d ? v : 0;
  }
  if (lane == 63) sums[wave] = scan;
  __syncthreads();
  int place = scan - sum;
#pragma unroll
  for (int w = 0; w < kGroupWaves; ++w) place += w < wave ? sums[w] : 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int r = threadIdx.x * EACH + i;
    const int64_t row = static_cast<int64_t>(r) * a.classes + mine;
    if (r < local) {
      cursor[r] = place;
      if (row < a.rows) a.info[row] = make_int2(base + place, count[i]);
    }
    place += count[i];
  }
  __syncthreads();
  // The tokens to their places, in order: 64 at a time, 4 such blocks a wave.
  // Equal rows of a block are found bit by bit by all waves at once; then the
  // waves take their rows' places one after another.
  constexpr int GO = 4, ROUND = NT * GO;
  int* list = a.list + base;
  for (int first = 0; first < n; first += ROUND) {
    int2 v[GO];
    uint64_t same[GO];
    int from[GO];
#pragma unroll
    for (int k = 0; k < GO; ++k) {
      const int i = first + (wave * GO + k) * 64 + lane;
      v[k] = i < n ? stage[i] : make_int2(-1, 0);
    }
#pragma unroll
    for (int k = 0; k < GO; ++k) {
      same[k] = __ballot(v[k].x >= 0);
      for (int b = 1; b < local; b *= 2) {
        const uint64_t ones = __ballot(v[k].y & b);
        same[k] &= (v[k].y & b) ? ones : ~ones;
      }
    }
    const int left = n - first, turns = left < ROUND ? (left + 64 * GO - 1) / (64 * GO) : kGroupWaves;
    for (int turn = 0; turn < turns; ++turn) {
      if (turn == wave) {
#pragma unroll
        for (int k = 0; k < GO; ++k) {
          from[k] = 0;
          if (v[k].x >= 0 && lanes_below(same[k]) == 0) from[k] = atomicAdd(&cursor[v[k].y], __popcll(same[k]));
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < GO; ++k) {
      const int start = __shfl(from[k], v[k].x >= 0 ? __builtin_ctzll(same[k]) : 0, 64);
      if (v[k].x >= 0) list[start + lanes_below(same[k])] = v[k].x;
    }
  }
}

// What LX lanes of a row do, NC chunks of 4 columns each, from column `at` on
// (slab: the columns of all lanes).
template <int LX, int NC>
struct Columns {
  static constexpr int kSlab = LX * NC * 4;
  float v[NC][4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[k][i] = 0.0f;
  }
  template <typename T>
  struct Raw {
    typename Pack<T, 4>::type x[NC];
  };
  template <typename T>
  __device__ __forceinline__ Raw<T> load(const T* row, int units, int at) const {
    Raw<T> r;
#pragma unroll
    for (int k = 0; k < NC; ++k) r.x[k] = load_pack<4>(row + at + k * LX * 4, units - at - k * LX * 4);
    return r;
  }
  template <typename T>
  __device__ __forceinline__ void add(const Raw<T>& r) {
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[k][i] += to_f32(r.x[k][i]);
  }
  template <bool PASS>
  __device__ __forceinline__ void store(float* row, int units, int at, float scale) {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      float s[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = v[k][i] * scale;
      store_pack<4, PASS>(row + at + k * LX * 4, units - at - k * LX * 4, s);
    }
  }
};

// Workgroups of the first `part_groups` sum parts, the others rows; blockIdx.y
// is the slab of columns. A row's lanes read its place and count, then its
// tokens, then their gradients: for kEach rows at once.
constexpr int kEach = 2;
template <typename T, int LX, int NC, bool PASS>
__global__ __launch_bounds__(256) void k_row_sums(LookArgs a, int part_groups) {
  using Sum = Columns<LX, NC>;
  constexpr int PER = 256 / LX;
  const int at = static_cast<int>(blockIdx.y) * Sum::kSlab + (threadIdx.x & (LX - 1)) * 4;
  const T* g = static_cast<const T*>(a.x);
  Sum sum;
  if (static_cast<int>(blockIdx.x) < part_groups) {
    const int total = *a.total;
    const int64_t p = static_cast<int64_t>(blockIdx.x) * PER + threadIdx.x / LX, begin = p * kPart;
    if (begin >= total) return;
    const int end = static_cast<int>(begin + kPart < total ? begin + kPart : total);
    const int64_t first = load_id(a.ids, a.wide, a.list[begin]), last = load_id(a.ids, a.wide, a.list[end - 1]);
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      if (h && first == last) return;
      const int2 row = a.info[h ? last : first];
      if (row.y <= kPart) continue;
      const int from = h ? row.x : static_cast<int>(begin), to = h || row.x + row.y > end ? end : row.x + row.y;
      sum.clear();
#pragma unroll 4
      for (int j = from; j < to; ++j) sum.add(sum.load(g + a.list[j] * a.line, a.units, at));
      sum.template store<false>(a.part + (2 * p + h) * a.units, a.units, at, 1.0f);
    }
    return;
  }
  const int64_t first = (static_cast<int64_t>(blockIdx.x - part_groups) * PER + threadIdx.x / LX) * kEach;
  int2 row[kEach];
  typename Sum::template Raw<T> x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) row[i] = first + i < a.rows ? a.info[first + i] : make_int2(0, -1);
  int token[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) token[i] = row[i].y > 0 ? a.list[row[i].x] : -1;
#pragma unroll
  for (int i = 0; i < kEach; ++i) x[i] = sum.load(g + (token[i] >= 0 ? token[i] : 0) * a.line, token[i] >= 0 ? a.units : 0, at);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (row[i].y < 0 || row[i].y > kPart) continue;
    sum.clear();
    sum.add(x[i]);
#pragma unroll 4
    for (int j = row[i].x + 1; j < row[i].x + row[i].y; ++j) sum.add(sum.load(g + a.list[j] * a.line, a.units, at));
    sum.template store<PASS>(static_cast<float*>(a.out) + (first + i) * a.units, a.units, at, row[i].y > 0 ? a.scale : 0.0f);
  }
}

// The longer rows. A workgroup looks at kJoin parts: a longer row that begins in a
// part is the row of the part's last place. Its parts go over the workgroup's
// groups of LX lanes, then over LDS (those that had any), both in order.
constexpr int kJoin = 8;
template <int LX>
__global__ __launch_bounds__(1024) void k_join_sums(LookArgs a) {
  using Sum = Columns<LX, 1>;
  constexpr int PER = 1024 / LX;
  __shared__ float joined[PER][Sum::kSlab];
  const int total = *a.total, lane = threadIdx.x & 63;
  const int tx = threadIdx.x & (LX - 1), group = threadIdx.x / LX;
  const int at = static_cast<int>(blockIdx.y) * Sum::kSlab + tx * 4;
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * kJoin + lane, begin = mine * kPart;
  int row = -1, place = 0, count = 0;
  if (lane < kJoin && begin < total) {
    row = static_cast<int>(load_id(a.ids, a.wide, a.list[begin + kPart < total ? begin + kPart - 1 : total - 1]));
    const int2 info = a.info[row];
    place = info.x, count = info.y;
    if (count <= kPart || place < begin) row = -1;
  }
  for (uint64_t found = __ballot(row >= 0); found; found &= found - 1) {  // (the same in all waves)
    const int from = __builtin_ctzll(found);
    const int64_t p = static_cast<int64_t>(blockIdx.x) * kJoin + from;
    const int r = __builtin_amdgcn_readlane(row, from), first = __builtin_amdgcn_readlane(place, from);
    const int64_t last = (first + __builtin_amdgcn_readlane(count, from) - 1) / kPart;
    Sum sum;
    sum.clear();
#pragma unroll 4
    for (int64_t q = p + group; q <= last; q += PER)
      sum.add(sum.load(a.part + (2 * q + (q == p && first > p * kPart)) * a.units, a.units, at));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) joined[group][i * LX + tx] = sum.v[0][i];
    __syncthreads();
    if (group) continue;
    const int some = static_cast<int>(last - p + 1 < PER ? last - p + 1 : PER);  // groups that had parts
#pragma unroll 4
    for (int o = 1; o < some; ++o)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum.v[0][i] += joined[o][i * LX + tx];
    sum.template store<true>(static_cast<float*>(a.out) + static_cast<int64_t>(r) * a.units, a.units, at, a.scale);
  }
}

struct LookPlan {
  int classes, shift;
  int64_t parts, info, list, stage, part, bytes;
};
LookPlan look_plan(int64_t tokens, int64_t rows, int64_t units) {
  LookPlan p{};
  p.shift = 8;
  while (div_up(rows, int64_t{1} << p.shift) > kLocal) ++p.shift;
  p.classes = 1 << p.shift;
  p.parts = tokens > kPart ? div_up(tokens, kPart) : 0;  // (no row has more than kPart tokens)
  p.info = 16;
  p.list = p.info + div_up(8 * rows, 16) * 16;
  p.stage = p.list + div_up(4 * tokens, 16) * 16;
  p.part = p.stage + div_up(8 * tokens, 16) * 16;
  p.bytes = p.part + 8 * p.parts * units;
  return p;
}

template <typename T, int LX, int NC>
void launch_sums(const LookArgs& a, const LookPlan& p, hipStream_t s) {
  constexpr int PER = 256 / LX;
  const unsigned slabs = static_cast<unsigned>(div_up(a.units, Columns<LX, NC>::kSlab));
  const int part_groups = static_cast<int>(div_up(p.parts, PER));
  const dim3 grid(static_cast<unsigned>(part_groups + div_up(a.rows, PER * kEach)), slabs);
  // (Past the caches where rows begin on 64 bytes; others would leave parts of lines: 71905 rows of 415 units 33 us,
  // through them 28.)
  if (((reinterpret_cast<uintptr_t>(a.out) | (a.units * sizeof(float))) & 63) == 0)
    k_row_sums<T, LX, NC, true><<<grid, 256, 0, s>>>(a, part_groups);
  else
    k_row_sums<T, LX, NC, false><<<grid, 256, 0, s>>>(a, part_groups);
  if (p.parts) {
    const dim3 join(static_cast<unsigned>(div_up(p.parts, kJoin)), static_cast<unsigned>(div_up(a.units, Columns<LX, 1>::kSlab)));
    k_join_sums<LX><<<join, 1024, 0, s>>>(a);
  }
}

constexpr int64_t kMaxSorted = int64_t{1} << 25;  // tokens of a gradient: a launch's parts stay below 2^31 lanes
inline bool look_fits(int64_t tokens, int64_t rows, int64_t units, int wide) {
  return batch_fits(tokens, units) && rows >= 0 && rows <= kMaxLevel && (wide == 0 || wide == 1);
}

}  // namespace

extern "C" {

int plx_look_up(int64_t tokens, int64_t rows, int64_t units, const void* ids, int32_t wide, int32_t dtype,
                const void* table, int64_t line, float scale, void* out, void* stream) {
  if (!look_fits(tokens, rows, units, wide)) return fail(PLX_ERR_INVALID, "plx_look_up: bad size");
  if (!known_type(dtype)) return fail(PLX_ERR_UNSUPPORTED, "plx_look_up: unknown element type");
  if (tokens == 0 || units == 0) return PLX_OK;
  if (!ids || (rows > 0 && !table) || !out) return fail(PLX_ERR_INVALID, "plx_look_up: null pointer");
  LookArgs a{};
  a.tokens = tokens, a.line = line, a.rows = static_cast<int>(rows), a.units = static_cast<int>(units);
  a.wide = wide, a.scale = scale, a.ids = ids, a.x = table, a.out = out;
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(dtype, [&](auto* e) {
    using T = PLX_DENSE_TYPE(e);
    int lx = 1;
    while (lx < 256 && lx < div_up(units, kChunk<T>)) lx *= 2;
    const int64_t groups = div_up(tokens, 256 / lx), most = int64_t{1} << 22;
    k_look_up<T><<<static_cast<unsigned>(groups < most ? groups : most), 256, 0, s>>>(a, lx);
  });
  return check_launch("plx_look_up");
}

int64_t plx_look_up_workspace(int64_t tokens, int64_t rows, int64_t units) {
  if (!look_fits(tokens, rows, units, 0) || tokens > kMaxSorted) return -1;
  return rows == 0 || units == 0 ? 0 : look_plan(tokens, rows, units).bytes;
}

int plx_look_up_grad(int64_t tokens, int64_t rows, int64_t units, const void* ids, int32_t wide, int32_t dtype,
                     const void* g, int64_t line, float scale, float* out, void* workspace, int64_t workspace_bytes,
                     void* stream) {
  if (!look_fits(tokens, rows, units, wide) || tokens > kMaxSorted)
    return fail(PLX_ERR_INVALID, "plx_look_up_grad: bad size");
  if (!known_type(dtype)) return fail(PLX_ERR_UNSUPPORTED, "plx_look_up_grad: unknown element type");
  if (rows == 0 || units == 0) return PLX_OK;
  if ((tokens > 0 && (!ids || !g)) || !out) return fail(PLX_ERR_INVALID, "plx_look_up_grad: null pointer");
  const LookPlan p = look_plan(tokens, rows, units);
  if (!workspace || !on_16(workspace) || workspace_bytes < p.bytes)
    return fail(PLX_ERR_INVALID, "plx_look_up_grad: plx_look_up_workspace() bytes on 16 bytes needed");
  char* work = static_cast<char*>(workspace);
  LookArgs a{};
  a.tokens = tokens, a.line = line, a.rows = static_cast<int>(rows), a.units = static_cast<int>(units);
  a.wide = wide, a.classes = p.classes, a.shift = p.shift, a.scale = scale, a.ids = ids, a.x = g, a.out = out;
  a.total = reinterpret_cast<int*>(work);
  a.info = reinterpret_cast<int2*>(work + p.info);
  a.list = reinterpret_cast<int*>(work + p.list);
  a.stage = reinterpret_cast<int2*>(work + p.stage);
  a.part = reinterpret_cast<float*>(work + p.part);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (wide)
    k_group<int64_t><<<static_cast<unsigned>(p.classes), 64 * kGroupWaves, 0, s>>>(a);
  else
    k_group<int32_t><<<static_cast<unsigned>(p.classes), 64 * kGroupWaves, 0, s>>>(a);
  with_type(dtype, [&](auto* e) {
    using T = PLX_DENSE_TYPE(e);
    if (units <= 32)
      launch_sums<T, 8, 1>(a, p, s);
    else if (units <= 128)
      launch_sums<T, 32, 1>(a, p, s);
    else if (units <= 256)
      launch_sums<T, 64, 1>(a, p, s);
    else if (units <= 512)
      launch_sums<T, 64, 2>(a, p, s);
    else
      launch_sums<T, 64, 4>(a, p, s);
  });
  return check_launch("plx_look_up_grad");
}

}  // extern "C"
