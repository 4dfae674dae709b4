// gp_route.hip — expert row routing (include/gp_reduce.h): the (token, choice)
// pairs of a router grouped by expert, rows moved to their places there, the
// places' rows brought back to the tokens with weights, and the gradient of
// that.  The row gather / scatter-add of gp_kernels.hpp move rows through an
// index that the host compiled; here the index is made on the device, in the
// same step that uses it.
//
// The moves are bound by HBM: no row takes part in a product with another.

#include <type_traits>

#include "gp_device.hpp"

namespace {

constexpr int kSortBlock = 1024;
constexpr int kSortWaves = kSortBlock / kWave;
constexpr int kMaxExperts = 1024;  // one thread of a sort block each
constexpr int kMaxChoices = kWave; // a token's choices lie in one wave's lanes

// ---------------------------------------------------------------------------
// Places: a stable counting sort of n = tokens * k choices by expert.
//   counts[e]   = #{a : id[a] = e}
//   offsets[e]  = sum over e' < e of counts[e'] rounded up to whole groups of `align`
//   position[a] = offsets[id[a]] + #{b < a : id[b] = id[a]}
// A block takes `per_block` choices in a row, a wave per_block / 16 of them, 64
// at a step.  Within a step, lanes with the same id find each other by one
// ballot per bit of the id; a lane's rank is the number of such lanes below
// it, and the first of them moves the wave's own counter in LDS.  What lies
// before the block comes from the block's own count of all choices, or, where
// these are many, from the counts that route_count_kernel has left of every
// block.  Integer sums only: the places do not depend on any order of arrival.
// Bound by latency, of the counts' sums and of one step after another: 131072
// choices of 128 experts, counts 4.7 us, places 8.8.
// ---------------------------------------------------------------------------
template <typename I>
__device__ __forceinline__ int key_of(I id, int experts) {
  return id >= 0 && id < (I)experts ? (int)id : experts;  // anything else: no expert here
}

template <typename I>
__global__ __launch_bounds__(kSortBlock) void route_count_kernel(const I *__restrict__ ids, unsigned n,
                                                                 unsigned per_block, int experts,
                                                                 int *__restrict__ hist) {
  __shared__ int count[kMaxExperts];
  if ((int)threadIdx.x < experts) count[threadIdx.x] = 0;
  __syncthreads();
  const unsigned lo = blockIdx.x * per_block, hi = min(n, lo + per_block);
  for (unsigned i = lo + threadIdx.x; i < hi; i += kSortBlock) {
    const int key = key_of(ids[i], experts);
    if (key < experts) atomicAdd(&count[key], 1);
  }
  __syncthreads();
  if ((int)threadIdx.x < experts) hist[(size_t)blockIdx.x * experts + threadIdx.x] = count[threadIdx.x];
}

// A block of W waves.
template <int W>
struct SortShared {
  int run[W][kMaxExperts];  // a wave's next place in every expert's group
  int total[kMaxExperts];
  int before[kMaxExperts];  // choices of earlier blocks
  int offset[kMaxExperts + 1];
  int wave[W];
};

// After it, s.run holds every wave's first places and s.total / s.offset the
// groups.  lo: the block's first choice, from..to: the wave's, all: they are all
// there are.  hist: the counts of `parts` runs of `per` choices, or NULL to
// count all n.  `key` is the lane's own first choice, so that a wave with one
// step reads its ids once.
template <int W, typename I>
__device__ __forceinline__ void route_prepare(SortShared<W> &s, int key, const I *__restrict__ ids, unsigned n,
                                              unsigned lo, unsigned from, unsigned to, bool all, int experts,
                                              int align, const int *__restrict__ hist, unsigned per, unsigned parts) {
  constexpr int kThreads = W * kWave;
  constexpr int kPer = kMaxExperts / kThreads;  // experts to a thread, next to each other
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  for (int e = tid; e < experts; e += kThreads) {
#pragma unroll
    for (int w = 0; w < W; ++w) s.run[w][e] = 0;
    s.total[e] = 0;
    s.before[e] = 0;
  }
  __syncthreads();
  if (key < experts) atomicAdd(&s.run[wave][key], 1);
  for (unsigned i = from + kWave + lane; i < to; i += kWave) {
    const int k = key_of(ids[i], experts);
    if (k < experts) atomicAdd(&s.run[wave][k], 1);
  }
  if (!all && !hist) {
    for (unsigned i = tid; i < n; i += kThreads) {
      const int k = key_of(ids[i], experts);
      if (k >= experts) continue;
      atomicAdd(i < lo ? &s.before[k] : &s.total[k], 1);
    }
  } else if (!all) {
    const unsigned mine = lo / per;            // the run that holds lo: its choices before lo one by one
    const unsigned rows = kThreads / experts;  // thread (row, expert) sums every rows-th run's count
    const unsigned e = tid % experts, row = tid / experts;
    if (row < rows) {
      int rest = 0, before = 0;
#pragma unroll 8
      for (unsigned g = row; g < parts; g += rows) {
        const int c = hist[(size_t)g * experts + e];
        rest += g < mine ? 0 : c;
        before += g < mine ? c : 0;
      }
      atomicAdd(&s.total[e], rest);
      atomicAdd(&s.before[e], before);
    }
    for (unsigned i = mine * per + tid; i < lo; i += kThreads) {
      const int k = key_of(ids[i], experts);
      if (k >= experts) continue;
      atomicAdd(&s.before[k], 1);
      atomicSub(&s.total[k], 1);
    }
  }
  __syncthreads();
  int padded[kPer], sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = tid * kPer + j;
    int mine = 0;
    if (e < experts) {
      if (all) {
#pragma unroll
        for (int w = 0; w < W; ++w) mine += s.run[w][e];
      } else {
        mine = s.total[e] + s.before[e];
      }
      s.total[e] = mine;
    }
    padded[j] = align == 1 ? mine : (mine + align - 1) / align * align;
    sum += padded[j];
  }
  int scan = sum;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int up = __shfl_up(scan, d, kWave);
    if (lane >= d) scan += up;
  }
  if (lane == kWave - 1) s.wave[wave] = scan;
  __syncthreads();
  int base = scan - sum;
  for (int w = 0; w < wave; ++w) base += s.wave[w];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = tid * kPer + j;
    if (e >= experts) break;
    s.offset[e] = base;
    int at = base + s.before[e];
    base += padded[j];
    if (e == experts - 1) s.offset[experts] = base;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int c = s.run[w][e];
      s.run[w][e] = at;
      at += c;
    }
  }
  __syncthreads();
}

// The wave's 64 choices of one step: each lane's place, or -1.
template <int W>
__device__ __forceinline__ int route_step(SortShared<W> &s, int key, int experts, int bits) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  uint64_t same = ~0ull;
  for (int b = 0; b < bits; ++b) {
    const uint64_t on = __ballot((key >> b) & 1);
    same &= (key >> b) & 1 ? on : ~on;
  }
  const int rank = __popcll(same & ((1ull << lane) - 1));
  const int first = __ffsll((long long)same) - 1;
  int at = 0;
  if (lane == first && key < experts) at = atomicAdd(&s.run[wave][key], __popcll(same));
  at = __shfl(at, first, kWave) + rank;
  return key < experts ? at : -1;
}

template <typename I>
__global__ __launch_bounds__(kSortBlock) void route_place_kernel(
    const I *__restrict__ ids, unsigned n, unsigned per_block, int experts, int bits, int align, unsigned rows,
    const int *__restrict__ hist, int *__restrict__ position, int *__restrict__ order, int *__restrict__ counts,
    int *__restrict__ offsets) {
  __shared__ SortShared<kSortWaves> s;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const unsigned lo = blockIdx.x * per_block, hi = min(n, lo + per_block);
  const unsigned per_wave = per_block / kSortWaves;
  const unsigned from = min(hi, lo + wave * per_wave), to = min(hi, from + per_wave);
  int key = from + lane < to ? key_of(ids[from + lane], experts) : experts;
  route_prepare(s, key, ids, n, lo, from, to, gridDim.x == 1, experts, align, hist, per_block, gridDim.x);
  if (blockIdx.x == 0) {
    if (tid < experts) {
      counts[tid] = s.total[tid];
      offsets[tid] = s.offset[tid];
    }
    if (tid == 0) offsets[experts] = s.offset[experts];
  }
  for (unsigned i0 = from; i0 < to; i0 += kWave) {
    const unsigned i = i0 + lane;
    if (i0 != from) key = i < to ? key_of(ids[i], experts) : experts;
    const int at = route_step(s, key, experts, bits);
    if (i < to) position[i] = at;
    if (at >= 0) order[at] = (int)i;
  }
  // places that hold no choice: the groups' padding, then all behind the last group
  const unsigned waves = gridDim.x * kSortWaves, me = blockIdx.x * kSortWaves + wave;
  // (unsigned: a lane's place and the step after it may pass 2^31 near the most rows)
  if (align > 1)
    for (unsigned e = me; e < (unsigned)experts; e += waves)
      for (unsigned p = (unsigned)(s.offset[e] + s.total[e]) + lane; p < (unsigned)s.offset[e + 1]; p += kWave)
        order[p] = -1;
  for (unsigned p = s.offset[experts] + me * kWave + lane; p < rows; p += waves * kWave) order[p] = -1;
}

// ---------------------------------------------------------------------------
// The moves.  A wave takes a token and a share of its columns, 64 lanes times
// 16 bytes at a step, so x is read once however many choices a token has, and
// every row of the grouped layout is touched once.  Bound by HBM (a copy reaches
// 4.9 TB/s): 16384 tokens of 4096 bf16, 8 choices, 1.23 GB in 215 us, 5.7 TB/s.
// ---------------------------------------------------------------------------
constexpr int kMoveBlock = 256;
constexpr int kMoveWaves = kMoveBlock / kWave;
// Places that one wave looks through for rows to clear: a dispatch of 8192 tokens
// of 4096 bf16 with 20000 rows of padding 172 us, 180 with sixteen, 173 with one;
// the gradient of 8192 of 2048, 64 experts in groups of 16, 104, 105 and 109.
constexpr unsigned kZeroRows = 4;

// Rows are read and written once, so they go past the caches (non-temporal):
// 8192 tokens of 2048 bf16, 8 choices: combine 52 us, 56 with its loads through
// them; its gradient 103, 114 with its stores through them; dispatch of 4096, 6
// choices: 91, 105.  But two waves' accesses share a line where rows do not start
// at one: dispatch's stores then go through the caches (32768 tokens of 1001 fp16,
// 10 choices: 210 us, 235 past them; 16384 of 600 bf16, 8 choices: 55, 57), and so
// do loads from 2, 4, ... bytes off a 16-byte boundary (the gradient of 4099
// tokens of 1001 floats: 22 us, 27 past them).
struct Shape {
  unsigned tokens, k, rows, width;
  unsigned splits;       // waves that share a token's columns
  unsigned token_waves;  // tokens * splits
  unsigned first_block;  // of this launch
};

// Clears row first + lane for every lane that finds it `empty`.
template <typename E, bool NT>
__device__ __forceinline__ void clear_rows(E *__restrict__ out, size_t stride, unsigned first, bool empty,
                                           unsigned width) {
  using V = Vec<E>;
  const int lane = threadIdx.x % kWave;
  for (uint64_t left = __ballot(empty); left; left &= left - 1) {
    E *row = out + (size_t)(first + (__ffsll((long long)left) - 1)) * stride;
    for (unsigned c = lane * V::N; c < width; c += kWave * V::N) {
      const typename V::Raw zero = (E)0.0f;
      if (c + V::N <= width)
        store_raw<E, NT>(row + c, zero);
      else
        store_part(row + c, zero, width - c);
    }
  }
}

// A row's 16 bytes from column c on.
template <typename E, bool NT = false>
__device__ __forceinline__ typename Vec<E>::Raw load_at(const E *__restrict__ row, unsigned c, unsigned width) {
  return c + Vec<E>::N <= width ? load_raw<E, NT>(row + c) : load_part(row + c, (int)(width - c));
}

// A token's columns of one wave, to the row of every choice; p: lane c's row, v:
// the lane's first values (any, where its column is behind the row).
template <typename E, bool NT>
__device__ __forceinline__ void dispatch_token(E *__restrict__ out, size_t out_stride, const E *__restrict__ from,
                                               int p, unsigned split, const Shape &d, typename Vec<E>::Raw v) {
  using V = Vec<E>;
  const int lane = threadIdx.x % kWave;
  const uint64_t held = __ballot((unsigned)p < d.rows);
  const unsigned first = (split * kWave + lane) * V::N, step = d.splits * kWave * V::N;
  for (unsigned c = first; c < d.width; c += step) {
    if (c != first) v = load_at(from, c, d.width);
    for (uint64_t left = held; left; left &= left - 1) {
      const int to = __builtin_amdgcn_readlane(p, __ffsll((long long)left) - 1);
      E *row = out + (size_t)to * out_stride + c;
      if (c + V::N <= d.width)
        store_raw<E, NT>(row, v);
      else
        store_part(row, v, d.width - c);
    }
  }
}

template <typename E>
__device__ __forceinline__ typename Vec<E>::Raw first_values(const E *__restrict__ from, unsigned split,
                                                             const Shape &d) {
  const unsigned c = (split * kWave + threadIdx.x % kWave) * Vec<E>::N;
  return c < d.width ? load_at(from, c, d.width) : (typename Vec<E>::Raw)((E)0.0f);
}

template <typename E, bool NT>
__global__ __launch_bounds__(kMoveBlock) void route_dispatch_kernel(E *__restrict__ out, size_t out_stride,
                                                                    const E *__restrict__ x, size_t x_stride,
                                                                    const int *__restrict__ position,
                                                                    const int *__restrict__ order, Shape d) {
  const unsigned wave = (d.first_block + blockIdx.x) * kMoveWaves + threadIdx.x / kWave;
  const int lane = threadIdx.x % kWave;
  if (wave >= d.token_waves) {
    const unsigned first = (wave - d.token_waves) * kZeroRows, at = first + lane;
    const bool mine = lane < (int)kZeroRows && at < d.rows;
    const int o = mine ? order[at] : 0;
    clear_rows<E, NT>(out, out_stride, first, mine && (o < 0 || (unsigned)o >= d.tokens * d.k), d.width);
    return;
  }
  const unsigned t = wave / d.splits;
  const int p = lane < (int)d.k ? position[(size_t)t * d.k + lane] : -1;
  const unsigned split = wave % d.splits;
  const E *from = x + (size_t)t * x_stride;
  dispatch_token<E, NT>(out, out_stride, from, p, split, d, first_values(from, split, d));
}

// A row's group is the last that starts at or before it; behind the group's
// choices the row is empty.
template <int W>
__device__ __forceinline__ bool row_empty(const SortShared<W> &s, int r, int experts) {
  int lo = 0, hi = experts;  // offset[lo] <= r < offset[hi], or r is behind the last group
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (s.offset[mid] <= r)
      lo = mid;
    else
      hi = mid;
  }
  return r - s.offset[lo] >= s.total[lo];
}

// Few choices: every block makes the places for itself, in LDS, and moves its
// own tokens, in one launch.  The first block leaves the places for later
// calls.  Bound by the launch: 16 tokens of 4096 bf16, 4 choices, 4.5 us on the
// device in a pass of 12.7; 21.9 a pass with the places in a launch of their own.
constexpr unsigned kSmallRoute = 1024;

template <typename E, typename I>
__global__ __launch_bounds__(kMoveBlock) void route_sort_dispatch_kernel(
    E *__restrict__ out, size_t out_stride, const E *__restrict__ x, size_t x_stride, const I *__restrict__ ids,
    int experts, int bits, int align, int *__restrict__ position, int *__restrict__ order, int *__restrict__ counts,
    int *__restrict__ offsets, Shape d) {
  __shared__ SortShared<kMoveWaves> s;
  __shared__ int place[kSmallRoute];
  const unsigned n = d.tokens * d.k;
  const bool leaves = d.first_block + blockIdx.x == 0;
  const int tid = threadIdx.x, in_block = tid / kWave, lane = tid % kWave;
  const unsigned per_wave = (n + kMoveBlock - 1) / kMoveBlock * kWave;
  const unsigned from = min(n, in_block * per_wave), to = min(n, from + per_wave);
  int key = from + lane < to ? key_of(ids[from + lane], experts) : experts;
  route_prepare(s, key, ids, n, 0u, from, to, true, experts, align, (const int *)nullptr, 1u, 1u);
  for (unsigned i0 = from; i0 < to; i0 += kWave) {
    const unsigned i = i0 + lane;
    if (i0 != from) key = i < to ? key_of(ids[i], experts) : experts;
    const int at = route_step(s, key, experts, bits);
    if (i < to) {
      place[i] = at;
      if (leaves) {
        position[i] = at;
        if (at >= 0) order[at] = (int)i;
      }
    }
  }
  __syncthreads();
  if (leaves) {
    for (int e = tid; e < experts; e += kMoveBlock) {
      counts[e] = s.total[e];
      offsets[e] = s.offset[e];
    }
    if (tid == 0) offsets[experts] = s.offset[experts];
  }
  const unsigned wave = (d.first_block + blockIdx.x) * kMoveWaves + in_block;
  if (wave >= d.token_waves) {
    const unsigned first = (wave - d.token_waves) * kZeroRows, r = first + lane;
    const bool empty = lane < (int)kZeroRows && r < d.rows && row_empty(s, (int)r, experts);
    if (empty) order[r] = -1;
    clear_rows<E, true>(out, out_stride, first, empty, d.width);
    return;
  }
  const unsigned t = wave / d.splits;
  const int p = lane < (int)d.k ? place[t * d.k + lane] : -1;
  const unsigned split = wave % d.splits;
  const E *row = x + (size_t)t * x_stride;
  dispatch_token<E, true>(out, out_stride, row, p, split, d, first_values(row, split, d));
}

// More choices: a block makes the places of its own share of the tokens and
// moves them, two blocks to a CU, so the places cost no launch and no pass over
// them of their own (kPlaceAndMove: where, and what it measured).  Bound by HBM:
// 4099 tokens of 1001 floats, 3 choices, 68 MB in 20.4 us a pass.
template <typename E, typename I, bool NT>
__global__ __launch_bounds__(kSortBlock) void route_place_dispatch_kernel(
    E *__restrict__ out, size_t out_stride, const E *__restrict__ x, size_t x_stride, const I *__restrict__ ids,
    int experts, int bits, int align, const int *__restrict__ hist, unsigned per_hist, unsigned hist_parts,
    int *position, int *__restrict__ order, int *__restrict__ counts, int *__restrict__ offsets, Shape d) {
  __shared__ SortShared<kSortWaves> s;
  const unsigned n = d.tokens * d.k;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const unsigned first = (unsigned)((uint64_t)d.tokens * blockIdx.x / gridDim.x);
  const unsigned last = (unsigned)((uint64_t)d.tokens * (blockIdx.x + 1) / gridDim.x);
  const unsigned lo = first * d.k, hi = last * d.k;
  const unsigned per_wave = (hi - lo + kSortBlock - 1) / kSortBlock * kWave;
  const unsigned from = min(hi, lo + wave * per_wave), to = min(hi, from + per_wave);
  int key = from + lane < to ? key_of(ids[from + lane], experts) : experts;
  route_prepare(s, key, ids, n, lo, from, to, false, experts, align, hist, per_hist, hist_parts);
  for (unsigned i0 = from; i0 < to; i0 += kWave) {
    const unsigned i = i0 + lane;
    if (i0 != from) key = i < to ? key_of(ids[i], experts) : experts;
    const int at = route_step(s, key, experts, bits);
    if (i < to) position[i] = at;
    if (at >= 0) order[at] = (int)i;
  }
  if (blockIdx.x == 0) {
    if (tid < experts) {
      counts[tid] = s.total[tid];
      offsets[tid] = s.offset[tid];
    }
    if (tid == 0) offsets[experts] = s.offset[experts];
  }
  __syncthreads();  // the block's positions are there
  // a unit, one split of a token: the next one's row is asked for before this one's is stored
  const unsigned units = (last - first) * d.splits;
  auto row_of = [&](unsigned u) { return x + (size_t)(first + u / d.splits) * x_stride; };
  auto places_of = [&](unsigned u) {
    return lane < (int)d.k ? position[(size_t)(first + u / d.splits) * d.k + lane] : -1;
  };
  int p = -1;
  typename Vec<E>::Raw v = (E)0.0f;
  if ((unsigned)wave < units) {
    p = places_of(wave);
    v = first_values(row_of(wave), wave % d.splits, d);
  }
  for (unsigned u = wave; u < units; u += kSortWaves) {
    const unsigned next = u + kSortWaves;
    int next_p = -1;
    typename Vec<E>::Raw next_v = v;
    if (next < units) {
      next_p = places_of(next);
      next_v = first_values(row_of(next), next % d.splits, d);
    }
    dispatch_token<E, NT>(out, out_stride, row_of(u), p, u % d.splits, d, v);
    p = next_p;
    v = next_v;
  }
  // rows that hold no choice
  for (unsigned r0 = (blockIdx.x * kSortWaves + wave) * kZeroRows; r0 < d.rows; r0 += gridDim.x * kSortWaves * kZeroRows) {
    const unsigned r = r0 + lane;
    const bool empty = lane < (int)kZeroRows && r < d.rows && row_empty(s, (int)r, experts);
    if (empty) order[r] = -1;
    clear_rows<E, NT>(out, out_stride, r0, empty, d.width);
  }
}

// Weights: none (1), float, or the rows' own type.
enum WeightType { kNoWeights = 0, kFloatWeights = 1, kRowWeights = 2 };

template <typename E>
__device__ __forceinline__ float weight_at(const void *w, int type, size_t i) {
  return type == kFloatWeights ? static_cast<const float *>(w)[i]
         : type == kRowWeights ? (float)static_cast<const E *>(w)[i]
                               : 1.0f;
}

// combine: a wave's lanes hold the token's rows and weights, and hand them out.
// Bound by HBM: 16384 tokens of 4096 bf16, 8 choices, 1.21 GB in 211 us, 5.7 TB/s.
// G held choices from `left` on: their rows' 16 bytes are all asked for before
// the first is used.
template <typename E, int G, bool NT>
__device__ __forceinline__ void combine_group(typename Vec<E>::F &acc, uint64_t &left, const E *__restrict__ rows,
                                              size_t stride, int p, float w, unsigned c, bool whole, unsigned width) {
  using V = Vec<E>;
  typename V::Raw v[G];
  float f[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int from = __ffsll((long long)left) - 1;
    left &= left - 1;
    const E *row = rows + (size_t)__builtin_amdgcn_readlane(p, from) * stride + c;
    f[g] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), from));
    v[g] = whole ? load_raw<E, NT>(row) : load_part(row, width - c);
  }
#pragma unroll
  for (int g = 0; g < G; ++g) acc += f[g] * to_float<E>(v[g]);  // choices in order, in 32 bits
}

template <typename E, bool NT>
__global__ __launch_bounds__(kMoveBlock) void route_combine_kernel(E *__restrict__ y, size_t y_stride,
                                                                   const E *__restrict__ rows, size_t row_stride,
                                                                   const int *__restrict__ position,
                                                                   const void *__restrict__ weights, int weight_type,
                                                                   Shape d) {
  using V = Vec<E>;
  const unsigned wave = (d.first_block + blockIdx.x) * kMoveWaves + threadIdx.x / kWave;
  const int lane = threadIdx.x % kWave;
  if (wave >= d.token_waves) return;
  const unsigned t = wave / d.splits, split = wave % d.splits;
  const size_t a = (size_t)t * d.k + lane;
  const int p = lane < (int)d.k ? position[a] : -1;
  const float w = lane < (int)d.k ? weight_at<E>(weights, weight_type, a) : 0.0f;
  const uint64_t held = __ballot((unsigned)p < d.rows);
  E *to = y + (size_t)t * y_stride;
  for (unsigned c = (split * kWave + lane) * V::N; c < d.width; c += d.splits * kWave * V::N) {
    const bool whole = c + V::N <= d.width;
    typename V::F acc = 0.0f;
    uint64_t left = held;
    int n = __popcll(held);
    for (; n >= 8; n -= 8) combine_group<E, 8, NT>(acc, left, rows, row_stride, p, w, c, whole, d.width);
    if (n >= 4) combine_group<E, 4, NT>(acc, left, rows, row_stride, p, w, c, whole, d.width), n -= 4;
    if (n >= 2) combine_group<E, 2, NT>(acc, left, rows, row_stride, p, w, c, whole, d.width), n -= 2;
    if (n >= 1) combine_group<E, 1, NT>(acc, left, rows, row_stride, p, w, c, whole, d.width);
    if (whole)
      store_raw<E, true>(to + c, from_float<E>(acc));
    else
      store_part(to + c, from_float<E>(acc), d.width - c);
  }
}

// ---------------------------------------------------------------------------
// The gradient of combine: d_rows[position[a]] = w[a] * dy[t], d_w[a] = dy[t] .
// rows[position[a]].  dy is read once per group of up to 8 choices; the dots
// are 32-bit sums, lane by lane, then over the wave, then over the splits' waves
// in their order.  Bound by HBM: 8192 tokens of 2048 bf16, 8 choices, 571 MB in
// 102 us, 5.6 TB/s.
// ---------------------------------------------------------------------------
template <typename E, int G, bool NT>
__device__ __forceinline__ void grad_group(uint64_t &left, E *__restrict__ d_rows, size_t d_stride,
                                           const E *__restrict__ dy, const E *__restrict__ rows, size_t row_stride,
                                           int p, float w, unsigned first, unsigned step, unsigned width, float &dot) {
  using V = Vec<E>;
  const int lane = threadIdx.x % kWave;
  int from[G];
  float f[G], sum[G];
  size_t at[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    from[g] = __ffsll((long long)left) - 1;
    left &= left - 1;
    at[g] = (size_t)__builtin_amdgcn_readlane(p, from[g]);
    f[g] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), from[g]));
    sum[g] = 0.0f;
  }
  for (unsigned c = first; c < width; c += step) {
    const bool whole = c + V::N <= width;
    const int part = (int)(width - c);
    const typename V::F o = to_float<E>(whole ? load_raw(dy + c) : load_part(dy + c, part));
    typename V::Raw v[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const E *row = rows + at[g] * row_stride + c;
      v[g] = whole ? load_raw<E, NT>(row) : load_part(row, part);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const typename V::F r = to_float<E>(v[g]);
#pragma unroll
      for (int i = 0; i < V::N; ++i) sum[g] += o[i] * r[i];
      E *row = d_rows + at[g] * d_stride + c;
      const typename V::Raw out = from_float<E>(f[g] * o);
      if (whole)
        store_raw<E, true>(row, out);
      else
        store_part(row, out, part);
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float total = wave_sum(sum[g]);
    if (lane == from[g]) dot = total;
  }
}

// S waves share a token (d.splits = S); a block holds kMoveWaves / S tokens.
template <typename E, int S, bool NT>
__global__ __launch_bounds__(kMoveBlock) void route_combine_grad_kernel(
    E *__restrict__ d_rows, size_t d_stride, void *__restrict__ d_weights, const E *__restrict__ dy, size_t dy_stride,
    const E *__restrict__ rows, size_t row_stride, const int *__restrict__ position, const int *__restrict__ order,
    const void *__restrict__ weights, int weight_type, Shape d) {
  using V = Vec<E>;
  __shared__ float part[kMoveWaves][kWave];
  const unsigned in_block = threadIdx.x / kWave;
  const unsigned wave = (d.first_block + blockIdx.x) * kMoveWaves + in_block;
  const int lane = threadIdx.x % kWave;
  const bool moves = wave < d.token_waves;
  if (!moves) {  // these waves clear, and meet the others at the barrier below
    const unsigned first = (wave - d.token_waves) * kZeroRows, at = first + lane;
    const bool look = lane < (int)kZeroRows && at < d.rows;
    const int o = look ? order[at] : 0;
    clear_rows<E, true>(d_rows, d_stride, first, look && (o < 0 || (unsigned)o >= d.tokens * d.k), d.width);
  }
  const unsigned t = wave / S, split = wave % S;
  const size_t a = (size_t)t * d.k + lane;
  const bool mine = moves && lane < (int)d.k;
  const int p = mine ? position[a] : -1;
  const uint64_t held = __ballot((unsigned)p < d.rows);
  float dot = 0.0f;
  if (moves) {
    const float w = mine ? weight_at<E>(weights, weight_type, a) : 0.0f;
    const E *o = dy + (size_t)t * dy_stride;
    const unsigned first = (split * kWave + lane) * V::N, step = S * kWave * V::N;
    uint64_t left = held;
    int n = __popcll(held);
    for (; n >= 8; n -= 8) grad_group<E, 8, NT>(left, d_rows, d_stride, o, rows, row_stride, p, w, first, step, d.width, dot);
    if (n >= 4) grad_group<E, 4, NT>(left, d_rows, d_stride, o, rows, row_stride, p, w, first, step, d.width, dot), n -= 4;
    if (n >= 2) grad_group<E, 2, NT>(left, d_rows, d_stride, o, rows, row_stride, p, w, first, step, d.width, dot), n -= 2;
    if (n >= 1) grad_group<E, 1, NT>(left, d_rows, d_stride, o, rows, row_stride, p, w, first, step, d.width, dot);
  }
  if constexpr (S > 1) {
    part[in_block][lane] = dot;
    __syncthreads();
    if (split == 0) {
      dot = 0.0f;
#pragma unroll
      for (int s = 0; s < S; ++s) dot += part[in_block + s][lane];
    }
  }
  if (mine && split == 0) {
    if (weight_type == kRowWeights)
      static_cast<E *>(d_weights)[a] = (E)dot;
    else
      static_cast<float *>(d_weights)[a] = dot;
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
// Up to this many choices every block counts them all for itself: one launch
// (4.6 us at 4096 choices, 5.5 at 8192, 7.2 at 16384, against 6.3, 6.7 and 7.3
// of two launches, the second of which costs the caller 3 more).
constexpr size_t kSelfCounted = GP_ROUTE_UNCOUNTED;
// Above, b blocks cost about 1.2 us for each of their n / (1024 b) steps and
// 2.6e-4 us for each of the b * experts counts that every block sums: least at
// b * b = 4.4 n / experts.  131072 choices of 512 experts: 25.5 us at 128
// blocks, 18.0 at 64, 16.1 at 32; of 128: 11.5, 10.3, 11.3.
constexpr size_t kMostSortBlocks = 1024;

// Up to this many bytes of tokens and of rows for them, the blocks that make the
// places also move the tokens: the launch that it saves is worth more than the
// blocks' fixed shares of the tokens cost.  In one launch (more than 16384
// choices: two), and in one more:
//   4099 tokens of 1001 floats, 3 choices (66 MB)   22.0 us, 27.5
//   700 of 7168 bf16, 6 choices (70 MB)             30.3 us, 33.0
//   2000 of 2048 bf16, 8 choices (74 MB)            47.6 us, 51.2
//   4000 of 2048 bf16, 4 choices (82 MB)            22.9 us, 24.2
//   6000 of 2048 bf16, 4 choices (123 MB)           28.1 us, 27.6
//   10000 of 4000 bf16, 1 choice (160 MB)           35.3 us, 32.3
//   8192 of 2048 bf16, 6 choices (235 MB)           47.2 us, 46.0
// The groups' padding is not counted: it is cleared after the moves, a block its
// share, by as many blocks as there are tokens, at most two to a CU.  From about
// 100 tokens that costs nothing (110 of 7168 bf16, 10 choices, 33344 rows, nearly
// all padding: 103 us, 102; 200 of 2048, 8 choices, 17728 rows: 18.7, 20.4); 17
// tokens are too few blocks (64 choices of 1024 experts in groups of 64, 65600
// rows of 4096: 267 us, 105).  The form of up to 1024 choices counts them in every
// block, those of padding too (128 choices of 512 experts in groups of 64, 8192
// rows of 7168: 25.9 us, 30.1).
constexpr size_t kPlaceAndMove = (size_t)96 << 20;

struct SortPlan {
  unsigned blocks, per_block;
  bool counted;  // by route_count_kernel
  int bits;
};

SortPlan sort_plan(size_t n, size_t experts) {
  SortPlan p;
  const size_t unit = kSortBlock;  // every wave takes whole steps of 64
  size_t most = 1;
  while (most < kMostSortBlocks && (most + 1) * (most + 1) * experts <= 4 * n + n / 2) ++most;
  size_t per = n > kSelfCounted ? (n + most - 1) / most : unit;
  per = (per + unit - 1) / unit * unit;
  p.counted = n > kSelfCounted;
  p.per_block = (unsigned)per;
  p.blocks = (unsigned)((n + per - 1) / per);
  p.bits = 1;
  while ((1u << p.bits) < experts + 1) ++p.bits;  // `experts` itself stands for no expert
  return p;
}

int check_groups(size_t tokens, size_t k, size_t experts, size_t align) {
  GP_REQUIRE(k >= 1 && k <= (size_t)kMaxChoices, "choices per token must be 1 to 64");
  GP_REQUIRE(experts >= 1 && experts <= (size_t)kMaxExperts, "experts must be 1 to 1024");
  GP_REQUIRE(align >= 1 && align <= (1u << 20), "align must be 1 to 2^20");
  GP_REQUIRE(tokens <= (size_t)INT32_MAX / k, "tokens * choices must be under 2^31");
  const size_t n = tokens * k;
  GP_REQUIRE(n + (n < experts ? n : experts) * (align - 1) <= (size_t)INT32_MAX, "grouped rows must be under 2^31");
  return GP_OK;
}

size_t grouped_rows(size_t tokens, size_t k, size_t experts, size_t align) {
  const size_t n = tokens * k;
  return (n + (n < experts ? n : experts) * (align - 1)) / align * align;
}

int check_move(size_t tokens, size_t k, size_t rows, size_t width, int type) {
  GP_REQUIRE(type_known(type), "row type must be GP_F32, GP_BF16 or GP_F16");
  GP_REQUIRE(k >= 1 && k <= (size_t)kMaxChoices, "choices per token must be 1 to 64");
  GP_REQUIRE(tokens <= (size_t)INT32_MAX / k, "tokens * choices must be under 2^31");
  GP_REQUIRE(rows <= (size_t)INT32_MAX, "grouped rows must be under 2^31");
  GP_REQUIRE(width <= (1u << 24), "row width must be at most 2^24");
  return GP_OK;
}

// Waves over a token's columns: `least`, where there are as many steps of 64
// lanes, more when tokens are few, until the chip has 4 waves per SIMD.  They
// keep a row's accesses together in time (8192 tokens of 2048 bf16, 8 choices:
// dispatch 52 us, 64 with 2 waves).  Eight for combine, and for dispatch with up
// to three choices (30000 tokens of 2048 floats, 3 choices: 175 us, 178 with
// four; 1 choice of 4000 bf16: 91, 95); with more choices four (20000 of 7168
// bf16, 4 choices: 268 us, 289 with eight; 16384 of 4096, 8 choices: 245, 253).
unsigned pick_splits(size_t tokens, size_t width, int type, size_t least) {
  const size_t per_step = kWave * 16 / type_size(type);
  const size_t steps = (width + per_step - 1) / per_step;
  const size_t want = (size_t)device_cus() * 16;
  size_t s = tokens ? want / tokens : 1;
  if (s < least) s = least;
  return (unsigned)(s < steps ? s : (steps ? steps : 1));
}

// Every row starts on a boundary of `bytes`.
bool rows_start_at(size_t bytes, const void *p, size_t stride, int type) {
  return ((reinterpret_cast<uintptr_t>(p) | stride * type_size(type)) & (bytes - 1)) == 0;
}
constexpr size_t kLine = 128;

int check_grid(size_t waves, size_t *blocks) {
  GP_REQUIRE(waves <= UINT32_MAX, "too many rows for one call");
  *blocks = (waves + kMoveWaves - 1) / kMoveWaves;
  return GP_OK;
}

// A grid has at most 2^32 threads: longer ones go in several launches.
constexpr size_t kMostBlocks = (size_t)1 << 23;

template <typename F>
void launch_moves(size_t blocks, Shape d, F launch) {
  for (size_t b = 0; b < blocks; b += kMostBlocks) {
    d.first_block = (unsigned)b;
    launch(dim3((unsigned)(blocks - b < kMostBlocks ? blocks - b : kMostBlocks)), d);
  }
}

#define GP_TRY(expr)             \
  do {                           \
    const int rc_ = (expr);      \
    if (rc_ != GP_OK) return rc_; \
  } while (0)

// f(E{}) with the element type of `type`.
template <typename F>
void with_type(int type, F f) {
  if (type == GP_F32)
    f((float)0);
  else if (type == GP_BF16)
    f((__bf16)0.0f);
  else
    f((_Float16)0);
}

template <typename I>
void launch_sort(const void *ids, const SortPlan &p, size_t n, int experts, int align, size_t rows, int *position,
                 int *order, int *counts, int *offsets, int *hist, hipStream_t s) {
  const I *in = static_cast<const I *>(ids);
  if (p.counted)
    hipLaunchKernelGGL((route_count_kernel<I>), dim3(p.blocks), dim3(kSortBlock), 0, s, in, (unsigned)n, p.per_block,
                       experts, hist);
  hipLaunchKernelGGL((route_place_kernel<I>), dim3(p.blocks), dim3(kSortBlock), 0, s, in, (unsigned)n, p.per_block,
                     experts, p.bits, align, (unsigned)rows, p.counted ? (const int *)hist : nullptr, position, order, counts, offsets);
}

size_t strided_bytes(size_t rows, size_t stride, size_t width, int type) {
  return rows && width ? ((rows - 1) * stride + width) * type_size(type) : 0;
}

// Two sets of rows of one width share a value.  Rows of one stride, as columns of
// one buffer are, lie in windows of it that repeat, and may pass between each
// other; of two strides only the spans are looked at.
bool rows_overlap(const void *a, size_t a_rows, size_t a_stride, const void *b, size_t b_rows, size_t b_stride,
                  size_t width, int type) {
  if (!bytes_overlap(a, strided_bytes(a_rows, a_stride, width, type), b, strided_bytes(b_rows, b_stride, width, type)))
    return false;
  if (a_rows == 1) a_stride = b_stride;  // a single row has any
  if (b_rows == 1) b_stride = a_stride;
  if (a_stride != b_stride) return true;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  const size_t bytes = width * type_size(type), step = a_stride * type_size(type);
  const size_t apart = x >= y ? (x - y) % step : (step - (y - x) % step) % step;  // from b's window to a's
  return apart < bytes || step - apart < bytes;
}

int plan_dispatch(const void *out, size_t out_stride, const void *x, size_t x_stride, int type, size_t tokens,
                  size_t k, size_t rows, size_t width, Shape *d, size_t *blocks) {
  GP_TRY(check_move(tokens, k, rows, width, type));
  GP_REQUIRE(out && (tokens == 0 || x), "null out or x");
  GP_REQUIRE(out_stride >= width && x_stride >= width, "row stride smaller than the width");
  GP_REQUIRE(!rows_overlap(out, rows, out_stride, x, tokens, x_stride, width, type), "out overlaps x");
  *d = Shape{(unsigned)tokens, (unsigned)k, (unsigned)rows, (unsigned)width, pick_splits(tokens, width, type, k < 4 ? 8 : 4), 0, 0};
  const size_t waves = tokens * (size_t)d->splits;
  GP_TRY(check_grid(waves + (rows + kZeroRows - 1) / kZeroRows, blocks));
  d->token_waves = (unsigned)waves;
  return GP_OK;
}

}  // namespace

extern "C" {

int gp_route_rows(size_t tokens, size_t k, size_t experts, size_t align, size_t *rows) {
  GP_REQUIRE(rows, "null rows");
  GP_TRY(check_groups(tokens, k, experts, align));
  *rows = grouped_rows(tokens, k, experts, align);
  return GP_OK;
}

int gp_route_workspace(size_t tokens, size_t k, size_t experts, size_t *bytes) {
  GP_REQUIRE(bytes, "null bytes");
  GP_TRY(check_groups(tokens, k, experts, 1));
  const SortPlan p = sort_plan(tokens * k, experts);
  *bytes = p.counted ? (size_t)p.blocks * experts * sizeof(int) : 0;
  return GP_OK;
}

int gp_route_sort(const void *ids, int id_bits, size_t tokens, size_t k, size_t experts, size_t align,
                  int32_t *position, int32_t *order, int32_t *counts, int32_t *offsets, void *workspace,
                  size_t workspace_bytes, gp_stream s) {
  GP_REQUIRE(id_bits == 32 || id_bits == 64, "ids must be 32 or 64 bits wide");
  size_t need = 0;
  GP_TRY(check_groups(tokens, k, experts, align));
  GP_TRY(gp_route_workspace(tokens, k, experts, &need));
  GP_REQUIRE(counts && offsets, "null counts or offsets");
  const size_t n = tokens * k;
  GP_REQUIRE(n == 0 || (ids && position && order), "null ids, position or order");
  GP_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "workspace missing or too small");
  SortPlan p = sort_plan(n, experts);
  if (p.blocks == 0) p.blocks = 1;  // no tokens: the empty groups
  const size_t rows = grouped_rows(tokens, k, experts, align);
  int *hist = static_cast<int *>(workspace);
  if (id_bits == 64)
    launch_sort<int64_t>(ids, p, n, (int)experts, (int)align, rows, position, order, counts, offsets, hist,
                         (hipStream_t)s);
  else
    launch_sort<int32_t>(ids, p, n, (int)experts, (int)align, rows, position, order, counts, offsets, hist,
                         (hipStream_t)s);
  GP_HIP_TRY(hipGetLastError());
  return GP_OK;
}

int gp_route_dispatch(void *out, size_t out_stride, const void *x, size_t x_stride, int type,
                      const int32_t *position, const int32_t *order, size_t tokens, size_t k, size_t rows,
                      size_t width, gp_stream s) {
  GP_TRY(check_move(tokens, k, rows, width, type));
  if (rows == 0 || width == 0) return GP_OK;
  GP_REQUIRE(order && (tokens == 0 || position), "null position or order");
  Shape d;
  size_t blocks = 0;
  GP_TRY(plan_dispatch(out, out_stride, x, x_stride, type, tokens, k, rows, width, &d, &blocks));
  with_type(type, [&](auto e) {
    using E = decltype(e);
    auto go = [&](auto kernel) {
      launch_moves(blocks, d, [&](dim3 grid, Shape d) {
        hipLaunchKernelGGL(kernel, grid, dim3(kMoveBlock), 0, (hipStream_t)s, static_cast<E *>(out), out_stride,
                           static_cast<const E *>(x), x_stride, position, order, d);
      });
    };
    if (rows_start_at(kLine, out, out_stride, type))
      go(route_dispatch_kernel<E, true>);
    else
      go(route_dispatch_kernel<E, false>);
  });
  GP_HIP_TRY(hipGetLastError());
  return GP_OK;
}

int gp_route_sort_dispatch(void *out, size_t out_stride, const void *x, size_t x_stride, int type, const void *ids,
                           int id_bits, size_t tokens, size_t k, size_t experts, size_t align, size_t width,
                           int32_t *position, int32_t *order, int32_t *counts, int32_t *offsets, void *workspace,
                           size_t workspace_bytes, gp_stream s) {
  GP_TRY(check_groups(tokens, k, experts, align));
  const size_t rows = grouped_rows(tokens, k, experts, align), n = tokens * k;
  if (n == 0 || width == 0 || (n > kSmallRoute && (n + tokens) * width * type_size(type) > kPlaceAndMove)) {
    GP_TRY(check_move(tokens, k, rows, width, type));
    GP_TRY(gp_route_sort(ids, id_bits, tokens, k, experts, align, position, order, counts, offsets, workspace,
                         workspace_bytes, s));
    return gp_route_dispatch(out, out_stride, x, x_stride, type, position, order, tokens, k, rows, width, s);
  }
  GP_REQUIRE(id_bits == 32 || id_bits == 64, "ids must be 32 or 64 bits wide");
  GP_REQUIRE(ids && position && order && counts && offsets, "null ids, position, order, counts or offsets");
  Shape d;
  size_t blocks = 0;
  GP_TRY(plan_dispatch(out, out_stride, x, x_stride, type, tokens, k, rows, width, &d, &blocks));
  const SortPlan p = sort_plan(n, experts);
  int *hist = p.counted ? static_cast<int *>(workspace) : nullptr;
  GP_REQUIRE(!p.counted || (hist && workspace_bytes >= (size_t)p.blocks * experts * sizeof(int)),
             "workspace missing or too small");
  with_type(type, [&](auto e) {
    using E = decltype(e);
    auto go = [&](auto id) {
      using I = decltype(id);
      const I *in = static_cast<const I *>(ids);
      if (n <= kSmallRoute) {
        launch_moves(blocks, d, [&](dim3 grid, Shape d) {
          hipLaunchKernelGGL((route_sort_dispatch_kernel<E, I>), grid, dim3(kMoveBlock), 0, (hipStream_t)s,
                             static_cast<E *>(out), out_stride, static_cast<const E *>(x), x_stride, in, (int)experts,
                             p.bits, (int)align, position, order, counts, offsets, d);
        });
        return;
      }
      if (p.counted)
        hipLaunchKernelGGL((route_count_kernel<I>), dim3(p.blocks), dim3(kSortBlock), 0, (hipStream_t)s, in,
                           (unsigned)n, p.per_block, (int)experts, hist);
      const size_t most = (size_t)device_cus() * 2;
      auto move = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(tokens < most ? tokens : most)), dim3(kSortBlock), 0,
                           (hipStream_t)s, static_cast<E *>(out), out_stride, static_cast<const E *>(x), x_stride, in,
                           (int)experts, p.bits, (int)align, (const int *)hist, p.per_block, p.blocks, position, order,
                           counts, offsets, d);
      };
      if (rows_start_at(kLine, out, out_stride, type))
        move(route_place_dispatch_kernel<E, I, true>);
      else
        move(route_place_dispatch_kernel<E, I, false>);
    };
    id_bits == 64 ? go((int64_t)0) : go((int32_t)0);
  });
  GP_HIP_TRY(hipGetLastError());
  return GP_OK;
}

int gp_route_combine(void *y, size_t y_stride, const void *rows_in, size_t row_stride, int type,
                     const int32_t *position, const void *weights, int weight_type, size_t tokens, size_t k,
                     size_t rows, size_t width, gp_stream s) {
  GP_TRY(check_move(tokens, k, rows, width, type));
  GP_REQUIRE(!weights || weight_type == GP_F32 || weight_type == type, "weights must be GP_F32 or of the rows' type");
  if (tokens == 0 || width == 0) return GP_OK;
  GP_REQUIRE(y && position && (rows == 0 || rows_in), "null y, rows or position");
  GP_REQUIRE(y_stride >= width && row_stride >= width, "row stride smaller than the width");
  GP_REQUIRE(!rows_overlap(y, tokens, y_stride, rows_in, rows, row_stride, width, type), "y overlaps the rows");
  const int wt = !weights ? kNoWeights : weight_type == GP_F32 ? kFloatWeights : kRowWeights;
  Shape d{(unsigned)tokens, (unsigned)k, (unsigned)rows, (unsigned)width, pick_splits(tokens, width, type, 8), 0, 0};
  const size_t waves = tokens * (size_t)d.splits;
  size_t blocks = 0;
  GP_TRY(check_grid(waves, &blocks));
  d.token_waves = (unsigned)waves;
  with_type(type, [&](auto e) {
    using E = decltype(e);
    auto go = [&](auto kernel) {
      launch_moves(blocks, d, [&](dim3 grid, Shape d) {
        hipLaunchKernelGGL(kernel, grid, dim3(kMoveBlock), 0, (hipStream_t)s, static_cast<E *>(y), y_stride,
                           static_cast<const E *>(rows_in), row_stride, position, weights, wt, d);
      });
    };
    if (rows_start_at(16, rows_in, row_stride, type))
      go(route_combine_kernel<E, true>);
    else
      go(route_combine_kernel<E, false>);
  });
  GP_HIP_TRY(hipGetLastError());
  return GP_OK;
}

int gp_route_combine_grad(void *d_rows, size_t d_stride, void *d_weights, const void *dy, size_t dy_stride,
                          const void *rows_in, size_t row_stride, int type, const int32_t *position,
                          const int32_t *order, const void *weights, int weight_type, size_t tokens, size_t k,
                          size_t rows, size_t width, gp_stream s) {
  GP_TRY(check_move(tokens, k, rows, width, type));
  GP_REQUIRE(weight_type == GP_F32 || weight_type == type, "weights must be GP_F32 or of the rows' type");
  if (tokens == 0 && rows == 0) return GP_OK;
  GP_REQUIRE(tokens == 0 || (position && weights && d_weights), "null position or weights");
  GP_REQUIRE(rows == 0 || order, "null order");
  GP_REQUIRE(width == 0 || ((tokens == 0 || dy) && (rows == 0 || (d_rows && rows_in))), "null dy, rows or d_rows");
  GP_REQUIRE(d_stride >= width && dy_stride >= width && row_stride >= width, "row stride smaller than the width");
  GP_REQUIRE(!rows_overlap(d_rows, rows, d_stride, dy, tokens, dy_stride, width, type), "d_rows overlaps dy");
  GP_REQUIRE(!rows_overlap(d_rows, rows, d_stride, rows_in, rows, row_stride, width, type),
             "d_rows overlaps the rows");
  const int wt = weight_type == GP_F32 ? kFloatWeights : kRowWeights;
  // A token's waves meet for its weights' gradients: four, a block (16384 tokens
  // of 1000 floats, 4 choices: 99 us, 105 with two, 113 with one); two where the
  // row has two steps for them (16384 of 600 bf16, 8 choices: 72 us, 88 with
  // four); one for short rows off a 16-byte boundary, whose lines they would
  // share, and for rows of one step.  Short rows off the boundary want four waves
  // while tokens are few, and where that ends lies between 2000 and 4000 tokens by
  // width and type; 4096 is late for the narrowest.  One wave, two, four:
  //                              2000 tokens        4000 tokens        8192 tokens
  //   1001 bf16, 3 choices    14.4 14.7 10.7 us  14.1 14.2 20.3 us  23.6 27.0 36.1 us
  //   333 floats, 4 choices   14.6 14.6 11.3     14.3 14.4 14.7     20.6 22.2 28.3
  //   777 floats, 5 choices   14.5 14.5 16.5     26.6 27.2 28.4     52.0 49.2 51.3
  //   1999 fp16, 4 choices    15.7 15.4 18.4     27.3 28.5 32.8     50.9 51.7 58.9
  const bool aligned = rows_start_at(16, rows_in, row_stride, type);
  const size_t step = kWave * 16 / type_size(type), steps = (width + step - 1) / step;
  const bool one = steps <= 1 || (!aligned && steps <= 4 && tokens >= 4096);
  const unsigned splits = one ? 1 : steps == 2 ? 2 : 4;
  Shape d{(unsigned)tokens, (unsigned)k, (unsigned)rows, (unsigned)width, splits, 0, 0};
  const size_t waves = tokens * (size_t)d.splits;
  size_t blocks = 0;
  GP_TRY(check_grid(waves + (rows + kZeroRows - 1) / kZeroRows, &blocks));
  d.token_waves = (unsigned)waves;
  with_type(type, [&](auto e) {
    using E = decltype(e);
    auto go = [&](auto kernel) {
      launch_moves(blocks, d, [&](dim3 grid, Shape d) {
        hipLaunchKernelGGL(kernel, grid, dim3(kMoveBlock), 0, (hipStream_t)s, static_cast<E *>(d_rows), d_stride,
                           d_weights, static_cast<const E *>(dy), dy_stride, static_cast<const E *>(rows_in),
                           row_stride, position, order, weights, wt, d);
      });
    };
    auto pick = [&](auto s) {
      constexpr int S = decltype(s)::value;
      if (aligned)
        go(route_combine_grad_kernel<E, S, true>);
      else
        go(route_combine_grad_kernel<E, S, false>);
    };
    if (splits == 4)
      pick(std::integral_constant<int, 4>());
    else if (splits == 2)
      pick(std::integral_constant<int, 2>());
    else
      pick(std::integral_constant<int, 1>());
  });
  GP_HIP_TRY(hipGetLastError());
  return GP_OK;
}

}  // extern "C"
