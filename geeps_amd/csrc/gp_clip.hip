// gp_clip.hip — updates scaled to a bound on their norm (include/gp_reduce.h):
// a list of gradients (a grad plan), and the server's N-way sum of client
// deltas (gp_bucket_sum_apply's operands) added to the master.
//
//   norm = sqrt(sum of squares),  f = scale * min(1, max_norm / norm)
//
// Two passes, because f needs every value: the first reads the values and
// leaves one 64-bit partial sum of squares per block, the second adds the
// partials up in each block (in one order: every block, and every run, gets the
// same f) and writes f times the values.  No counter, no atomic, no third
// launch.  Squares and sums are 64-bit: a float's square passes the float range
// from 1.8e19 up and vanishes from 1e-23 down, and the sum of 10^9 of them in
// 32 bits would lose the small ones; the 64-bit multiply-adds are hidden behind
// the loads.

#include <algorithm>
#include <new>
#include <vector>

#include "gp_device.hpp"

namespace {

constexpr int kClipBlock = 256;
constexpr int kClipBlocksPerCU = 8;
constexpr unsigned kMostPartials = GP_CLIP_WORKSPACE_BYTES / sizeof(double);
constexpr int kMostStreams = 8;  // buckets that one launch reads

struct Bound {
  double max_norm, scale;
  int skip;  // a norm that is no finite number: nothing is added, zeros are written
};

struct Factor {
  float f;
  bool skip;
};

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kClipBlock / kWave];
  v = wave_sum(v);
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
  __syncthreads();
  double total = part[0];
#pragma unroll
  for (int w = 1; w < kClipBlock / kWave; ++w) total += part[w];
  return total;
}

__device__ __forceinline__ double sum_partials(const double *__restrict__ partial, unsigned count) {
  double v = 0.0;
#pragma unroll 8
  for (unsigned i = threadIdx.x; i < count; i += kClipBlock) v += partial[i];
  return block_sum(v);
}

// The block's view of f; the first block also leaves the norm.
__device__ __forceinline__ Factor clip_factor(const double *__restrict__ partial, unsigned count, const Bound &b,
                                              float *__restrict__ norm_out) {
  const double norm = sqrt(sum_partials(partial, count));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const double f = b.scale * (norm <= b.max_norm ? 1.0 : b.max_norm / norm);
  return {(float)f, b.skip && !(norm < __builtin_inf())};
}

__global__ __launch_bounds__(kClipBlock) void sum_partials_kernel(const double *__restrict__ partial, unsigned count,
                                                                  double *__restrict__ sum, float *__restrict__ norm) {
  const double total = sum_partials(partial, count);
  if (threadIdx.x == 0) {
    if (sum) *sum = total;
    if (norm) *norm = (float)sqrt(total);
  }
}

template <int N, typename F>
__device__ __forceinline__ void add_squares(double &sum, F v) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double d = (double)v[i];
    sum += d * d;
  }
}

// ---------------------------------------------------------------------------
// Grad plans: a list of gradients and of the buffers that their scaled values
// go to, cut into chunks of one length; a block takes every gridDim-th chunk.
// Bound by HBM: 604 M bf16, 1.21 GB squared in 180 us (6.7 TB/s), 2.42 GB scaled
// in 420 us (5.8 TB/s); a list of a few MB by its two launches, 11 us.
// ---------------------------------------------------------------------------
struct Chunk {
  const void *in;
  void *out;
  unsigned n;
  short type, out_type;
};

template <typename E, bool NT>
__device__ __forceinline__ void square_chunk(double &sum, const Chunk &c) {
  using V = Vec<E>;
  constexpr int U = 4;
  constexpr unsigned kStep = kClipBlock * V::N;
  const E *in = static_cast<const E *>(c.in);
  double acc[U] = {};
  unsigned i = threadIdx.x * V::N;
  for (; i + (U - 1) * kStep + V::N <= c.n; i += U * kStep) {
    typename V::Raw v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load_raw<E, NT>(in + i + u * kStep);
#pragma unroll
    for (int u = 0; u < U; ++u) add_squares<V::N>(acc[u], to_float<E>(v[u]));
  }
  for (; i < c.n; i += kStep)
    add_squares<V::N>(acc[0], to_float<E>(i + V::N <= c.n ? load_raw(in + i) : load_part(in + i, c.n - i)));
#pragma unroll
  for (int u = 0; u < U; ++u) sum += acc[u];
}

template <bool NT>
__device__ __forceinline__ void square_any(double &sum, const Chunk &c) {
  if (c.type == GP_F32)
    square_chunk<float, NT>(sum, c);
  else if (c.type == GP_BF16)
    square_chunk<__bf16, NT>(sum, c);
  else
    square_chunk<_Float16, NT>(sum, c);
}

// The first `past` chunks go past the caches (non-temporal), the others are left
// there for the second pass.
__global__ __launch_bounds__(kClipBlock) void grad_square_kernel(const Chunk *__restrict__ chunks, unsigned count,
                                                                 unsigned past, double *__restrict__ partial) {
  double sum = 0.0;
  Chunk next = {};
  if (blockIdx.x < count) next = chunks[blockIdx.x];
  for (unsigned k = blockIdx.x; k < count; k += gridDim.x) {
    const Chunk c = next;
    if (k + gridDim.x < count) next = chunks[k + gridDim.x];  // asked for before this chunk's values are
    if (k < past)
      square_any<true>(sum, c);
    else
      square_any<false>(sum, c);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// N values next to each other, wherever they start.
template <typename E, int N>
struct Group {
  typedef E Raw __attribute__((ext_vector_type(N)));
  typedef Raw Loose __attribute__((aligned(sizeof(E))));
  typedef float F __attribute__((ext_vector_type(N)));
};

// O: the gradient's own type, or float; one rounding.  Past the caches (61 M bf16
// 60 us, 74 through them; 61 M floats 116, not 144), whose lines the stores must
// then fill whole: a lane takes the values of 16 bytes of the output, next to its
// neighbours' (bf16 to float 77 us; 119 in 16-byte loads with two stores 32 bytes
// apart).  Rows that start off a 16-byte boundary gain less: 122 us, not 144.
template <typename E, typename O>
__device__ __forceinline__ void scale_chunk(const Chunk &c, const Factor &f) {
  constexpr int N = 16 / (int)sizeof(O);
  constexpr int U = 4 * (int)(sizeof(O) / sizeof(E));  // 64 bytes of a lane's loads in flight
  using G = Group<E, N>;
  using H = Group<O, N>;
  constexpr unsigned kStep = kClipBlock * N;
  const E *in = static_cast<const E *>(c.in);
  O *out = static_cast<O *>(c.out);
  auto load = [&](unsigned i) {
    return __builtin_nontemporal_load(reinterpret_cast<const typename G::Loose *>(in + i));
  };
  auto store = [&](unsigned i, typename G::Raw v) {
    const typename G::F s = f.skip ? (typename G::F)(0.0f) : f.f * __builtin_convertvector(v, typename G::F);
    __builtin_nontemporal_store(__builtin_convertvector(s, typename H::Raw),
                                reinterpret_cast<typename H::Loose *>(out + i));
  };
  unsigned i = threadIdx.x * N;
  for (; i + (U - 1) * kStep + N <= c.n; i += U * kStep) {
    typename G::Raw v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load(i + u * kStep);
#pragma unroll
    for (int u = 0; u < U; ++u) store(i + u * kStep, v[u]);
  }
  for (; i + N <= c.n; i += kStep) store(i, load(i));
  if (i < c.n) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j < c.n) out[i + j] = (O)(f.skip ? 0.0f : f.f * (float)in[i + j]);
  }
}

__global__ __launch_bounds__(kClipBlock) void grad_scale_kernel(const Chunk *__restrict__ chunks, unsigned count,
                                                                const double *__restrict__ partial, unsigned partials,
                                                                Bound b, float *__restrict__ norm) {
  const Factor f = clip_factor(partial, partials, b, norm);
  // last chunks first: they are what the caches still hold of the first pass
  for (unsigned k = blockIdx.x; k < count; k += gridDim.x) {
    const Chunk c = chunks[count - 1 - k];
    if (c.type == GP_F32)
      scale_chunk<float, float>(c, f);
    else if (c.type == GP_BF16)
      c.out_type == GP_F32 ? scale_chunk<__bf16, float>(c, f) : scale_chunk<__bf16, __bf16>(c, f);
    else
      c.out_type == GP_F32 ? scale_chunk<_Float16, float>(c, f) : scale_chunk<_Float16, _Float16>(c, f);
  }
}

// ---------------------------------------------------------------------------
// The server's sum.  s = b0 + b1 + ..., in bucket order, in 32 bits as
// gp_bucket_sum_apply adds them; out = in + f * s.
// ---------------------------------------------------------------------------
typedef Vec<float>::F f4;

struct Streams {
  const float *p[kMostStreams];
};

// Four block-strides of every bucket in flight, two blocks to a CU, the buckets
// past the caches, the sum into them.  Eight buckets of 61 M floats: 365 us
// (6.0 TB/s); 440 through the caches at two strides and eight blocks; 401 with
// the sum past the caches too.
constexpr int kSumU = 4;
constexpr int kSumBlocksPerCU = 2;

// s = (CARRY ? sum : 0) + b0 + ... + b{NB-1}; WRITE: left in `sum`; SQ: its squares.
template <int NB, bool CARRY, bool WRITE, bool SQ>
__global__ __launch_bounds__(kClipBlock) void sum_square_kernel(float *__restrict__ sum, Streams b, size_t n,
                                                                double *__restrict__ partial) {
  constexpr int U = kSumU;
  const size_t tile = (size_t)kClipBlock * 4 * U;
  double acc[U] = {};
  for (size_t base = blockIdx.x * tile; base < n; base += gridDim.x * tile) {
    const size_t i = base + threadIdx.x * 4;
    f4 s[U];
    if (base + tile <= n) {
      f4 v[NB][U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if constexpr (CARRY) s[u] = load_raw(sum + i + u * kClipBlock * 4);
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int u = 0; u < U; ++u) v[k][u] = load_raw<float, true>(b.p[k] + i + u * kClipBlock * 4);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u] = CARRY ? s[u] + v[0][u] : v[0][u];
#pragma unroll
        for (int k = 1; k < NB; ++k) s[u] += v[k][u];
        if constexpr (WRITE) store_raw(sum + i + u * kClipBlock * 4, s[u]);
        if constexpr (SQ) add_squares<4>(acc[u], s[u]);
      }
    } else {
      for (int u = 0; u < U; ++u) {
        const size_t at = i + u * kClipBlock * 4;
        if (at >= n) break;
        const int left = n - at < 4 ? (int)(n - at) : 4;
        f4 t = CARRY ? load_part(sum + at, left) : f4(0.0f);
        for (int k = 0; k < NB; ++k) {
          const f4 x = load_part(b.p[k] + at, left);
          t = !CARRY && k == 0 ? x : t + x;
        }
        if constexpr (WRITE) store_part(sum + at, t, left);
        if constexpr (SQ) add_squares<4>(acc[0], t);
      }
    }
  }
  if constexpr (SQ) {
    double total = 0.0;
#pragma unroll
    for (int u = 0; u < U; ++u) total += acc[u];
    total = block_sum(total);
    if (threadIdx.x == 0) partial[blockIdx.x] = total;
  }
}

// out = in + f * (b0 + ... + b{NB-1}); LEFT: b0 is the sum that the first pass
// left, partly still in the memory-side cache, and is read through the caches
// (61 M floats of three buckets: both passes 255 us, 271 past them), all else
// past them (one stream of 61 M floats: this pass 124 us, 136 through them).
template <int NB, bool LEFT>
__global__ __launch_bounds__(kClipBlock) void add_scaled_kernel(float *__restrict__ out, const float *__restrict__ in,
                                                                Streams b, size_t n,
                                                                const double *__restrict__ partial, unsigned partials,
                                                                Bound bound, float *__restrict__ norm) {
  constexpr int U = 4;
  const Factor f = clip_factor(partial, partials, bound, norm);
  const size_t tile = (size_t)kClipBlock * 4 * U;
  const size_t tiles = (n + tile - 1) / tile;
  for (size_t k = blockIdx.x; k < tiles; k += gridDim.x) {
    const size_t base = (tiles - 1 - k) * tile;  // last first, as grad_scale_kernel
    const size_t i = base + threadIdx.x * 4;
    if (base + tile <= n) {
      f4 m[U], v[NB][U];
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int u = 0; u < U; ++u) v[j][u] = load_raw<float, !LEFT>(b.p[j] + i + u * kClipBlock * 4);
#pragma unroll
      for (int u = 0; u < U; ++u) m[u] = load_raw<float, true>(in + i + u * kClipBlock * 4);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        f4 s = v[0][u];
#pragma unroll
        for (int j = 1; j < NB; ++j) s += v[j][u];
        store_raw<float, true>(out + i + u * kClipBlock * 4, f.skip ? m[u] : m[u] + f.f * s);
      }
    } else {
      for (int u = 0; u < U; ++u) {
        const size_t at = i + u * kClipBlock * 4;
        if (at >= n) break;
        const int left = n - at < 4 ? (int)(n - at) : 4;
        f4 s = load_part(b.p[0] + at, left);
        for (int j = 1; j < NB; ++j) s += load_part(b.p[j] + at, left);
        const f4 m = load_part(in + at, left);
        store_part(out + at, f.skip ? m : m + f.f * s, left);
      }
    }
  }
}

unsigned clip_grid(size_t units) {
  size_t g = (size_t)device_cus() * kClipBlocksPerCU;
  if (g > kMostPartials) g = kMostPartials;
  return (unsigned)(units < g ? (units ? units : 1) : g);
}

unsigned sum_grid(size_t n) {
  const size_t tile = (size_t)kClipBlock * 4 * kSumU, tiles = (n + tile - 1) / tile;
  const size_t most = (size_t)device_cus() * kSumBlocksPerCU;
  return clip_grid(tiles < most ? tiles : most);
}

template <bool CARRY, bool WRITE, bool SQ>
void launch_sum_square(int nb, float *sum, const Streams &b, size_t n, double *partial, hipStream_t s) {
  const dim3 grid(sum_grid(n)), block(kClipBlock);
#define GP_CASE(NB) \
  case NB: hipLaunchKernelGGL((sum_square_kernel<NB, CARRY, WRITE, SQ>), grid, block, 0, s, sum, b, n, partial); break
  switch (nb) {
    GP_CASE(1);
    GP_CASE(2);
    GP_CASE(3);
    GP_CASE(4);
    GP_CASE(5);
    GP_CASE(6);
    GP_CASE(7);
    GP_CASE(8);
  }
#undef GP_CASE
}

// From three buckets on their sum is left in `scratch` between the passes: N + 4
// streams in all up to kMostStreams buckets.  Each further kMostStreams take a
// launch of their own, which reads that sum and writes it again: N + 6 from 9 to
// 16, N + 8 at 17 (61 M floats: 8 buckets 467 us, 9 578, 16 859, 17 979; 64 K
// floats: 17.6, 20.8, 24.7, 28.1).  One or two are read again (2 N + 2).
constexpr int kReread = 2;

int launch_squares(float *scratch, const float *const *buckets, int nb, size_t n, double *partial, unsigned *partials,
                   hipStream_t s) {
  int done = 0;
  while (done < nb) {
    const int take = nb - done < kMostStreams ? nb - done : kMostStreams;
    Streams b = {};
    for (int k = 0; k < take; ++k) b.p[k] = buckets[done + k];
    const bool last = done + take == nb;
    if (nb <= kReread)
      launch_sum_square<false, false, true>(take, nullptr, b, n, partial, s);
    else if (done == 0 && last)
      launch_sum_square<false, true, true>(take, scratch, b, n, partial, s);
    else if (done == 0)
      launch_sum_square<false, true, false>(take, scratch, b, n, partial, s);
    else if (last)
      launch_sum_square<true, true, true>(take, scratch, b, n, partial, s);
    else
      launch_sum_square<true, true, false>(take, scratch, b, n, partial, s);
    if (last) *partials = sum_grid(n);
    done += take;
  }
  GP_HIP_TRY(hipGetLastError());
  return GP_OK;
}

int check_bound(double max_norm, double scale, int nonfinite) {
  GP_REQUIRE(max_norm >= 0.0, "max_norm must not be negative or NaN");
  GP_REQUIRE(scale - scale == 0.0, "scale must be finite");
  GP_REQUIRE(nonfinite == GP_CLIP_PROPAGATE || nonfinite == GP_CLIP_SKIP,
             "nonfinite must be GP_CLIP_PROPAGATE or GP_CLIP_SKIP");
  return GP_OK;
}

int check_buckets(const float *scratch, const float *const *buckets, int nb, size_t n) {
  GP_REQUIRE(nb >= 0, "negative bucket count");
  GP_REQUIRE(n <= SIZE_MAX / 8, "too many values");
  if (n == 0) return GP_OK;
  GP_REQUIRE(nb == 0 || buckets, "null buckets");
  for (int k = 0; k < nb; ++k) GP_REQUIRE(buckets[k], "null bucket");
  GP_REQUIRE(nb <= kReread || scratch, "null scratch: needed from three buckets on");
  if (nb > kReread)
    for (int k = 0; k < nb; ++k)
      GP_REQUIRE(!bytes_overlap(scratch, n * 4, buckets[k], n * 4), "scratch overlaps a bucket");
  return GP_OK;
}

// hipFree while a stream is being captured.
struct RelaxedCapture {
  hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
  RelaxedCapture() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
  ~RelaxedCapture() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
};

}  // namespace

struct gp_grad_plan_s {
  Chunk *chunks = nullptr;  // device
  size_t count = 0;
  size_t bytes = 0;  // of the gradients
  int device = -1;  // of an empty plan: any
};

namespace {

// What the memory-side cache holds of the gradients until the second pass, which
// starts where the first ended.  1.2 GB of bf16, both passes: 603 us; 2 % more
// with 192 or 384 MiB left there, 6 % with none, 8 % with all of it read through
// the caches.
constexpr size_t kCachedBytes = (size_t)256 << 20;

unsigned chunks_past(const gp_grad_plan_s *p) {
  if (p->bytes <= kCachedBytes) return 0;
  return (unsigned)((double)p->count * ((double)(p->bytes - kCachedBytes) / (double)p->bytes));
}

void launch_grad_square(const gp_grad_plan_s *p, unsigned grid, double *partial, hipStream_t s) {
  hipLaunchKernelGGL(grad_square_kernel, dim3(grid), dim3(kClipBlock), 0, s, (const Chunk *)p->chunks,
                     (unsigned)p->count, chunks_past(p), partial);
}

int check_grad_plan(const gp_grad_plan_s *p, const void *workspace) {
  GP_REQUIRE(p, "null grad plan");
  GP_REQUIRE(workspace, "null workspace");
  if (p->count == 0) return GP_OK;
  int dev = -1;
  GP_HIP_TRY(hipGetDevice(&dev));
  GP_REQUIRE(dev == p->device, "grad plan used on another device than its own");
  return GP_OK;
}

struct Span {
  uintptr_t lo, hi;
  size_t i;
};

// Beside one for each gradient's end: 2^40 values, more than the device's memory holds.
constexpr size_t kMostChunks = (size_t)1 << 25;

// Chunk length: a whole number of 16-byte steps of a block, long enough that
// the table stays small, short enough that every block of the grid gets some.
size_t chunk_length(size_t total) {
  size_t c = 2048;
  while (c < 32768 && total / c > 4096) c *= 2;
  return c;
}

int build_grad_plan(gp_grad_plan_s *p, size_t count, const void *const *grads, const int *types, void *const *outs,
                    const int *out_types, const size_t *sizes) {
  std::vector<Span> spans;
  size_t total = 0;
  for (size_t i = 0; i < count; ++i) {
    GP_REQUIRE(type_known(types[i]) && type_known(out_types[i]), "types must be GP_F32, GP_BF16 or GP_F16");
    GP_REQUIRE(out_types[i] == types[i] || out_types[i] == GP_F32,
               "an output has its gradient's type or GP_F32");
    if (sizes[i] == 0) continue;
    GP_REQUIRE(grads[i] && outs[i], "null gradient or output");
    GP_REQUIRE(sizes[i] <= SIZE_MAX / 8, "gradient too long");
    const uintptr_t lo = reinterpret_cast<uintptr_t>(outs[i]);
    spans.push_back({lo, lo + sizes[i] * type_size(out_types[i]), i});
    GP_REQUIRE(total <= SIZE_MAX / 8 - sizes[i], "gradients too long");
    total += sizes[i];
    p->bytes += sizes[i] * type_size(types[i]);
  }
  std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.lo < b.lo; });
  for (size_t k = 1; k < spans.size(); ++k)
    GP_REQUIRE(spans[k - 1].hi <= spans[k].lo, "two outputs overlap (in place: a gradient listed twice)");
  for (size_t i = 0; i < count; ++i) {
    if (sizes[i] == 0) continue;
    const uintptr_t lo = reinterpret_cast<uintptr_t>(grads[i]), hi = lo + sizes[i] * type_size(types[i]);
    auto at = std::upper_bound(spans.begin(), spans.end(), lo,
                               [](uintptr_t v, const Span &s) { return v < s.hi; });
    for (; at != spans.end() && at->lo < hi; ++at)
      GP_REQUIRE(at->i == i && at->lo == lo && types[i] == out_types[i],
                 "an output overlaps a gradient and is not that gradient itself");
  }
  const size_t len = chunk_length(total);
  size_t needed = 0;  // known before the table takes any memory: 32 bytes each
  for (size_t i = 0; i < count; ++i) needed += sizes[i] / len + (sizes[i] % len != 0);
  GP_REQUIRE(needed <= kMostChunks + count && needed <= (size_t)INT32_MAX, "too many values for one plan");
  std::vector<Chunk> chunks;
  chunks.reserve(needed);
  for (size_t i = 0; i < count; ++i)
    for (size_t at = 0; at < sizes[i]; at += len)
      chunks.push_back({static_cast<const char *>(grads[i]) + at * type_size(types[i]),
                        static_cast<char *>(outs[i]) + at * type_size(out_types[i]),
                        (unsigned)std::min(len, sizes[i] - at), (short)types[i], (short)out_types[i]});
  p->count = chunks.size();
  if (chunks.empty()) return GP_OK;
  GP_HIP_TRY(hipGetDevice(&p->device));
  GP_HIP_TRY(hipMalloc(&p->chunks, chunks.size() * sizeof(Chunk)));
  GP_HIP_TRY(hipMemcpy(p->chunks, chunks.data(), chunks.size() * sizeof(Chunk), hipMemcpyHostToDevice));
  return GP_OK;
}

}  // namespace

extern "C" {

int gp_grad_plan_create(gp_grad_plan *plan, size_t count, const void *const *grads, const int *grad_types,
                        void *const *outs, const int *out_types, const size_t *sizes) {
  GP_REQUIRE(plan, "null plan");
  *plan = nullptr;
  GP_REQUIRE(count == 0 || (grads && grad_types && outs && out_types && sizes), "null gradient list");
  gp_grad_plan_s *p = nullptr;
  int rc;
  try {
    p = new gp_grad_plan_s();
    rc = build_grad_plan(p, count, grads, grad_types, outs, out_types, sizes);
  } catch (const std::bad_alloc &) {
    rc = set_error(GP_ERR_INVALID, "out of host memory");
  }
  if (rc != GP_OK) {
    gp_grad_plan_destroy(p);
    return rc;
  }
  *plan = p;
  return GP_OK;
}

int gp_grad_plan_destroy(gp_grad_plan plan) {
  if (!plan) return GP_OK;
  hipError_t e = hipSuccess;
  if (plan->chunks) {
    RelaxedCapture relaxed;
    e = hipFree(plan->chunks);
  }
  delete plan;
  GP_HIP_TRY(e);
  return GP_OK;
}

int gp_grad_sum_squares(gp_grad_plan plan, double *sum, void *workspace, gp_stream s) {
  GP_REQUIRE(sum, "null sum");
  const int rc = check_grad_plan(plan, workspace);
  if (rc != GP_OK) return rc;
  const unsigned grid = clip_grid(plan->count);
  double *partial = static_cast<double *>(workspace);
  launch_grad_square(plan, grid, partial, (hipStream_t)s);
  hipLaunchKernelGGL(sum_partials_kernel, dim3(1), dim3(kClipBlock), 0, (hipStream_t)s, (const double *)partial, grid,
                     sum, (float *)nullptr);
  GP_HIP_TRY(hipGetLastError());
  return GP_OK;
}

int gp_grad_clip(gp_grad_plan plan, double max_norm, double scale, int nonfinite, const double *sum, float *norm,
                 void *workspace, gp_stream s) {
  int rc = check_bound(max_norm, scale, nonfinite);
  if (rc == GP_OK) rc = check_grad_plan(plan, workspace);
  if (rc != GP_OK) return rc;
  const unsigned grid = clip_grid(plan->count);
  double *partial = static_cast<double *>(workspace);
  if (!sum) launch_grad_square(plan, grid, partial, (hipStream_t)s);
  const Bound b{max_norm, scale, nonfinite == GP_CLIP_SKIP};
  hipLaunchKernelGGL(grad_scale_kernel, dim3(grid), dim3(kClipBlock), 0, (hipStream_t)s, (const Chunk *)plan->chunks,
                     (unsigned)plan->count, sum ? sum : (const double *)partial, sum ? 1u : grid, b, norm);
  GP_HIP_TRY(hipGetLastError());
  return GP_OK;
}

int gp_bucket_sum_squares(float *scratch, const float *const *buckets, int num_buckets, size_t num_vals, double *sum,
                          void *workspace, gp_stream s) {
  GP_REQUIRE(sum && workspace, "null sum or workspace");
  int rc = check_buckets(scratch, buckets, num_buckets, num_vals);
  if (rc != GP_OK) return rc;
  unsigned partials = 0;
  double *partial = static_cast<double *>(workspace);
  if (num_buckets && num_vals) {
    rc = launch_squares(scratch, buckets, num_buckets, num_vals, partial, &partials, (hipStream_t)s);
    if (rc != GP_OK) return rc;
  }
  hipLaunchKernelGGL(sum_partials_kernel, dim3(1), dim3(kClipBlock), 0, (hipStream_t)s, (const double *)partial,
                     partials, sum, (float *)nullptr);
  GP_HIP_TRY(hipGetLastError());
  return GP_OK;
}

int gp_bucket_sum_clipped(float *out, const float *in, const float *const *buckets, int num_buckets, size_t num_vals,
                          float *scratch, double max_norm, double scale, int nonfinite, const double *sum,
                          float *norm, void *workspace, gp_stream s) {
  int rc = check_bound(max_norm, scale, nonfinite);
  if (rc == GP_OK) rc = check_buckets(scratch, buckets, num_buckets, num_vals);
  if (rc != GP_OK) return rc;
  GP_REQUIRE(workspace, "null workspace");
  double *partial = static_cast<double *>(workspace);
  if (num_vals) {
    const size_t bytes = num_vals * sizeof(float);
    GP_REQUIRE(out && in, "null out or in");
    GP_REQUIRE(out == in || !bytes_overlap(out, bytes, in, bytes), "out overlaps in and is not in itself");
    for (int k = 0; k < num_buckets; ++k)
      GP_REQUIRE(!bytes_overlap(out, bytes, buckets[k], bytes), "out overlaps a bucket");
    if (num_buckets > kReread)
      GP_REQUIRE(!bytes_overlap(scratch, bytes, out, bytes) && !bytes_overlap(scratch, bytes, in, bytes),
                 "scratch overlaps out or in");
  }
  if (num_buckets == 0 || num_vals == 0) {
    if (num_vals && out != in) {
      rc = gp_bucket_sum_into(out, in, nullptr, 0, num_vals, s);
      if (rc != GP_OK) return rc;
    }
    if (norm) {
      hipLaunchKernelGGL(sum_partials_kernel, dim3(1), dim3(kClipBlock), 0, (hipStream_t)s,
                         sum ? sum : (const double *)partial, sum ? 1u : 0u, (double *)nullptr, norm);
      GP_HIP_TRY(hipGetLastError());
    }
    return GP_OK;
  }
  unsigned partials = 1;
  if (!sum) {
    rc = launch_squares(scratch, buckets, num_buckets, num_vals, partial, &partials, (hipStream_t)s);
    if (rc != GP_OK) return rc;
  }
  const Bound b{max_norm, scale, nonfinite == GP_CLIP_SKIP};
  Streams st = {};
  const bool reread = num_buckets <= kReread;
  st.p[0] = reread ? buckets[0] : scratch;
  if (num_buckets == 2) st.p[1] = buckets[1];
  const dim3 grid(clip_grid((num_vals + kClipBlock * 16 - 1) / (kClipBlock * 16))), block(kClipBlock);
  const double *from = sum ? sum : partial;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, block, 0, (hipStream_t)s, out, in, st, num_vals, from, partials, b, norm);
  };
  if (!reread)
    go(add_scaled_kernel<1, true>);
  else if (num_buckets == 2)
    go(add_scaled_kernel<2, false>);
  else
    go(add_scaled_kernel<1, false>);
  GP_HIP_TRY(hipGetLastError());
  return GP_OK;
}

}  // extern "C"
