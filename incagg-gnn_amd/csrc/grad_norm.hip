// Global norm of the gradients of many tensors, clipping by it, and an Adam step that clips as it
// reads (main.py:81-85: loss.backward(), clip_grad_norm_, optimizer.step()).
//
//     total = (sum_t sum_i |x_t[i]|^p)^(1/p)   (p = 1, 2; max |x| for p = inf)
//     coef  = min(1, max_norm / (total + 1e-6))
//     clip:  x_t[i] *= coef            Adam:  g' = coef g + wd p, then torch.optim.Adam's update
//
// Two launches each (more for more than 128 tensors, 64 in Adam's second).  The first sums: every
// workgroup walks units of 8192 consecutive elements of ONE tensor and leaves one partial in the
// caller's workspace.  The second clips (or updates), and every one of its workgroups first adds up
// all partials by itself, in a fixed order: at most 1024 doubles from the L2 for 128 tensors, a
// microsecond, where a finishing launch would cost several and a last-arriver counter would be state
// that two recorded graphs share.  Same order everywhere and every time: the same bits.
//
// Numerics: sums and the total are held in 64 bits, so neither the square of a large float32
// value nor the sum of 10^9 small ones loses anything (the float64 pipes keep up: a multiply-add
// per element against 2 or 4 bytes of memory traffic).  coef is rounded to float32 once; a scaled
// value is rounded once, to its own type.
//
// Bound by memory once there is enough of it: the norm of 200 M bfloat16 elements (400 MB) in one
// tensor takes 72 us (5.5 TB/s), of 100 M float32 ones 70 us.  In 300 tensors it takes 87 us (4.6 TB/s):
// three launches, the next of which starts when the last workgroup of the one before has ended.
// Clipping those 300 (nearly all bfloat16, some short float32) takes 265 us where they are scaled (1.2
// GB, 4.5 TB/s) and 110 us where they are not: three more launches, which add up the partials and end.
// Adam with clipping over 64 M parameters 412 us (28 bytes each at 5.1 TB/s: 351 us, and the norm in
// front of it).  Small ones are two launches: 10 tensors of 110 k elements 11-13 us, Adam over 20
// tensors of 1.1 M 14.5-17 us, most of both on the host.
#include "common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <cmath>
#include <vector>

namespace incagg {

constexpr int kNormThreads = 512;
constexpr int kUnit = 8192;               // elements of a unit of work
constexpr int kMaxPartials = 1024;        // partials of one launch
// Tensors of one launch: the table travels as a kernel argument, whose size is limited to 4 KB.
constexpr int kNormSegments = 128;
constexpr int kUpdateSegments = 64;
constexpr int kHyperGroups = 8;

struct NormTable {
  void *x[kNormSegments];
  float *step[kNormSegments];             // advanced by one when not NULL
  long long n[kNormSegments];
  int first_unit[kNormSegments + 1];
  unsigned char dtype[kNormSegments];
  int n_segs;
};
static_assert(sizeof(NormTable) <= 3900, "kernel argument limit");

// Vectors that may start at any multiple of their element's size (global memory takes unaligned
// 16-byte accesses; parameters cut from a flat buffer start anywhere).
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[N]; };

struct Bf16 {
  unsigned short bits;
  __device__ float get() const { return __uint_as_float((unsigned)bits << 16); }
  __device__ void set(float f) {
    const __hip_bfloat16 h = __float2bfloat16(f);   // nearest even
    bits = *reinterpret_cast<const unsigned short *>(&h);
  }
};
struct F16 {
  _Float16 h;
  __device__ float get() const { return (float)h; }
  __device__ void set(float f) { h = (_Float16)f; }
};
struct F32 {
  float f;
  __device__ float get() const { return f; }
  __device__ void set(float v) { f = v; }
};

template <int P> __device__ inline void norm_add(double &acc, float x) {
  if constexpr (P == 2) {
    acc = fma((double)x, (double)x, acc);
  } else if constexpr (P == 1) {
    acc += fabs((double)x);
  } else {
    const double a = fabs((double)x);
    acc = (a > acc || a != a) ? a : acc;     // a NaN stays
  }
}
template <int P> __device__ inline double norm_join(double a, double b) {
  if constexpr (P == 0) return (b > a || b != b) ? b : a;
  return a + b;
}

// Sum (or maximum) over the workgroup in a fixed order; the result in every thread.
template <int P, int THREADS> __device__ double block_join(double v, double *lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = norm_join<P>(v, __shfl_down(v, o));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = lds[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; w++) s = norm_join<P>(s, lds[w]);
  return s;
}

template <int P, typename T> __device__ double unit_norm(const T *x, long long begin, int count) {
  constexpr int V = 16 / sizeof(T), STEP = kNormThreads * V;
  const T *p = x + begin;
  double acc = 0.0;
  if (count == kUnit) {
    Pack<T, V> q[kUnit / STEP];
#pragma unroll
    for (int i = 0; i < kUnit / STEP; i++)
      q[i] = *reinterpret_cast<const Pack<T, V> *>(p + i * STEP + (int)threadIdx.x * V);
#pragma unroll
    for (int i = 0; i < kUnit / STEP; i++)
#pragma unroll
      for (int j = 0; j < V; j++) norm_add<P>(acc, q[i].v[j].get());
  } else {
    for (int i = (int)threadIdx.x * V; i < count; i += STEP) {
      if (i + V <= count) {
        const Pack<T, V> q = *reinterpret_cast<const Pack<T, V> *>(p + i);
#pragma unroll
        for (int j = 0; j < V; j++) norm_add<P>(acc, q.v[j].get());
      } else {
        for (int j = i; j < count; j++) norm_add<P>(acc, p[j].get());
      }
    }
  }
  return acc;
}

template <int P>
__global__ __launch_bounds__(kNormThreads) void norm_partials_kernel(const NormTable t,
                                                                     double *partials) {
  __shared__ double lds[kNormThreads / 64];
  const int n_units = t.first_unit[t.n_segs];
  double acc = 0.0;
  int seg = 0;
  for (int u = blockIdx.x; u < n_units; u += gridDim.x) {
    while (u >= t.first_unit[seg + 1]) seg++;
    const long long begin = (long long)(u - t.first_unit[seg]) * kUnit;
    const int count = (int)min((long long)kUnit, t.n[seg] - begin);
    double a;
    if (t.dtype[seg] == INCAGG_DTYPE_F32)
      a = unit_norm<P>(static_cast<const F32 *>(t.x[seg]), begin, count);
    else if (t.dtype[seg] == INCAGG_DTYPE_BF16)
      a = unit_norm<P>(static_cast<const Bf16 *>(t.x[seg]), begin, count);
    else
      a = unit_norm<P>(static_cast<const F16 *>(t.x[seg]), begin, count);
    acc = norm_join<P>(acc, a);
  }
  const double s = block_join<P, kNormThreads>(acc, lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
  if (blockIdx.x == 0)
    for (int k = threadIdx.x; k < t.n_segs; k += kNormThreads)
      if (t.step[k]) *t.step[k] += 1.f;
}

template <int P, int THREADS>
__device__ double total_norm(const double *partials, int n_partials, double *lds) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n_partials; i += THREADS) s = norm_join<P>(s, partials[i]);
  s = block_join<P, THREADS>(s, lds);
  return P == 2 ? sqrt(s) : s;
}

// torch.nn.utils.clip_grad_norm_'s coefficient; a NaN total gives NaN.
__device__ inline float clip_coefficient(double total, double max_norm) {
  const double c = max_norm / (total + 1e-6);
  return (float)(c > 1.0 ? 1.0 : c);
}

template <int P>
__global__ __launch_bounds__(256) void norm_finish_kernel(const double *partials, int n_partials,
                                                          float *norm) {
  __shared__ double lds[4];
  const double s = total_norm<P, 256>(partials, n_partials, lds);
  if (threadIdx.x == 0) *norm = (float)s;
}

template <typename T> __device__ void unit_scale(T *x, long long begin, int count, float coef) {
  constexpr int V = 16 / sizeof(T), STEP = kNormThreads * V;
  T *p = x + begin;
  if (count == kUnit) {
    Pack<T, V> q[kUnit / STEP];
#pragma unroll
    for (int i = 0; i < kUnit / STEP; i++)
      q[i] = *reinterpret_cast<const Pack<T, V> *>(p + i * STEP + (int)threadIdx.x * V);
#pragma unroll
    for (int i = 0; i < kUnit / STEP; i++) {
#pragma unroll
      for (int j = 0; j < V; j++) q[i].v[j].set(q[i].v[j].get() * coef);
      *reinterpret_cast<Pack<T, V> *>(p + i * STEP + (int)threadIdx.x * V) = q[i];
    }
  } else {
    for (int i = (int)threadIdx.x * V; i < count; i += STEP) {
      if (i + V <= count) {
        Pack<T, V> q = *reinterpret_cast<const Pack<T, V> *>(p + i);
#pragma unroll
        for (int j = 0; j < V; j++) q.v[j].set(q.v[j].get() * coef);
        *reinterpret_cast<Pack<T, V> *>(p + i) = q;
      } else {
        for (int j = i; j < count; j++) p[j].set(p[j].get() * coef);
      }
    }
  }
}

template <int P>
__global__ __launch_bounds__(kNormThreads) void clip_kernel(const NormTable t,
                                                            const double *partials, int n_partials,
                                                            double max_norm, float *norm) {
  __shared__ double lds[kNormThreads / 64];
  const double total = total_norm<P, kNormThreads>(partials, n_partials, lds);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  const float coef = clip_coefficient(total, max_norm);
  if (coef == 1.f) return;                 // nothing to scale: nothing is read or written
  const int n_units = t.first_unit[t.n_segs];
  int seg = 0;
  for (int u = blockIdx.x; u < n_units; u += gridDim.x) {
    while (u >= t.first_unit[seg + 1]) seg++;
    const long long begin = (long long)(u - t.first_unit[seg]) * kUnit;
    const int count = (int)min((long long)kUnit, t.n[seg] - begin);
    if (t.dtype[seg] == INCAGG_DTYPE_F32)
      unit_scale(static_cast<F32 *>(t.x[seg]), begin, count, coef);
    else if (t.dtype[seg] == INCAGG_DTYPE_BF16)
      unit_scale(static_cast<Bf16 *>(t.x[seg]), begin, count, coef);
    else
      unit_scale(static_cast<F16 *>(t.x[seg]), begin, count, coef);
  }
}

// ---- Adam with clipped gradients -----------------------------------------------------------
struct UpdateTable {
  float *p[kUpdateSegments];
  const float *g[kUpdateSegments];
  float *m[kUpdateSegments];
  float *v[kUpdateSegments];
  const float *step[kUpdateSegments];     // already advanced by the launch in front
  long long n[kUpdateSegments];
  int first_block[kUpdateSegments + 1];
  unsigned char hyper[kUpdateSegments];
  double lr[kHyperGroups], b1[kHyperGroups], b2[kHyperGroups], eps[kHyperGroups], wd[kHyperGroups];
  int n_segs;
};
static_assert(sizeof(UpdateTable) <= 3900, "kernel argument limit");

// A workgroup updates PER_BLOCK consecutive elements of ONE tensor: 28 bytes of traffic for each.
// The loads of its first elements are in flight while the total is added up and the bias
// corrections 1 - beta^t are evaluated (in 64 bits: 1 - 0.999f^t in 32 bits is off by 3e-5).
template <int PER_BLOCK>
__global__ __launch_bounds__(256) void adam_clip_kernel(const UpdateTable t, const double *partials,
                                                        int n_partials, double max_norm,
                                                        float *norm) {
  __shared__ double lds[4];
  __shared__ float scalars[2];
  typedef Pack<float, 4> f4;
  int seg = 0;
  while ((int)blockIdx.x >= t.first_block[seg + 1]) seg++;     // scalar
  const long long begin = (long long)((int)blockIdx.x - t.first_block[seg]) * PER_BLOCK;
  const int count = (int)min((long long)PER_BLOCK, t.n[seg] - begin);
  float *p = t.p[seg] + begin, *m = t.m[seg] + begin, *v = t.v[seg] + begin;
  const float *g = t.g[seg] + begin;
  const int h = t.hyper[seg];

  constexpr int ROUNDS = PER_BLOCK / 1024;
  f4 pp[ROUNDS], gg[ROUNDS], mm[ROUNDS], vv[ROUNDS];
  const bool whole = count == PER_BLOCK;
  if (whole) {
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
      const int at = i * 1024 + (int)threadIdx.x * 4;
      gg[i] = *reinterpret_cast<const f4 *>(g + at);
      pp[i] = *reinterpret_cast<const f4 *>(p + at);
      mm[i] = *reinterpret_cast<const f4 *>(m + at);
      vv[i] = *reinterpret_cast<const f4 *>(v + at);
    }
  }
  if (threadIdx.x == 64) {
    const double steps = *t.step[seg];
    scalars[0] = (float)(t.lr[h] / (1.0 - pow(t.b1[h], steps)));
    scalars[1] = (float)sqrt(1.0 - pow(t.b2[h], steps));
  }
  const double total = total_norm<2, 256>(partials, n_partials, lds);   // (contains the barrier)
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  const float coef = clip_coefficient(total, max_norm);
  const float step_size = scalars[0], bc2_sqrt = scalars[1];
  const float c1 = (float)(1.0 - t.b1[h]), b2 = (float)t.b2[h], c2 = (float)(1.0 - t.b2[h]);
  const float wd = (float)t.wd[h], eps = (float)t.eps[h];
  auto one = [&](float &pe, float ge, float &me, float &ve) {
    ge = ge * coef + wd * pe;
    me += (ge - me) * c1;
    ve = ve * b2 + c2 * ge * ge;
    pe -= step_size * me / (sqrtf(ve) / bc2_sqrt + eps);
  };
  if (whole) {
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
      const int at = i * 1024 + (int)threadIdx.x * 4;
#pragma unroll
      for (int j = 0; j < 4; j++) one(pp[i].v[j], gg[i].v[j], mm[i].v[j], vv[i].v[j]);
      *reinterpret_cast<f4 *>(p + at) = pp[i];
      *reinterpret_cast<f4 *>(m + at) = mm[i];
      *reinterpret_cast<f4 *>(v + at) = vv[i];
    }
  } else {
    for (int at = threadIdx.x; at < count; at += 256) {
      float pe = p[at], me = m[at], ve = v[at];
      one(pe, g[at], me, ve);
      p[at] = pe;
      m[at] = me;
      v[at] = ve;
    }
  }
}

// ---- host side -----------------------------------------------------------------------------
// Segments of the list that launch number i takes, and how many partials it leaves.
static int element_size(int dtype) { return dtype == INCAGG_DTYPE_F32 ? 4 : 2; }

struct NormLaunch {
  NormTable table;
  int blocks;
};

// Splits the list into launches; empty tensors are dropped.
static int plan_norm(const incagg_norm_segment *segs, int64_t n_segs, std::vector<NormLaunch> &out,
                     int64_t *n_partials) {
  int64_t i = 0;
  *n_partials = 0;
  while (i < n_segs) {
    out.emplace_back();
    NormLaunch &l = out.back();
    l.table = NormTable{};
    int k = 0;
    int64_t units = 0;
    for (; i < n_segs && k < kNormSegments; i++) {
      const incagg_norm_segment &s = segs[i];
      INCAGG_REQUIRE(s.n >= 0 && s.n < (1ll << 40), "segment length %lld out of range",
                     (long long)s.n);
      if (s.n == 0) continue;
      INCAGG_REQUIRE(s.x, "null segment pointer");
      INCAGG_REQUIRE(s.dtype == INCAGG_DTYPE_F32 || s.dtype == INCAGG_DTYPE_BF16 ||
                         s.dtype == INCAGG_DTYPE_F16, "unknown element type %lld",
                     (long long)s.dtype);
      INCAGG_REQUIRE(reinterpret_cast<uintptr_t>(s.x) % element_size((int)s.dtype) == 0,
                     "segment not aligned to its element type");
      const int64_t u = (s.n + kUnit - 1) / kUnit;
      INCAGG_REQUIRE(units + u < (1ll << 30), "too many elements for one call");
      l.table.x[k] = s.x;
      l.table.step[k] = nullptr;
      l.table.n[k] = s.n;
      l.table.dtype[k] = (unsigned char)s.dtype;
      l.table.first_unit[k] = (int)units;
      units += u;
      k++;
    }
    l.table.first_unit[k] = (int)units;
    l.table.n_segs = k;
    l.blocks = (int)std::min<int64_t>(units, kMaxPartials);
    if (k == 0) out.pop_back();
    else *n_partials += l.blocks;
  }
  return INCAGG_OK;
}

template <int P>
static int launch_partials(const std::vector<NormLaunch> &launches, double *ws, hipStream_t s) {
  for (const NormLaunch &l : launches) {
    hipLaunchKernelGGL(norm_partials_kernel<P>, dim3((unsigned)l.blocks), dim3(kNormThreads), 0, s,
                       l.table, ws);
    INCAGG_HIP_TRY(hipGetLastError());
    ws += l.blocks;
  }
  return INCAGG_OK;
}

template <int P>
static int run_norm(const std::vector<NormLaunch> &launches, int n_partials, bool clip,
                    double max_norm, double *ws, float *norm, hipStream_t s) {
  int rc = launch_partials<P>(launches, ws, s);
  if (rc) return rc;
  if (!clip || launches.empty()) {
    hipLaunchKernelGGL(norm_finish_kernel<P>, dim3(1), dim3(256), 0, s, ws, n_partials, norm);
    INCAGG_HIP_TRY(hipGetLastError());
    return INCAGG_OK;
  }
  for (size_t i = 0; i < launches.size(); i++) {
    const NormLaunch &l = launches[i];
    const unsigned blocks = (unsigned)std::min(l.table.first_unit[l.table.n_segs], 4096);
    hipLaunchKernelGGL(clip_kernel<P>, dim3(blocks), dim3(kNormThreads), 0, s, l.table, ws,
                       n_partials, max_norm, i == 0 ? norm : nullptr);
    INCAGG_HIP_TRY(hipGetLastError());
  }
  return INCAGG_OK;
}

// Whether two of the byte ranges meet (both would be scaled by workgroups that race).
static bool ranges_overlap(std::vector<std::pair<uintptr_t, uintptr_t>> &r) {
  std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); i++)
    if (r[i].first < r[i - 1].second) return true;
  return false;
}

static int grad_norm_call(const incagg_norm_segment *segs, int64_t n_segs, int norm_type, bool clip,
                          double max_norm, double *ws, int64_t ws_doubles, float *norm,
                          void *stream) {
  INCAGG_REQUIRE(n_segs >= 0 && (n_segs == 0 || segs), "bad segment list");
  INCAGG_REQUIRE(norm_type == 0 || norm_type == 1 || norm_type == 2,
                 "norm type must be 1, 2 or 0 (maximum)");
  INCAGG_REQUIRE(norm, "null output");
  std::vector<NormLaunch> launches;
  int64_t n_partials = 0;
  int rc = plan_norm(segs, n_segs, launches, &n_partials);
  if (rc) return rc;
  INCAGG_REQUIRE(n_partials == 0 || (ws && ws_doubles >= n_partials),
                 "workspace too small: %lld < %lld", (long long)ws_doubles, (long long)n_partials);
  if (clip) {
    INCAGG_REQUIRE(max_norm >= 0.0, "max_norm must not be negative or NaN");
    std::vector<std::pair<uintptr_t, uintptr_t>> r;
    for (int64_t i = 0; i < n_segs; i++)
      if (segs[i].n > 0)
        r.emplace_back(reinterpret_cast<uintptr_t>(segs[i].x),
                       reinterpret_cast<uintptr_t>(segs[i].x) +
                           (uintptr_t)segs[i].n * element_size((int)segs[i].dtype));
    INCAGG_REQUIRE(!ranges_overlap(r), "two gradients overlap in memory");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (norm_type == 2) return run_norm<2>(launches, (int)n_partials, clip, max_norm, ws, norm, s);
  if (norm_type == 1) return run_norm<1>(launches, (int)n_partials, clip, max_norm, ws, norm, s);
  return run_norm<0>(launches, (int)n_partials, clip, max_norm, ws, norm, s);
}

// A C entry lets no C++ exception out.
template <typename F> static int guarded(F &&f) {
  try {
    return f();
  } catch (const std::exception &e) {
    return fail(INCAGG_E_NOMEM, "host allocation failed: %s", e.what());
  }
}

}  // namespace incagg

using namespace incagg;

extern "C" int64_t incagg_grad_norm_ws_doubles(int64_t n_segs, int64_t n_elements) {
  if (n_segs < 0 || n_elements < 0) return fail(INCAGG_E_INVALID, "negative size");
  // every launch takes 128 tensors (fewer non-empty ones need no more partials); its units are
  // at most its elements / kUnit + its tensors
  const int64_t launches = (n_segs + kNormSegments - 1) / kNormSegments;
  return std::min(launches * kMaxPartials, n_elements / kUnit + n_segs);
}

extern "C" int incagg_grad_norm(const incagg_norm_segment *segs, int64_t n_segs, int norm_type,
                                double *ws, int64_t ws_doubles, float *norm, void *stream) {
  return guarded([&] {
    return grad_norm_call(segs, n_segs, norm_type, false, 0.0, ws, ws_doubles, norm, stream);
  });
}

extern "C" int incagg_grad_clip(const incagg_norm_segment *segs, int64_t n_segs, int norm_type,
                                double max_norm, double *ws, int64_t ws_doubles, float *norm,
                                void *stream) {
  return guarded([&] {
    return grad_norm_call(segs, n_segs, norm_type, true, max_norm, ws, ws_doubles, norm, stream);
  });
}

static int adam_clip_call(const incagg_adam_clip_segment *segs, int64_t n_segs,
                          const incagg_adam_hyper *hyper, int64_t n_hyper, double max_norm,
                          double *ws, int64_t ws_doubles, float *norm, void *stream) {
  INCAGG_REQUIRE(n_segs >= 0 && (n_segs == 0 || segs), "bad segment list");
  INCAGG_REQUIRE(n_hyper >= 1 && hyper, "bad list of hyperparameters");
  INCAGG_REQUIRE(max_norm >= 0.0, "max_norm must not be negative or NaN");
  INCAGG_REQUIRE(norm, "null output");
  hipStream_t s = static_cast<hipStream_t>(stream);
  std::vector<incagg_norm_segment> grads;
  std::vector<const incagg_adam_clip_segment *> live;
  std::vector<std::pair<uintptr_t, uintptr_t>> written;
  for (int64_t i = 0; i < n_segs; i++) {
    const incagg_adam_clip_segment &a = segs[i];
    INCAGG_REQUIRE(a.n >= 0 && a.n < (1ll << 40), "segment length %lld out of range",
                   (long long)a.n);
    INCAGG_REQUIRE(a.hyper >= 0 && a.hyper < n_hyper, "segment names hyperparameters %lld of %lld",
                   (long long)a.hyper, (long long)n_hyper);
    if (a.n == 0) continue;
    INCAGG_REQUIRE(a.p && a.g && a.m && a.v && a.step, "null segment pointer");
    grads.push_back({const_cast<float *>(a.g), a.n, INCAGG_DTYPE_F32});
    live.push_back(&a);
    for (const float *q : {a.p, a.m, a.v}) {
      const uintptr_t b = reinterpret_cast<uintptr_t>(q);
      INCAGG_REQUIRE(b % 4 == 0, "segment not aligned to its element type");
      written.emplace_back(b, b + (uintptr_t)a.n * 4);
    }
    const uintptr_t b = reinterpret_cast<uintptr_t>(a.step);
    written.emplace_back(b, b + 4);
  }
  INCAGG_REQUIRE(!ranges_overlap(written),
                 "parameters, moments or step counts overlap in memory (a parameter listed twice?)");
  std::vector<NormLaunch> launches;
  int64_t n_partials = 0;
  int rc = plan_norm(grads.data(), (int64_t)grads.size(), launches, &n_partials);
  if (rc) return rc;
  INCAGG_REQUIRE(n_partials == 0 || (ws && ws_doubles >= n_partials),
                 "workspace too small: %lld < %lld", (long long)ws_doubles, (long long)n_partials);
  if (live.empty()) return run_norm<2>(launches, 0, false, 0.0, ws, norm, s);
  size_t at = 0;
  for (NormLaunch &l : launches)
    for (int k = 0; k < l.table.n_segs; k++) l.table.step[k] = live[at++]->step;

  // the update launches are laid out before the first launch, so that a refusal comes first
  int64_t total = 0;
  for (const auto *a : live) total += a->n;
  // Small models: many small workgroups (1 M parameters: 1065 instead of 270).  Large ones: fewer
  // repeat the sum over the partials and the powers.
  const int per_block = total < (8ll << 20) ? 1024 : 4096;
  std::vector<UpdateTable> tables;
  for (size_t i = 0; i < live.size();) {
    tables.emplace_back();
    UpdateTable &t = tables.back();
    t = UpdateTable{};
    int64_t blocks = 0;
    int k = 0, n_groups = 0;
    int64_t groups[kHyperGroups];
    for (; i < live.size() && k < kUpdateSegments; i++, k++) {
      const incagg_adam_clip_segment &a = *live[i];
      int h = 0;
      while (h < n_groups && groups[h] != a.hyper) h++;
      if (h == n_groups) {
        if (n_groups == kHyperGroups) break;
        const incagg_adam_hyper &y = hyper[a.hyper];
        groups[n_groups++] = a.hyper;
        t.lr[h] = y.lr; t.b1[h] = y.beta1; t.b2[h] = y.beta2; t.eps[h] = y.eps;
        t.wd[h] = y.weight_decay;
      }
      t.p[k] = a.p; t.g[k] = a.g; t.m[k] = a.m; t.v[k] = a.v; t.step[k] = a.step;
      t.n[k] = a.n;
      t.hyper[k] = (unsigned char)h;
      t.first_block[k] = (int)blocks;
      blocks += (a.n + per_block - 1) / per_block;
      INCAGG_REQUIRE(blocks < (1ll << 24), "grid too large");      // (2^32 threads a launch)
    }
    t.first_block[k] = (int)blocks;
    t.n_segs = k;
  }
  rc = launch_partials<2>(launches, ws, s);
  if (rc) return rc;
  for (size_t i = 0; i < tables.size(); i++) {
    const UpdateTable &t = tables[i];
    const dim3 grid((unsigned)t.first_block[t.n_segs]), block(256);
    float *out = i == 0 ? norm : nullptr;
    if (per_block == 1024)
      hipLaunchKernelGGL(adam_clip_kernel<1024>, grid, block, 0, s, t, ws, (int)n_partials, max_norm,
                         out);
    else
      hipLaunchKernelGGL(adam_clip_kernel<4096>, grid, block, 0, s, t, ws, (int)n_partials, max_norm,
                         out);
    INCAGG_HIP_TRY(hipGetLastError());
  }
  return INCAGG_OK;
}

extern "C" int incagg_adam_step_clipped_f32(const incagg_adam_clip_segment *segs, int64_t n_segs,
                                            const incagg_adam_hyper *hyper, int64_t n_hyper,
                                            double max_norm, double *ws, int64_t ws_doubles,
                                            float *norm, void *stream) {
  return guarded([&] {
    return adam_clip_call(segs, n_segs, hyper, n_hyper, max_norm, ws, ws_doubles, norm, stream);
  });
}
