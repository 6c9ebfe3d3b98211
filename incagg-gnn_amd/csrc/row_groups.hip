// Rows ordered by the group (node type, expert, partition) each of them belongs to:
//
//     key[i]  = ids[i] in [0, G), or G for a row of no group (id -1)
//     order   = the row numbers by ascending key, equal keys in row order
//     ptr[g]  = number of rows with key < g,  g = 0 .. G
//
// A counting sort with ranks.  Every workgroup owns kChunk consecutive rows, every wave of it a
// quarter of them, eight to a lane, whose keys stay in registers from the count to the ranking.
//   1. count:  keys per workgroup (LDS histogram)             -> table[key][workgroup]
//   2. scan:   one workgroup per key, exclusive over workgroups, and the key's total
//   3. place:  each workgroup scans the totals (where each key begins), adds its own offset, and
//      ranks its rows: a wave takes 64 rows at a time, finds the lanes of equal key with one
//      ballot per key bit, and the lanes before a lane in its set are its rank.
// Nothing depends on the order in which atomics arrive (the counts are sums of integers, the ranks
// come from lane numbers), so the result is the stable one, every time.  Up to kChunk rows are
// one launch: a single workgroup counts, scans and places.
//
// Bound by latency and by the two reads of the ids: 2 449 029 rows of 16 groups take 21 us (bytes at
// 5.1 TB/s: 6 us; count 7.8, scan 2.9, place 6.7), 517 rows of 64 groups 5.6 us in one launch.
// 2048 rows to a workgroup: the table that the scan walks stays small, and 1196 workgroups fill the chip.
#include "common.h"

#include <algorithm>
#include <climits>

namespace incagg {

constexpr int kChunk = 2048;              // rows of a workgroup
constexpr int kMaxGroups = 2048;       // (a counter per wave and key in LDS)
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kWaveRows = kChunk / kWaves, kLaneRows = kWaveRows / 64;

// Key of a row; ids outside [-1, G) are reported and count as rows of no group.
template <typename I> __device__ inline int key_of(I id, int n_groups, int *err) {
  if (id >= 0 && id < (I)n_groups) return (int)id;
  if (id != (I)-1) *err = 1;
  return n_groups;
}

// Keys of this lane's rows: rows begin + 64 j + lane, -1 behind the last.
template <typename I>
__device__ inline void load_keys(const I *ids, int begin, int end, int n_groups, int *err,
                                 int (&key)[kLaneRows]) {
  const int lane = threadIdx.x & 63;
  I id[kLaneRows];
#pragma unroll
  for (int j = 0; j < kLaneRows; j++) id[j] = ids[min(begin + 64 * j + lane, end - 1)];
#pragma unroll
  for (int j = 0; j < kLaneRows; j++)
    key[j] = begin + 64 * j + lane < end ? key_of(id[j], n_groups, err) : -1;
}

template <typename I>
__global__ __launch_bounds__(kThreads) void count_kernel(const I *ids, int rows, int n_groups,
                                                         int n_blocks, int *table, int *err) {
  extern __shared__ int hist[];           // [n_groups + 1]
  const int n_keys = n_groups + 1;
  const int begin = (int)blockIdx.x * kChunk + (int)(threadIdx.x >> 6) * kWaveRows;
  int key[kLaneRows];
  load_keys(ids, begin, rows, n_groups, err, key);
  for (int k = threadIdx.x; k < n_keys; k += kThreads) hist[k] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kLaneRows; j++)
    if (key[j] >= 0) atomicAdd(&hist[key[j]], 1);
  __syncthreads();
  for (int k = threadIdx.x; k < n_keys; k += kThreads)
    table[(long long)k * n_blocks + blockIdx.x] = hist[k];
}

// Exclusive scan over the workgroup of one value per thread; *sum: the total.
__device__ inline int block_exclusive(int v, int *lds, int *sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(s, o);
    if (lane >= o) s += u;
  }
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    const int t = lds[w];
    if (w < wave) before += t;
    all += t;
  }
  __syncthreads();
  *sum = all;
  return before + s - v;
}

__global__ __launch_bounds__(kThreads) void scan_kernel(int *table, int n_blocks, int *totals) {
  __shared__ int lds[kWaves];
  int *row = table + (long long)blockIdx.x * n_blocks;
  int carry = 0;
  for (int first = 0; first < n_blocks; first += kThreads) {
    const int i = first + (int)threadIdx.x;
    const int v = i < n_blocks ? row[i] : 0;
    int sum;
    const int s = block_exclusive(v, lds, &sum);
    if (i < n_blocks) row[i] = carry + s;
    carry += sum;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

template <typename I, bool SINGLE>
__global__ __launch_bounds__(kThreads) void place_kernel(const I *ids, int rows, int n_groups,
                                                         int key_bits, int n_blocks,
                                                         const int *table, const int *totals,
                                                         int *order, int *ptr, int *err) {
  extern __shared__ int next[];           // [kWaves][n_groups + 1], then kWaves of scan space
  const int n_keys = n_groups + 1;
  int *scan_lds = next + kWaves * n_keys;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int begin = (int)blockIdx.x * kChunk + wave * kWaveRows;
  const int end = min(rows, begin + kWaveRows);

  // this wave's keys, counted
  int *mine = next + wave * n_keys;
  int key[kLaneRows];
  if (begin < end) load_keys(ids, begin, end, n_groups, err, key);
  for (int k = threadIdx.x; k < kWaves * n_keys; k += kThreads) next[k] = 0;
  __syncthreads();
  if (begin < end)
#pragma unroll
    for (int j = 0; j < kLaneRows; j++)
      if (key[j] >= 0) atomicAdd(&mine[key[j]], 1);
  __syncthreads();

  // where each key begins, plus the rows of it in front of this workgroup and wave
  int carry = 0;
  for (int first = 0; first < n_keys; first += kThreads) {
    const int k = first + (int)threadIdx.x;
    int count[kWaves], here = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      count[w] = k < n_keys ? next[w * n_keys + k] : 0;
      here += count[w];
    }
    const int all = SINGLE ? here : (k < n_keys ? totals[k] : 0);
    int sum;
    const int start = carry + block_exclusive(all, scan_lds, &sum);
    carry += sum;
    if (k < n_keys) {
      if (blockIdx.x == 0) ptr[k] = start;
      int at = start + (SINGLE ? 0 : table[(long long)k * n_blocks + blockIdx.x]);
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        next[w * n_keys + k] = at;
        at += count[w];
      }
    }
  }
  __syncthreads();

  // 64 rows at a time, in order: rank among the lanes of the same key
  if (begin >= end) return;
  const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
  for (int j = 0; j < kLaneRows; j++) {
    const bool live = key[j] >= 0;
    unsigned long long same = __ballot(live);
    for (int b = 0; b < key_bits; b++) {
      const unsigned long long set = __ballot((key[j] >> b) & 1);
      same &= ((key[j] >> b) & 1) ? set : ~set;
    }
    const bool leader = live && (same & below) == 0;
    if (live) order[mine[key[j]] + __popcll(same & below)] = begin + 64 * j + lane;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (leader) mine[key[j]] += __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// ptr of rows that lie sorted already: a running maximum, clamped to [0, rows], with out[0] = 0.
template <typename I>
__global__ __launch_bounds__(kThreads) void ptr_kernel(const I *in, int n_groups, int rows,
                                                       int *out, int *err) {
  __shared__ int lds[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int carry = 0;
  for (int first = 0; first <= n_groups; first += kThreads) {
    const int k = first + (int)threadIdx.x;
    int v = 0;
    I raw = 0;
    if (k <= n_groups) {
      raw = in[k];
      v = k == 0 || raw < 0 ? 0 : (raw > (I)rows ? rows : (int)raw);
    }
    int s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(s, o);
      if (lane >= o) s = max(s, u);
    }
    if (lane == 63) lds[wave] = s;
    __syncthreads();
    int before = carry, all = carry;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      if (w < wave) before = max(before, lds[w]);
      all = max(all, lds[w]);
    }
    __syncthreads();
    s = max(s, before);
    carry = all;
    if (k <= n_groups) {
      out[k] = s;
      if ((I)s != raw) *err = 1;
    }
  }
}

static int bits_for(int n_keys) {
  int b = 0;
  while ((1 << b) < n_keys) b++;
  return b;
}

template <typename I>
static int group_rows(const I *ids, int rows, int n_groups, int *ws, int *order, int *ptr,
                      hipStream_t s) {
  int *err = nullptr;
  int rc = error_flag_address(&err);
  if (rc) return rc;
  const int n_keys = n_groups + 1, n_blocks = (rows + kChunk - 1) / kChunk;
  const size_t count_lds = sizeof(int) * (size_t)n_keys;
  const size_t place_lds = sizeof(int) * ((size_t)kWaves * n_keys + kWaves);
  const int bits = bits_for(n_keys);
  if (n_blocks <= 1) {
    hipLaunchKernelGGL((place_kernel<I, true>), dim3(1), dim3(kThreads), place_lds, s, ids, rows,
                       n_groups, bits, 1, nullptr, nullptr, order, ptr, err);
    INCAGG_HIP_TRY(hipGetLastError());
    return INCAGG_OK;
  }
  int *table = ws, *totals = ws + (size_t)n_keys * n_blocks;
  hipLaunchKernelGGL(count_kernel<I>, dim3(n_blocks), dim3(kThreads), count_lds, s, ids, rows,
                     n_groups, n_blocks, table, err);
  INCAGG_HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL(scan_kernel, dim3(n_keys), dim3(kThreads), 0, s, table, n_blocks, totals);
  INCAGG_HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL((place_kernel<I, false>), dim3(n_blocks), dim3(kThreads), place_lds, s, ids,
                     rows, n_groups, bits, n_blocks, table, totals, order, ptr, err);
  INCAGG_HIP_TRY(hipGetLastError());
  return INCAGG_OK;
}

}  // namespace incagg

using namespace incagg;

extern "C" int64_t incagg_group_rows_max_groups(void) { return kMaxGroups; }

extern "C" int64_t incagg_group_rows_ws_ints(int64_t rows, int64_t n_groups) {
  if (rows < 0 || n_groups < 1 || n_groups > kMaxGroups || rows > INT_MAX - kChunk)
    return fail(INCAGG_E_INVALID, "size out of range");
  const int64_t n_blocks = (rows + kChunk - 1) / kChunk;
  return n_blocks <= 1 ? 0 : (n_groups + 1) * (n_blocks + 1);
}

extern "C" int incagg_group_rows(const void *ids, int ids_are_64, int64_t rows, int64_t n_groups,
                                 int32_t *ws, int64_t ws_ints, int32_t *order, int32_t *ptr,
                                 void *stream) {
  INCAGG_REQUIRE(rows >= 0 && rows <= INT_MAX - kChunk, "rows %lld out of range", (long long)rows);
  INCAGG_REQUIRE(n_groups >= 1 && n_groups <= kMaxGroups, "n_groups %lld out of range [1, %d]",
                 (long long)n_groups, kMaxGroups);
  INCAGG_REQUIRE(ptr && (rows == 0 || (ids && order)), "null pointer");
  const int64_t need = incagg_group_rows_ws_ints(rows, n_groups);
  INCAGG_REQUIRE(need == 0 || (ws && ws_ints >= need), "workspace too small: %lld < %lld",
                 (long long)ws_ints, (long long)need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return ids_are_64 ? group_rows(static_cast<const long long *>(ids), (int)rows, (int)n_groups, ws,
                                 order, ptr, s)
                    : group_rows(static_cast<const int *>(ids), (int)rows, (int)n_groups, ws, order,
                                 ptr, s);
}

extern "C" int incagg_group_ptr(const void *in, int in_is_64, int64_t n_groups, int64_t rows,
                                int32_t *out, void *stream) {
  INCAGG_REQUIRE(rows >= 0 && rows <= INT_MAX - kChunk, "rows %lld out of range", (long long)rows);
  INCAGG_REQUIRE(n_groups >= 1 && n_groups <= kMaxGroups, "n_groups %lld out of range [1, %d]",
                 (long long)n_groups, kMaxGroups);
  INCAGG_REQUIRE(in && out, "null pointer");
  int *err = nullptr;
  int rc = error_flag_address(&err);
  if (rc) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (in_is_64)
    hipLaunchKernelGGL(ptr_kernel<long long>, dim3(1), dim3(kThreads), 0, s,
                       static_cast<const long long *>(in), (int)n_groups, (int)rows, out, err);
  else
    hipLaunchKernelGGL(ptr_kernel<int>, dim3(1), dim3(kThreads), 0, s, static_cast<const int *>(in),
                       (int)n_groups, (int)rows, out, err);
  INCAGG_HIP_TRY(hipGetLastError());
  return INCAGG_OK;
}
