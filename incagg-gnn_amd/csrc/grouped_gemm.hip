// Products of rows with the weight matrix of the group each row belongs to.  Rows of group g are
// order[ptr[g] .. ptr[g+1]) (order NULL: they lie sorted already):
//
//     rows:     Y[i] = X[i] @ W_g + b_g      W: [G, K, N], or W_g^T: [G, N, K]   (forward, dX)
//     weights:  D_g = sum_i A[i]^T B[i]      D: [G, M, N], and the column sums of A  (dW, db)
//
// Rows of no group (order[ptr[G] ..]) give zeros.  The group sizes stay on the device: the grid
// is made for the worst case, rows / TILE + G + 1 row tiles, and every workgroup finds its tile
// from ptr.  Slot s belongs to the last g with ptr[g] / TILE + g <= s: a group has at most
// ptr[g+1] / TILE - ptr[g] / TILE + 1 tiles, so every tile gets a slot of its own and at most
// G + 1 slots stay empty.
//
// Sums are held in float32; results are rounded once, to the type of the operands.
#include "common.h"

#include <hip/hip_bf16.h>

#include <algorithm>
#include <climits>

namespace incagg {

struct GroupedArgs {
  const void *x, *w, *bias;
  void *y;
  long long ldx, ldw, w_group, ld_bias, ldy;
  const int *ptr, *order;
  int n_groups, rows, k, n;
  int *err;
};

struct TnArgs {
  const void *a, *b;
  void *d, *sums;
  long long lda, ldb, d_group;
  const int *ptr, *order;
  int n_groups, rows, m, n;
  int *err;
};

template <typename T> __device__ inline float to_float(T v);
template <> __device__ inline float to_float(float v) { return v; }
template <> __device__ inline float to_float(__hip_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ inline float to_float(_Float16 v) { return (float)v; }
template <typename T> __device__ inline T from_float(float v);
template <> __device__ inline float from_float(float v) { return v; }
template <> __device__ inline __hip_bfloat16 from_float(float v) { return __float2bfloat16(v); }
template <> __device__ inline _Float16 from_float(float v) { return (_Float16)v; }

// First row of group g; entries that are out of order or range never lead outside [0, rows].
__device__ inline int group_begin(const int *ptr, int g, int rows) {
  return g == 0 ? 0 : min(max(ptr[g], 0), rows);
}

// The row tile of a slot: false if the slot is empty.  g == n_groups: rows of no group.
template <int TILE, int THREADS>
__device__ inline bool tile_of_slot(const int *ptr, int n_groups, int rows, int slot, int *g,
                                    int *first, int *end) {
  int before = 0;
  for (int base = 1; base <= n_groups; base += THREADS) {
    const int j = base + (int)threadIdx.x;
    before += __syncthreads_count(j <= n_groups && group_begin(ptr, j, rows) / TILE + j <= slot);
  }
  const int p0 = group_begin(ptr, before, rows);
  const int tile = slot - (p0 / TILE + before);
  *g = before;
  *first = p0 + tile * TILE;
  *end = before == n_groups ? rows : group_begin(ptr, before + 1, rows);
  return tile >= 0 && *first < *end;
}

constexpr int kTile = 64, kDepth = 16, kTilePitch = kTile + 4;

// One workgroup: 64 rows x 64 columns of Y, 4 x 4 per thread.
template <typename T, bool TRANS_W>
__global__ __launch_bounds__(256) void grouped_rows_kernel(const GroupedArgs a) {
  __shared__ float xs[kDepth][kTilePitch], ws[kDepth][kTilePitch];
  __shared__ int row_ids[kTile];
  int g, first, end;
  if (!tile_of_slot<kTile, 256>(a.ptr, a.n_groups, a.rows, blockIdx.x, &g, &first, &end)) return;
  const int col0 = (int)blockIdx.y * kTile, tid = threadIdx.x;
  T *y = static_cast<T *>(a.y);
  if (tid < kTile) {
    const int r = first + tid;
    int id = -1;
    if (r < end) {
      id = a.order ? a.order[r] : r;
      if ((unsigned)id >= (unsigned)a.rows) {
        *a.err = 1;
        id = -1;
      }
    }
    row_ids[tid] = id;
  }
  __syncthreads();
  float acc[4][4] = {};
  const int ty = tid >> 4, tx = tid & 15;
  if (g < a.n_groups) {
    const T *x = static_cast<const T *>(a.x);
    const T *w = static_cast<const T *>(a.w) + (long long)g * a.w_group;
    for (int k0 = 0; k0 < a.k; k0 += kDepth) {
      for (int e = tid; e < kTile * kDepth; e += 256) {
        const int r = e / kDepth, kk = e % kDepth, id = row_ids[r];
        xs[kk][r] = id >= 0 && k0 + kk < a.k ? to_float(x[(long long)id * a.ldx + k0 + kk]) : 0.f;
        const int c = TRANS_W ? e / kDepth : e % kTile, kw = TRANS_W ? e % kDepth : e / kTile;
        const bool in = col0 + c < a.n && k0 + kw < a.k;
        const long long at = TRANS_W ? (long long)(col0 + c) * a.ldw + k0 + kw
                                     : (long long)(k0 + kw) * a.ldw + col0 + c;
        ws[kw][c] = in ? to_float(w[at]) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < kDepth; kk++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            acc[i][j] = fmaf(xs[kk][ty * 4 + i], ws[kk][tx * 4 + j], acc[i][j]);
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int id = row_ids[ty * 4 + i];
    if (id < 0) continue;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int c = col0 + tx * 4 + j;
      if (c >= a.n) continue;
      float v = acc[i][j];
      if (a.bias && g < a.n_groups)
        v += to_float(static_cast<const T *>(a.bias)[(long long)g * a.ld_bias + c]);
      y[(long long)id * a.ldy + c] = from_float<T>(v);
    }
  }
}

// One workgroup: 64 x 64 of D_g, over all rows of the group.
template <typename T> __global__ __launch_bounds__(256) void grouped_tn_kernel(const TnArgs t) {
  __shared__ float as[kDepth][kTilePitch], bs[kDepth][kTilePitch];
  const int g = blockIdx.z, m0 = (int)blockIdx.y * kTile, n0 = (int)blockIdx.x * kTile;
  const int begin = group_begin(t.ptr, g, t.rows), end = group_begin(t.ptr, g + 1, t.rows);
  const T *a = static_cast<const T *>(t.a), *b = static_cast<const T *>(t.b);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  float acc[4][4] = {}, sum = 0.f;
  for (int r0 = begin; r0 < end; r0 += kDepth) {
    for (int e = tid; e < kTile * kDepth; e += 256) {
      const int rr = e / kTile, c = e % kTile, r = r0 + rr;
      int id = -1;
      if (r < end) {
        id = t.order ? t.order[r] : r;
        if ((unsigned)id >= (unsigned)t.rows) {
          *t.err = 1;
          id = -1;
        }
      }
      as[rr][c] = id >= 0 && m0 + c < t.m ? to_float(a[(long long)id * t.lda + m0 + c]) : 0.f;
      bs[rr][c] = id >= 0 && n0 + c < t.n ? to_float(b[(long long)id * t.ldb + n0 + c]) : 0.f;
    }
    __syncthreads();
    if (tid < kTile)
      for (int rr = 0; rr < kDepth; rr++) sum += as[rr][tid];
#pragma unroll
    for (int rr = 0; rr < kDepth; rr++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
          acc[i][j] = fmaf(as[rr][ty * 4 + i], bs[rr][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  T *d = static_cast<T *>(t.d) + (long long)g * t.d_group;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m < t.m && n < t.n) d[(long long)m * t.n + n] = from_float<T>(acc[i][j]);
    }
  if (t.sums && blockIdx.x == 0 && tid < kTile && m0 + tid < t.m)
    static_cast<T *>(t.sums)[(long long)g * t.m + m0 + tid] = from_float<T>(sum);
}

template <typename T>
static int launch_rows(const GroupedArgs &a, bool trans_w, hipStream_t s) {
  const dim3 grid((unsigned)(a.rows / kTile + a.n_groups + 1), (unsigned)((a.n + kTile - 1) / kTile));
  if (trans_w) hipLaunchKernelGGL((grouped_rows_kernel<T, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((grouped_rows_kernel<T, false>), grid, dim3(256), 0, s, a);
  INCAGG_HIP_TRY(hipGetLastError());
  return INCAGG_OK;
}

template <typename T> static int launch_tn(const TnArgs &t, hipStream_t s) {
  const dim3 grid((unsigned)((t.n + kTile - 1) / kTile), (unsigned)((t.m + kTile - 1) / kTile),
                  (unsigned)t.n_groups);
  hipLaunchKernelGGL(grouped_tn_kernel<T>, grid, dim3(256), 0, s, t);
  INCAGG_HIP_TRY(hipGetLastError());
  return INCAGG_OK;
}

static int check_groups(const int32_t *ptr, int64_t n_groups, int64_t rows, int dtype) {
  INCAGG_REQUIRE(dtype == INCAGG_DTYPE_F32 || dtype == INCAGG_DTYPE_BF16 || dtype == INCAGG_DTYPE_F16,
                 "unknown element type %d", dtype);
  INCAGG_REQUIRE(rows >= 0 && rows <= INT_MAX - 4096, "rows %lld out of range", (long long)rows);
  INCAGG_REQUIRE(n_groups >= 1 && n_groups <= incagg_group_rows_max_groups(),
                 "n_groups %lld out of range", (long long)n_groups);
  INCAGG_REQUIRE(ptr, "null pointer");
  return INCAGG_OK;
}

}  // namespace incagg

using namespace incagg;

extern "C" int incagg_grouped_gemm(const void *x, int64_t ldx, const void *w, int64_t ldw,
                                   int64_t w_group, int trans_w, const void *bias, int64_t ld_bias,
                                   const int32_t *ptr, const int32_t *order, int64_t n_groups,
                                   int64_t rows, int64_t k, int64_t n, int dtype, void *y,
                                   int64_t ldy, void *stream) {
  int rc = check_groups(ptr, n_groups, rows, dtype);
  if (rc) return rc;
  INCAGG_REQUIRE(k >= 1 && n >= 1 && k < (1 << 20) && n < (1 << 20), "widths out of range");
  if (rows == 0) return INCAGG_OK;
  INCAGG_REQUIRE(x && w && y, "null pointer");
  INCAGG_REQUIRE(ldx >= k && ldy >= n && ldw >= (trans_w ? k : n) && (!bias || ld_bias >= n),
                 "leading dimension too small");
  INCAGG_REQUIRE(w_group >= 0 && w != y && x != y, "y must not alias an operand");
  GroupedArgs a{};
  a.x = x; a.w = w; a.bias = bias; a.y = y;
  a.ldx = ldx; a.ldw = ldw; a.w_group = w_group; a.ld_bias = ld_bias; a.ldy = ldy;
  a.ptr = ptr; a.order = order; a.n_groups = (int)n_groups; a.rows = (int)rows;
  a.k = (int)k; a.n = (int)n;
  rc = error_flag_address(&a.err);
  if (rc) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case INCAGG_DTYPE_F32: return launch_rows<float>(a, trans_w != 0, s);
    case INCAGG_DTYPE_BF16: return launch_rows<__hip_bfloat16>(a, trans_w != 0, s);
    default: return launch_rows<_Float16>(a, trans_w != 0, s);
  }
}

extern "C" int64_t incagg_grouped_tn_ws_bytes(int64_t n_groups, int64_t rows, int64_t m, int64_t n,
                                              int dtype) {
  return 0;
}

extern "C" int incagg_grouped_tn(const void *a, int64_t lda, const void *b, int64_t ldb,
                                 const int32_t *ptr, const int32_t *order, int64_t n_groups,
                                 int64_t rows, int64_t m, int64_t n, int dtype, void *d,
                                 int64_t d_group, void *sums, void *ws, int64_t ws_bytes,
                                 void *stream) {
  int rc = check_groups(ptr, n_groups, rows, dtype);
  if (rc) return rc;
  INCAGG_REQUIRE(m >= 1 && n >= 1 && m < (1 << 20) && n < (1 << 20), "widths out of range");
  INCAGG_REQUIRE(d && d_group >= m * n, "null pointer or d_group < m * n");
  INCAGG_REQUIRE(rows == 0 || (a && b), "null pointer");
  INCAGG_REQUIRE(rows == 0 || (lda >= m && ldb >= n), "leading dimension too small");
  INCAGG_REQUIRE(d != a && d != b, "d must not alias an operand");
  TnArgs t{};
  t.a = a; t.b = b; t.d = d; t.sums = sums; t.lda = lda; t.ldb = ldb; t.d_group = d_group;
  t.ptr = ptr; t.order = order; t.n_groups = (int)n_groups; t.rows = (int)rows;
  t.m = (int)m; t.n = (int)n;
  rc = error_flag_address(&t.err);
  if (rc) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case INCAGG_DTYPE_F32: return launch_tn<float>(t, s);
    case INCAGG_DTYPE_BF16: return launch_tn<__hip_bfloat16>(t, s);
    default: return launch_tn<_Float16>(t, s);
  }
}
