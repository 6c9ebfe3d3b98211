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
// Matrix cores.  Everything runs on v_mfma_f32_16x16x32_{bf16,f16}: 16 times the rate of the
// float32 instruction.  bfloat16 and float16 operands go in as they are.  A float32 value goes in
// as three bfloat16 values, x = h + m + l, each the nearest to what the ones before it leave:
// |x - h - m - l| <= 2^-27 |x|.  A product of two of them is hh + hm + mh + mm + hl + lh; what is
// left out (ml, lm, ll and the two remainders) is below 2^-25 of the product, half a float32
// rounding, and the sums are float32 as ever.  Six instructions against sixteen.  (A value under
// 2^-110 keeps an absolute error of 2^-134, bfloat16's smallest step, in place of the relative one.)
// Infinities, NaNs and values that round to infinity as bfloat16 do not split: the staging code
// looks for them, and a tile that has one is computed again with plain float32 multiply-adds.
//
// LDS holds K-contiguous tiles, [row][BK], one per part of the split, in 16-byte pieces that are
// permuted within 128 bytes so that both the fragment reads and the writes spread over the banks.
// Operands whose reduction index is not the contiguous one (W in dX, both operands in dW) are
// transposed on their way there, in registers: a thread loads 8 rows by V columns and writes V
// pieces of 8.
//
// Sums are held in float32; results are rounded once, to the type of the operands.
#include "common.h"

#include <algorithm>
#include <climits>

namespace incagg {

struct GroupedArgs {
  const void *x, *w, *bias;
  void *y;
  long long ldx, ldw, w_group, ld_bias, ldy;
  const int *ptr, *order;
  int n_groups, rows, k, n, n_tiles;
  int *err;
};

struct TnArgs {
  const void *a, *b;
  void *d, *sums;
  float *partials;
  long long lda, ldb, d_group;
  const int *ptr, *order;
  int n_groups, rows, m, n, m_tiles, n_tiles, segment;
  int *err;
};

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

// Vectors that start at any multiple of their element's size.
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[N]; };

template <int D> struct Type {               // bfloat16, float16
  typedef unsigned short Raw;
  static constexpr int P = 1, BK = 64;       // parts of the split, depth of a tile
};
template <> struct Type<INCAGG_DTYPE_F32> {
  typedef float Raw;
  static constexpr int P = 3, BK = 32;
};

template <int D> __device__ inline float raw_to_float(typename Type<D>::Raw r) {
  if constexpr (D == INCAGG_DTYPE_F32) return r;
  else if constexpr (D == INCAGG_DTYPE_BF16) return __uint_as_float((unsigned)r << 16);
  else return (float)__builtin_bit_cast(_Float16, r);
}

// ---- LDS tiles -------------------------------------------------------------------------------
// Where piece `chunk` (8 values along k) of a row is, in values.  Eight consecutive rows at one
// chunk, and the rows 4 t + v (t = 0 .. 7) that a transposing store writes at once, fall on
// different 16-byte columns.
template <int BK> __device__ inline int piece_at(int row, int chunk) {
  if constexpr (BK == 64) return row * 64 + ((chunk ^ ((row ^ (row >> 3)) & 7)) << 3);
  else return row * 32 + ((chunk ^ (((row >> 1) ^ (row >> 3)) & 3)) << 3);
}

// Eight values along k of one row: into the parts of its tile (PLANE values apart).
template <int D, int PLANE>
__device__ inline void put_piece(unsigned short *tile, int at, const typename Type<D>::Raw (&v)[8],
                                 unsigned &largest) {
  if constexpr (D == INCAGG_DTYPE_F32) {
    u4 h, m, l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      f2 x = {v[2 * i], v[2 * i + 1]};
      largest = max(largest, max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu));
      const unsigned hb = __builtin_bit_cast(unsigned, __builtin_convertvector(x, bf2));
      x.x -= __uint_as_float(hb << 16);
      x.y -= __uint_as_float(hb & 0xffff0000u);
      const unsigned mb = __builtin_bit_cast(unsigned, __builtin_convertvector(x, bf2));
      x.x -= __uint_as_float(mb << 16);
      x.y -= __uint_as_float(mb & 0xffff0000u);
      h[i] = hb;
      m[i] = mb;
      l[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(x, bf2));
    }
    *reinterpret_cast<u4 *>(tile + at) = h;
    *reinterpret_cast<u4 *>(tile + PLANE + at) = m;
    *reinterpret_cast<u4 *>(tile + 2 * PLANE + at) = l;
  } else {
    u4 h;
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = (unsigned)v[2 * i] | ((unsigned)v[2 * i + 1] << 16);
    *reinterpret_cast<u4 *>(tile + at) = h;
  }
}

// A value whose nearest bfloat16 is not finite.
constexpr unsigned kUnsplittable = 0x7f7f8000u;

// Rows whose k values are contiguous: ROWS x BK, a thread takes U pieces.
template <int D, int ROWS, int THREADS> struct RowStage {
  typedef typename Type<D>::Raw Raw;
  static constexpr int BK = Type<D>::BK, CH = BK / 8, UNITS = ROWS * CH;
  static constexpr int U = (UNITS + THREADS - 1) / THREADS;
  const Raw *src[U];
  Pack<Raw, 8> r[U];
  template <typename F> __device__ void init(F &&row_of) {
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int u = (int)threadIdx.x + i * THREADS;
      src[i] = row_of(min(u / CH, ROWS - 1)) + (u % CH) * 8;
    }
  }
  __device__ void load(int k0, int k) {
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int u = (int)threadIdx.x + i * THREADS, at = k0 + (u % CH) * 8;
      if (UNITS % THREADS != 0 && u >= UNITS) continue;
      if (at + 8 <= k) {
        r[i] = *reinterpret_cast<const Pack<Raw, 8> *>(src[i] + k0);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) r[i].v[e] = at + e < k ? src[i][k0 + e] : (Raw)0;
      }
    }
  }
  __device__ void store(unsigned short *tile, unsigned &largest) {
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int u = (int)threadIdx.x + i * THREADS;
      if (UNITS % THREADS != 0 && u >= UNITS) continue;
      Raw v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = r[i].v[e];
      put_piece<D, ROWS * BK>(tile, piece_at<BK>(u / CH, u % CH), v, largest);
    }
  }
};

// The transposing form: rows along the reduction, COLS columns of them become the tile's rows.  A
// thread takes 8 rows x V columns.
template <int D, int COLS, int THREADS> struct ColStage {
  typedef typename Type<D>::Raw Raw;
  static constexpr int BK = Type<D>::BK;
  static constexpr int V = COLS * BK / 8 >= THREADS ? COLS * BK / 8 / THREADS : 1;
  static constexpr int GROUPS = COLS / V;
  Pack<Raw, V> r[8];
  static __device__ int col() { return ((int)threadIdx.x % GROUPS) * V; }
  static __device__ int row() { return ((int)threadIdx.x / GROUPS) * 8; }
  static __device__ bool active() { return GROUPS * (BK / 8) >= THREADS || row() < BK; }
  // row i (0 .. 7) of this thread starts at row_of(i), NULL for none; `cols`: columns from this
  // thread's first one to the matrix's end
  template <typename F> __device__ void load(int cols, F &&row_of) {
    if (!active()) return;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const Raw *p = row_of(i);
      if (p && cols >= V) {
        r[i] = *reinterpret_cast<const Pack<Raw, V> *>(p);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) r[i].v[e] = p && e < cols ? p[e] : (Raw)0;
      }
    }
  }
  __device__ void store(unsigned short *tile, unsigned &largest) {
    if (!active()) return;
#pragma unroll
    for (int e = 0; e < V; e++) {
      Raw v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = r[i].v[e];
      put_piece<D, COLS * BK>(tile, piece_at<BK>(col() + e, row() / 8), v, largest);
    }
  }
};

// ---- the matrix-core loop over one pair of tiles ------------------------------------------------
// acc[i][j]: 16 x 16 blocks; lane l holds columns 4 (l / 16) .. + 3 of block j (the fast index of
// the result) at row l % 16 of block i.
template <int D> __device__ inline f4 mfma(u4 a, u4 b, f4 c) {
  if constexpr (D == INCAGG_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b),
                                                  c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a),
                                                   __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

template <int D, int ROWS, int COLS, int MI, int NJ>
__device__ inline void multiply(const unsigned short *rows, const unsigned short *cols, int row0,
                                int col0, f4 (&acc)[MI][NJ]) {
  constexpr int BK = Type<D>::BK, P = Type<D>::P;
  const int l16 = threadIdx.x & 15, quad = (threadIdx.x >> 4) & 3;
#pragma unroll
  for (int kk = 0; kk < BK / 32; kk++) {
    u4 a[MI][P];
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
      for (int p = 0; p < P; p++)
        a[i][p] = *reinterpret_cast<const u4 *>(
            rows + p * ROWS * BK + piece_at<BK>(row0 + 16 * i + l16, kk * 4 + quad));
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      u4 b[P];
#pragma unroll
      for (int p = 0; p < P; p++)
        b[p] = *reinterpret_cast<const u4 *>(
            cols + p * COLS * BK + piece_at<BK>(col0 + 16 * j + l16, kk * 4 + quad));
      if constexpr (P == 1) {
#pragma unroll
        for (int i = 0; i < MI; i++) acc[i][j] = mfma<D>(b[0], a[i][0], acc[i][j]);
      } else {
        constexpr int PA[6] = {0, 0, 1, 1, 0, 2}, PB[6] = {0, 1, 0, 1, 2, 0};
#pragma unroll
        for (int t = 0; t < 6; t++)
#pragma unroll
          for (int i = 0; i < MI; i++) acc[i][j] = mfma<D>(b[PB[t]], a[i][PA[t]], acc[i][j]);
      }
    }
  }
}

// Four neighbouring results of a row, rounded to their type.
template <int D> __device__ inline void put_results(void *base, long long at, int count, f4 v) {
  typedef typename Type<D>::Raw Raw;
  Raw *p = static_cast<Raw *>(base) + at;
  Pack<Raw, 4> q;
  if constexpr (D == INCAGG_DTYPE_F32) {
    q = __builtin_bit_cast(Pack<Raw, 4>, v);
  } else if constexpr (D == INCAGG_DTYPE_BF16) {
    q = __builtin_bit_cast(Pack<Raw, 4>, __builtin_convertvector(v, bf4));   // nearest even
  } else {
    q = __builtin_bit_cast(Pack<Raw, 4>, __builtin_convertvector(v, h4));
  }
  if (count >= 4) {
    *reinterpret_cast<Pack<Raw, 4> *>(p) = q;
  } else {
#pragma unroll
    for (int e = 0; e < 3; e++)
      if (e < count) p[e] = q.v[e];
  }
}

// ---- finding the work ----------------------------------------------------------------------------
// First row of group g; entries that are out of order or range never lead outside [0, rows].
__device__ inline int group_begin(const int *ptr, int g, int rows) {
  return g == 0 ? 0 : min(max(ptr[g], 0), rows);
}

// The row tile of a slot: false if the slot is empty.  g == n_groups: rows of no group.
template <int THREADS>
__device__ inline bool tile_of_slot(const int *ptr, int n_groups, int rows, int tile_rows, int slot,
                                    int *g, int *first, int *end, int *tile) {
  int before = 0;
  for (int base = 1; base <= n_groups; base += THREADS) {
    const int j = base + (int)threadIdx.x;
    before += __syncthreads_count(j <= n_groups &&
                                  group_begin(ptr, j, rows) / tile_rows + j <= slot);
  }
  const int p0 = group_begin(ptr, before, rows);
  *tile = slot - (p0 / tile_rows + before);
  *g = before;
  *first = p0 + *tile * tile_rows;
  *end = before == n_groups ? rows : group_begin(ptr, before + 1, rows);
  return *tile >= 0 && *first < *end;
}

// Workgroups go round-robin over the 8 XCDs; this gives each XCD a contiguous range of the work,
// so that the column tiles of a row tile meet in one L2.
__device__ inline int xcd_contiguous(int block, int blocks) {
  const int xcd = block & 7, per = blocks >> 3, rem = blocks & 7;
  return xcd * per + min(xcd, rem) + (block >> 3);
}

// A row number of `order`, -1 (and reported) outside the matrix.
__device__ inline int row_at(const int *order, int r, int rows, int *err) {
  const int id = order ? order[r] : r;
  if ((unsigned)id < (unsigned)rows) return id;
  *err = 1;
  return -1;
}

// ---- Y = X W + b -----------------------------------------------------------------------------------
template <int D, int BM, int BN, int WM, int WN, bool TRANS_W, int STAGES>
__global__ __launch_bounds__(64 * WM * WN) void grouped_rows_kernel(const GroupedArgs a) {
  typedef typename Type<D>::Raw Raw;
  constexpr int T = 64 * WM * WN, BK = Type<D>::BK, P = Type<D>::P;
  constexpr int MI = BM / WM / 16, NJ = BN / WN / 16;
  __shared__ __align__(16) unsigned short xt[STAGES][P * BM * BK], wt[STAGES][P * BN * BK];
  __shared__ int row_ids[BM];
  const int work = xcd_contiguous(blockIdx.x, gridDim.x);
  const int slot = work / a.n_tiles, n0 = (work - slot * a.n_tiles) * BN;
  int g, first, end, tile;
  if (!tile_of_slot<T>(a.ptr, a.n_groups, a.rows, BM, slot, &g, &first, &end, &tile)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row0 = (wave / WN) * (BM / WM), col0 = (wave % WN) * (BN / WN);
  for (int i = tid; i < BM; i += T)
    row_ids[i] = first + i < end ? row_at(a.order, first + i, a.rows, a.err) : -1;
  __syncthreads();

  f4 acc[MI][NJ] = {};
  const Raw *x = static_cast<const Raw *>(a.x);
  const Raw *w = static_cast<const Raw *>(a.w) + (long long)g * a.w_group;
  if (g < a.n_groups) {
    // (rows and columns outside the matrices repeat one inside; their results are dropped)
    RowStage<D, BM, T> xs;
    xs.init([&](int r) { return x + (long long)max(row_ids[r], 0) * a.ldx; });
    RowStage<D, TRANS_W ? BN : 16, T> wr;
    ColStage<D, TRANS_W ? 16 : BN, T> wc;
    if constexpr (TRANS_W) wr.init([&](int c) { return w + (long long)min(n0 + c, a.n - 1) * a.ldw; });
    const int n_chunks = (a.k + BK - 1) / BK;
    unsigned largest = 0;
    auto load = [&](int c) {
      xs.load(c * BK, a.k);
      if constexpr (TRANS_W) {
        wr.load(c * BK, a.k);
      } else {
        const int r0 = c * BK + wc.row(), n = n0 + wc.col();
        const Raw *p = w + (long long)r0 * a.ldw + n;
        wc.load(a.n - n, [&](int i) { return r0 + i < a.k ? p + i * a.ldw : nullptr; });
      }
    };
    auto store = [&](int s) {
      xs.store(xt[s], largest);
      if constexpr (TRANS_W) wr.store(wt[s], largest);
      else wc.store(wt[s], largest);
    };
    load(0);
    if constexpr (STAGES == 2) {
      store(0);
      __syncthreads();
      for (int c = 0; c < n_chunks; c++) {
        if (c + 1 < n_chunks) load(c + 1);
        multiply<D, BM, BN>(xt[c & 1], wt[c & 1], row0, col0, acc);
        if (c + 1 < n_chunks) store((c + 1) & 1);
        __syncthreads();
      }
    } else {
      for (int c = 0; c < n_chunks; c++) {
        if (c > 0) __syncthreads();
        store(0);
        __syncthreads();
        if (c + 1 < n_chunks) load(c + 1);
        multiply<D, BM, BN>(xt[0], wt[0], row0, col0, acc);
      }
    }
    if constexpr (D == INCAGG_DTYPE_F32) {
      if (__syncthreads_or(largest >= kUnsplittable)) {
        for (int i = 0; i < MI; i++)
          for (int j = 0; j < NJ; j++)
            for (int r = 0; r < 4; r++) {
              const int id = row_ids[row0 + 16 * i + (lane & 15)];
              const int n = n0 + col0 + 16 * j + 4 * (lane >> 4) + r;
              float s = 0.f;
              if (id >= 0 && n < a.n) {
                const Raw *px = x + (long long)id * a.ldx;
                const Raw *pw = TRANS_W ? w + (long long)n * a.ldw : w + n;
                const long long step = TRANS_W ? 1 : a.ldw;
                for (int k = 0; k < a.k; k++) s = fmaf(px[k], pw[k * step], s);
              }
              acc[i][j][r] = s;
            }
      }
    }
  }

  const Raw *bias = a.bias && g < a.n_groups
                        ? static_cast<const Raw *>(a.bias) + (long long)g * a.ld_bias : nullptr;
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    const int n = n0 + col0 + 16 * j + 4 * (lane >> 4);
    if (n >= a.n) continue;
    f4 b = {0.f, 0.f, 0.f, 0.f};
    if (bias)
#pragma unroll
      for (int e = 0; e < 4; e++) b[e] = n + e < a.n ? raw_to_float<D>(bias[n + e]) : 0.f;
#pragma unroll
    for (int i = 0; i < MI; i++) {
      const int id = row_ids[row0 + 16 * i + (lane & 15)];
      if (id < 0) continue;
      f4 v;
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = acc[i][j][e] + b[e];
      put_results<D>(a.y, (long long)id * a.ldy + n, a.n - n, v);
    }
  }
}

// ---- D_g = sum A^T B ---------------------------------------------------------------------------------
// A group's rows are cut into segments of `segment` rows; a group of one segment writes its D
// itself (an empty one zeros), the segments of a longer one leave float32 partials that a second
// launch adds up in order.  Partials of group g start at 3 ptr[g] / segment: a group of n > segment
// rows has at most 3 n / segment - 1 segments, so no two groups meet.
__device__ inline long long partial_at(const int *ptr, int g, int rows, int segment, int tile) {
  return 3ll * group_begin(ptr, g, rows) / segment + tile;
}

template <int D, int BM, int BN>
__global__ __launch_bounds__(256) void grouped_tn_kernel(const TnArgs t) {
  typedef typename Type<D>::Raw Raw;
  constexpr int T = 256, BK = Type<D>::BK, P = Type<D>::P;
  constexpr int MI = BM / 32, NJ = BN / 32;
  constexpr int TILES = P * (BM + BN) * BK;
  __shared__ __align__(16) unsigned short tiles[TILES];
  unsigned short *at = tiles, *bt = tiles + P * BM * BK;
  const int work = xcd_contiguous(blockIdx.x, gridDim.x);
  const int per_slot = t.m_tiles * t.n_tiles, slot = work / per_slot, mn = work - slot * per_slot;
  const int m0 = (mn / t.n_tiles) * BM, n0 = (mn % t.n_tiles) * BN;
  int g, first, end, seg;
  const bool any = tile_of_slot<T>(t.ptr, t.n_groups, t.rows, t.segment, slot, &g, &first, &end, &seg);
  if (g >= t.n_groups || seg < 0 || (!any && seg > 0)) return;
  const int begin = group_begin(t.ptr, g, t.rows);
  const bool whole = end - begin <= t.segment;       // the group's only segment (or an empty group)
  const int last = min(end, first + t.segment);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row0 = (wave >> 1) * (BM / 2), col0 = (wave & 1) * (BN / 2);
  const Raw *a = static_cast<const Raw *>(t.a), *b = static_cast<const Raw *>(t.b);
  const bool want_sums = t.sums && n0 == 0;

  f4 acc[MI][NJ] = {};
  ColStage<D, BM, T> as;
  ColStage<D, BN, T> bs;
  float sums[decltype(as)::V] = {};
  unsigned largest = 0;
  const int acols = t.m - m0 - as.col(), bcols = t.n - n0 - bs.col();
  auto load = [&](int r0) {
    const int ra = r0 + as.row(), rb = r0 + bs.row();
    as.load(acols, [&](int i) -> const Raw * {
      const int id = ra + i < last ? row_at(t.order, ra + i, t.rows, t.err) : -1;
      return id < 0 ? nullptr : a + (long long)id * t.lda + m0 + as.col();
    });
    bs.load(bcols, [&](int i) -> const Raw * {
      const int id = rb + i < last ? row_at(t.order, rb + i, t.rows, t.err) : -1;
      return id < 0 ? nullptr : b + (long long)id * t.ldb + n0 + bs.col();
    });
  };
  if (first < last) {
    load(first);
    for (int r0 = first; r0 < last; r0 += BK) {
      if (r0 > first) __syncthreads();
      as.store(at, largest);
      bs.store(bt, largest);
      if (want_sums && as.active())
#pragma unroll
        for (int e = 0; e < decltype(as)::V; e++) {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < 8; i++) s += raw_to_float<D>(as.r[i].v[e]);
          sums[e] += s;
        }
      __syncthreads();
      if (r0 + BK < last) load(r0 + BK);
      multiply<D, BM, BN>(at, bt, row0, col0, acc);
    }
  }
  if constexpr (D == INCAGG_DTYPE_F32) {
    if (__syncthreads_or(largest >= kUnsplittable)) {
      for (int i = 0; i < MI; i++)
        for (int j = 0; j < NJ; j++)
          for (int e = 0; e < 4; e++) {
            const int m = m0 + row0 + 16 * i + (lane & 15), n = n0 + col0 + 16 * j + 4 * (lane >> 4) + e;
            float s = 0.f;
            if (m < t.m && n < t.n)
              for (int r = first; r < last; r++) {
                const int id = row_at(t.order, r, t.rows, t.err);
                if (id >= 0) s = fmaf(a[(long long)id * t.lda + m], b[(long long)id * t.ldb + n], s);
              }
            acc[i][j][e] = s;
          }
    }
  }

  const long long part = (long long)t.m * t.n + (t.sums ? t.m : 0);
  float *partial = t.partials + partial_at(t.ptr, g, t.rows, t.segment, seg) * part;
#pragma unroll
  for (int i = 0; i < MI; i++) {
    const int m = m0 + row0 + 16 * i + (lane & 15);
    if (m >= t.m) continue;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int n = n0 + col0 + 16 * j + 4 * (lane >> 4);
      if (n >= t.n) continue;
      const long long e = (long long)m * t.n + n;
      if (whole) put_results<D>(t.d, g * t.d_group + e, t.n - n, acc[i][j]);
      else put_results<INCAGG_DTYPE_F32>(partial, e, t.n - n, acc[i][j]);
    }
  }
  if (!want_sums) return;
  // column sums: threads of one column group, row groups in order
  constexpr int V = decltype(as)::V, GROUPS = decltype(as)::GROUPS, RG = BK / 8;
  static_assert(sizeof(float) * RG * BM <= sizeof(tiles), "reduction space");
  float *red = reinterpret_cast<float *>(tiles);
  __syncthreads();
  if (as.active())
#pragma unroll
    for (int e = 0; e < V; e++) red[(as.row() / 8) * BM + as.col() + e] = sums[e];
  __syncthreads();
  (void)GROUPS;
  for (int c = tid; c < BM && m0 + c < t.m; c += T) {
    float s = 0.f;
    for (int r = 0; r < RG; r++) s += red[r * BM + c];
    if (whole) {
      const f4 v = {s, 0.f, 0.f, 0.f};
      put_results<D>(t.sums, (long long)g * t.m + m0 + c, 1, v);
    } else {
      partial[(long long)t.m * t.n + m0 + c] = s;
    }
  }
}

template <int D> __global__ __launch_bounds__(256) void grouped_tn_finish_kernel(const TnArgs t) {
  const int g = blockIdx.y;
  const int begin = group_begin(t.ptr, g, t.rows), end = group_begin(t.ptr, g + 1, t.rows);
  if (end - begin <= t.segment) return;
  const int segments = (end - begin + t.segment - 1) / t.segment;
  const long long mn = (long long)t.m * t.n, part = mn + (t.sums ? t.m : 0);
  const long long e = (blockIdx.x * 256ll + threadIdx.x) * 4;
  if (e >= part) return;
  const float *p = t.partials + partial_at(t.ptr, g, t.rows, t.segment, 0) * part + e;
  const int count = (int)min(4ll, part - e);
  f4 s = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < segments; i++, p += part) {
    if (count == 4) {
      const Pack<float, 4> q = *reinterpret_cast<const Pack<float, 4> *>(p);
#pragma unroll
      for (int j = 0; j < 4; j++) s[j] += q.v[j];
    } else {
      for (int j = 0; j < count; j++) s[j] += p[j];
    }
  }
  if (e + 4 <= mn) {
    put_results<D>(t.d, g * t.d_group + e, 4, s);
  } else {
    for (int j = 0; j < count; j++) {
      const f4 v = {s[j], 0.f, 0.f, 0.f};
      if (e + j < mn) put_results<D>(t.d, g * t.d_group + e + j, 1, v);
      else put_results<D>(t.sums, (long long)g * t.m + (e + j - mn), 1, v);
    }
  }
}

// ---- host side ---------------------------------------------------------------------------------------
template <int D, int BM, int BN, int WM, int WN, int STAGES>
static int launch_rows_tile(GroupedArgs &a, bool trans_w, hipStream_t s) {
  a.n_tiles = (a.n + BN - 1) / BN;
  const int64_t blocks = ((int64_t)a.rows / BM + a.n_groups + 1) * a.n_tiles;
  INCAGG_REQUIRE(blocks < (1ll << 31), "too many rows and columns for one call");
  const dim3 grid((unsigned)blocks), block(64 * WM * WN);
  if (trans_w)
    hipLaunchKernelGGL((grouped_rows_kernel<D, BM, BN, WM, WN, true, STAGES>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((grouped_rows_kernel<D, BM, BN, WM, WN, false, STAGES>), grid, block, 0, s, a);
  INCAGG_HIP_TRY(hipGetLastError());
  return INCAGG_OK;
}

template <int D> static int launch_rows(GroupedArgs &a, bool trans_w, hipStream_t s) {
  constexpr int STAGES = D == INCAGG_DTYPE_F32 ? 1 : 2;
  // few rows to a group: the weights are what is read, and a tall tile would be mostly empty
  if ((int64_t)a.rows <= 48ll * a.n_groups)
    return launch_rows_tile<D, 16, 64, 1, 4, STAGES>(a, trans_w, s);
  if (a.n <= 64) return launch_rows_tile<D, 128, 64, 4, 1, STAGES>(a, trans_w, s);
  return launch_rows_tile<D, 128, 128, 2, 2, STAGES>(a, trans_w, s);
}

// Rows of a segment: enough segments to fill the chip (about 1024 workgroups), at least 512 rows.
static int tn_segment(int64_t rows, int64_t m, int64_t n) {
  const int64_t tiles = ((m + 127) / 128) * ((n + 127) / 128);
  const int64_t wanted = std::max<int64_t>(1, 1024 / tiles);
  const int64_t s = std::max<int64_t>(512, (rows + wanted - 1) / wanted);
  return (int)((s + 63) / 64 * 64);
}

template <int D, int BM, int BN> static int launch_tn_tile(TnArgs &t, hipStream_t s) {
  t.m_tiles = (t.m + BM - 1) / BM;
  t.n_tiles = (t.n + BN - 1) / BN;
  const int64_t blocks = ((int64_t)t.rows / t.segment + t.n_groups) * t.m_tiles * t.n_tiles;
  INCAGG_REQUIRE(blocks < (1ll << 31), "too many rows and columns for one call");
  hipLaunchKernelGGL((grouped_tn_kernel<D, BM, BN>), dim3((unsigned)blocks), dim3(256), 0, s, t);
  INCAGG_HIP_TRY(hipGetLastError());
  if (t.rows > t.segment) {
    const int64_t part = (int64_t)t.m * t.n + (t.sums ? t.m : 0);
    hipLaunchKernelGGL(grouped_tn_finish_kernel<D>,
                       dim3((unsigned)((part + 1023) / 1024), (unsigned)t.n_groups), dim3(256), 0, s, t);
    INCAGG_HIP_TRY(hipGetLastError());
  }
  return INCAGG_OK;
}

template <int D> static int launch_tn(TnArgs &t, hipStream_t s) {
  if (t.m <= 64) return t.n <= 64 ? launch_tn_tile<D, 64, 64>(t, s) : launch_tn_tile<D, 64, 128>(t, s);
  return t.n <= 64 ? launch_tn_tile<D, 128, 64>(t, s) : launch_tn_tile<D, 128, 128>(t, s);
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
    case INCAGG_DTYPE_F32: return launch_rows<INCAGG_DTYPE_F32>(a, trans_w != 0, s);
    case INCAGG_DTYPE_BF16: return launch_rows<INCAGG_DTYPE_BF16>(a, trans_w != 0, s);
    default: return launch_rows<INCAGG_DTYPE_F16>(a, trans_w != 0, s);
  }
}

extern "C" int64_t incagg_grouped_tn_ws_bytes(int64_t n_groups, int64_t rows, int64_t m, int64_t n,
                                              int dtype) {
  if (n_groups < 1 || rows < 0 || rows > INT_MAX - 4096 || m < 1 || n < 1 || m >= (1 << 20) ||
      n >= (1 << 20))
    return fail(INCAGG_E_INVALID, "size out of range");
  const int64_t segment = tn_segment(rows, m, n);
  return rows <= segment ? 0 : (3 * rows / segment + 1) * (m * n + m) * (int64_t)sizeof(float);
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
  const int64_t need = incagg_grouped_tn_ws_bytes(n_groups, rows, m, n, dtype);
  if (need < 0) return (int)need;
  INCAGG_REQUIRE(need == 0 || (ws && ws_bytes >= need), "workspace too small: %lld < %lld",
                 (long long)ws_bytes, (long long)need);
  TnArgs t{};
  t.partials = static_cast<float *>(ws);
  t.segment = tn_segment(rows, m, n);
  t.a = a; t.b = b; t.d = d; t.sums = sums; t.lda = lda; t.ldb = ldb; t.d_group = d_group;
  t.ptr = ptr; t.order = order; t.n_groups = (int)n_groups; t.rows = (int)rows;
  t.m = (int)m; t.n = (int)n;
  rc = error_flag_address(&t.err);
  if (rc) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case INCAGG_DTYPE_F32: return launch_tn<INCAGG_DTYPE_F32>(t, s);
    case INCAGG_DTYPE_BF16: return launch_tn<INCAGG_DTYPE_BF16>(t, s);
    default: return launch_tn<INCAGG_DTYPE_F16>(t, s);
  }
}
