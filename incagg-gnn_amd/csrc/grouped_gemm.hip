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
// as three bfloat16 values, 2^16 x = h + m + l, each the nearest to what the ones before it leave.
// The sum is exact: 3 x 8 bits, and the last bit of the smallest float32 value, 2^-149, times 2^16 is
// bfloat16's own last bit (without the factor, values under 2^-110 lose bits: errors of 3e-4 for 1e37 x
// 1e-37).  A product of two of them is hh + hm + mh + mm + hl + lh; what is left out, ml + lm + ll, is
// at most 2^-24 of the product (|m| <= 2^-8, |l| <= 2^-17 of a value in [1, 2)), one float32 rounding,
// and the sums are float32 as ever, scaled by 2^-32 at their end.  Six instructions against sixteen.
// (The scaling costs 2 %: 128064 x 100 -> 256 77.0 / 78.8 us without / with.  The float32 figures at the
// choices of tiles below were taken without it, on both sides.)
// Infinities, NaNs, values from 2^112 on and sums from 2^96 on do not go through: their parts or sums
// are not finite, and a tile with such a result is computed again with plain float32 multiply-adds, a
// loop over k for each of its results, over the rows of its segment in the weight gradient.  Right, but
// slow: one row of NaNs takes 128064 x 100 -> 256 from 76 to 339 us and its weight gradient from 97 to
// 2100, 200000 x 512 -> 256 in one group from 380 us to 4 ms and from 390 us to 17 ms; one in every 16
// rows, the former from 380 us to 49 ms.
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
  int n_groups, rows, m, n, m_tiles, n_tiles, segment, slots;
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

// Eight float32 values along k of one row: into the three parts of its tile (PLANE values apart).
constexpr float kSplitScale = 0x1p16f, kSplitUnscale = 0x1p-32f;      // of a value, of a sum of products
template <int PLANE>
__device__ inline void put_split(unsigned short *tile, int at, const float (&v)[8]) {
  u4 h, m, l;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f2 x = {v[2 * i] * kSplitScale, v[2 * i + 1] * kSplitScale};
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
}

// 16 bytes shifted down by `halves` times 16 bits (0 .. 8), zeros behind.
__device__ inline void shift_down(unsigned *v, int halves) {
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = halves & 2 ? (e < 3 ? v[e + 1] : 0u) : v[e];
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = halves & 4 ? (e < 2 ? v[e + 2] : 0u) : v[e];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const unsigned odd = v[e] >> 16 | (e < 3 ? v[e + 1] << 16 : 0u);
    v[e] = halves & 8 ? 0u : (halves & 1 ? odd : v[e]);
  }
}

// Loads at ragged edges are whole vectors as well, of what lies in front of the edge, shifted: a
// load per element under a condition of its own would wait for the one before it.

// Rows whose k values are contiguous: ROWS x BK, a thread takes U pieces of 8 values.
template <int D, int ROWS, int THREADS> struct RowStage {
  typedef typename Type<D>::Raw Raw;
  static constexpr int BK = Type<D>::BK, CH = BK / 8, UNITS = ROWS * CH;
  static constexpr int U = (UNITS + THREADS - 1) / THREADS, W = 2 * sizeof(Raw);
  const Raw *src[U];
  Pack<unsigned, W> r[U];               // 8 values
  static __device__ int unit(int i) {
    const int u = (int)threadIdx.x + i * THREADS;
    return UNITS % THREADS ? min(u, UNITS - 1) : u;      // (the last piece more than once)
  }
  template <typename F> __device__ void init(F &&row_of) {
#pragma unroll
    for (int i = 0; i < U; i++) src[i] = row_of(unit(i) / CH) + (unit(i) % CH) * 8;
  }
  __device__ void load(int k0) {
#pragma unroll
    for (int i = 0; i < U; i++)
      r[i] = __builtin_bit_cast(Pack<unsigned, W>,
                                *reinterpret_cast<const Pack<Raw, 8> *>(src[i] + k0));
  }
  // the last chunk of a row of k values; settle() moves them to where they belong
  static constexpr int N = 16 / sizeof(Raw);    // values of a load
  __device__ void load_tail(int k0, int k) {
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int at = (unit(i) % CH) * 8;
      const Raw *row = src[i] - at;
#pragma unroll
      for (int h = 0; h < 8; h += N) {
        Pack<unsigned, 4> q;
        if (k >= N) {
          q = *reinterpret_cast<const Pack<unsigned, 4> *>(
              reinterpret_cast<const Pack<Raw, N> *>(row + min(k0 + at + h, k - N)));
        } else {
          Pack<Raw, N> v;
#pragma unroll
          for (int e = 0; e < N; e++) v.v[e] = at + h + e < k ? row[at + h + e] : (Raw)0;
          q = __builtin_bit_cast(Pack<unsigned, 4>, v);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) r[i].v[h * (int)sizeof(Raw) / 4 + e] = q.v[e];
      }
    }
  }
  // in front of the store of a chunk with `left` values along k: where the values are waited for
  // anyhow (at the load, the wait would stand in front of the products of the chunk before)
  __device__ void settle(int left, int k) {
    if (left >= BK || k < N) return;
#pragma unroll
    for (int i = 0; i < U; i++)
#pragma unroll
      for (int h = 0; h < 8; h += N) {
        const int here = left - (unit(i) % CH) * 8 - h;       // values from here to the row's end
        shift_down(&r[i].v[h * (int)sizeof(Raw) / 4],
                   (N - min(max(here, 0), N)) * ((int)sizeof(Raw) / 2));
      }
  }
  __device__ void store(unsigned short *tile) {
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int at = piece_at<BK>(unit(i) / CH, unit(i) % CH);
      if constexpr (D == INCAGG_DTYPE_F32) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = __uint_as_float(r[i].v[e]);
        put_split<ROWS * BK>(tile, at, v);
      } else {
        *reinterpret_cast<u4 *>(tile + at) = u4{r[i].v[0], r[i].v[1], r[i].v[2], r[i].v[3]};
      }
    }
  }
};

// The transposing form: rows along the reduction, COLS columns of them (from `first` of a matrix of n
// on) become the tile's rows.  A thread takes 8 rows x V columns.
template <int D, int COLS, int THREADS> struct ColStage {
  typedef typename Type<D>::Raw Raw;
  static constexpr int BK = Type<D>::BK, V = COLS * BK / 8 / THREADS, GROUPS = COLS / V;
  static_assert(V >= 1 && V <= 4 && GROUPS * (BK / 8) == THREADS, "every thread takes 8 x V values");
  typedef Raw Row __attribute__((ext_vector_type(V)));
  Row r[8];
  int at, shift;                        // where this thread's columns are loaded from, moved by what
  static __device__ int col() { return ((int)threadIdx.x % GROUPS) * V; }
  static __device__ int row() { return ((int)threadIdx.x / GROUPS) * 8; }
  __device__ void init(int first, int n) {
    const int begin = first + col();
    at = n < V ? begin : min(begin, n - V);
    shift = begin >= n ? 0 : begin - at;        // (columns behind the last: dropped)
  }
  // row i (0 .. 7) of this thread starts at row_of(i), which has to be a row of the matrix of n columns
  template <typename F> __device__ void load(int n, F &&row_of) {
    if (n >= V) {
#pragma unroll
      for (int i = 0; i < 8; i++)
        r[i] = __builtin_bit_cast(Row, *reinterpret_cast<const Pack<Raw, V> *>(row_of(i) + at));
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const Raw *p = row_of(i) + at;
#pragma unroll
        for (int e = 0; e < V; e++) r[i][e] = at + e < n ? p[e] : (Raw)0;
      }
    }
  }
  // rows from `count` on are not part of the reduction
  __device__ void clear_from(int count) {
#pragma unroll
    for (int i = 0; i < 8; i++) clear_row(i, i < count);
  }
  __device__ void clear_row(int i, bool keep) {
#pragma unroll
    for (int e = 0; e < V; e++) r[i][e] = keep ? r[i][e] : (Raw)0;
  }
  // moves the columns of the edge's thread to where they belong (once, in front of store)
  __device__ void settle() {
    if (V == 1 || shift == 0) return;
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
      for (int e = 0; e < V; e++) {
        Raw v = (Raw)0;
#pragma unroll
        for (int f = e + 1; f < V; f++) v = f - e == shift ? r[i][f] : v;
        r[i][e] = v;
      }
  }
  __device__ void store(unsigned short *tile) {
#pragma unroll
    for (int e = 0; e < V; e++) {
      const int at = piece_at<BK>(col() + e, row() / 8);
      if constexpr (D == INCAGG_DTYPE_F32) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = r[i][e];
        put_split<COLS * BK>(tile, at, v);
      } else {
        u4 h;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if constexpr (V >= 2) {       // halves of two dwords into one
            typedef unsigned Pairs __attribute__((ext_vector_type(V / 2)));
            const unsigned lo = __builtin_bit_cast(Pairs, r[2 * i])[e / 2];
            const unsigned hi = __builtin_bit_cast(Pairs, r[2 * i + 1])[e / 2];
            h[i] = __builtin_amdgcn_perm(hi, lo, e & 1 ? 0x07060302u : 0x05040100u);
          } else {
            h[i] = (unsigned)r[2 * i][e] | ((unsigned)r[2 * i + 1][e] << 16);
          }
        }
        *reinterpret_cast<u4 *>(tile + at) = h;
      }
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

// Whether this lane's results are all finite: of the rows that keeps(i) names (of blocks i) and the
// first `columns` columns from its own first on.  What is not stored may come from any row or column
// of the operands, and does not count.
template <int MI, int NJ, typename Keeps>
__device__ inline bool all_finite(const f4 (&acc)[MI][NJ], int columns, Keeps &&keeps) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < MI; i++) {
    const int count = keeps(i) ? columns : 0;
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int e = 0; e < 4; e++)         // NaN once one is not finite
        s = fmaf(16 * j + e < count ? acc[i][j][e] : 0.f, 0.f, s);
  }
  return s == 0.f;
}

// Sums of products of split values, back from their scale.
template <int MI, int NJ> __device__ inline void unscale(f4 (&acc)[MI][NJ]) {
#pragma unroll
  for (int i = 0; i < MI; i++)
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[i][j][e] *= kSplitUnscale;
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

// The blocks of a wave as whole rows: each row of 16 blocks goes through LDS (`scratch`, this wave's
// own, kRowScratch<D, NJ> values), from where a lane stores 16 bytes and neighbouring lanes the next
// ones.  Straight from the accumulators a store instruction covers 16 rows by 32 or 64 bytes, parts
// of lines only: 131072 x 2048 bfloat16 results at 1.8 TB/s, 300 us of an 890 us launch.
// at(row): where the row's first column lies in memory, NULL for a row that is not stored.
template <int D, int NJ>
constexpr int kRowScratch = 16 * NJ * 16 * sizeof(typename Type<D>::Raw) / 2;   // (16-bit values)

template <int D, int NJ, typename At>
__device__ __forceinline__ void put_rows(unsigned short *scratch, const f4 (&v)[NJ], int count,
                                         At &&at) {
  typedef typename Type<D>::Raw Raw;
  constexpr int V = 16 / sizeof(Raw), PIECES = NJ * 16 / V, Q = (16 * PIECES + 63) / 64;
  static_assert((PIECES & (PIECES - 1)) == 0, "a row is a power of two of pieces");
  const int lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
  Raw *rows = reinterpret_cast<Raw *>(scratch);
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    const int col = 16 * j + 4 * quad, place = (col / V) ^ (l16 & (PIECES - 1));
    put_results<D>(rows, (l16 * PIECES + place) * V + col % V, 4, v[j]);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int q = 0; q < Q; q++) {
    if (Q * 64 > 16 * PIECES && lane >= 16 * PIECES) continue;
    const int row = (q * 64 + lane) / PIECES, col = ((lane % PIECES) ^ (row & (PIECES - 1))) * V;
    const Pack<Raw, V> piece = *reinterpret_cast<const Pack<Raw, V> *>(rows + (q * 64 + lane) * V);
    Raw *p = at(row);
    if (!p) continue;
    if (col + V <= count) {
      *reinterpret_cast<Pack<Raw, V> *>(p + col) = piece;
    } else {
#pragma unroll
      for (int e = 0; e < V - 1; e++)
        if (col + e < count) p[col + e] = piece.v[e];
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---- finding the work ----------------------------------------------------------------------------
// First row of group g; entries that are out of order or range never lead outside [0, rows].
__device__ inline int group_begin(const int *ptr, int g, int rows) {
  return g == 0 ? 0 : min(max(ptr[g], 0), rows);
}

// The row tile of a slot: false if the slot is empty.  g == n_groups: rows of no group.  The
// thread that holds a bound hands it on through LDS: reading ptr again would put another memory
// latency in front of every tile.
template <int THREADS>
__device__ inline bool tile_of_slot(const int *ptr, int n_groups, int rows, int tile_rows, int slot,
                                    int *g, int *first, int *end, int *tile) {
  __shared__ int bounds[2];
  int before = 0, mine = 0;
  for (int base = 1; base <= n_groups; base += THREADS) {
    const int j = base + (int)threadIdx.x;
    mine = j <= n_groups ? group_begin(ptr, j, rows) : rows;
    before += __syncthreads_count(j <= n_groups && mine / tile_rows + j <= slot);
  }
  int p0 = 0, p1 = rows;
  if (n_groups <= THREADS) {
    if ((int)threadIdx.x + 1 == before) bounds[0] = mine;
    if ((int)threadIdx.x == before) bounds[1] = mine;       // (rows, behind the last group)
    __syncthreads();
    if (before > 0) p0 = bounds[0];
    if (before < n_groups) p1 = bounds[1];
  } else {
    p0 = group_begin(ptr, before, rows);
    if (before < n_groups) p1 = group_begin(ptr, before + 1, rows);
  }
  *tile = slot - (p0 / tile_rows + before);
  *g = before;
  *first = p0 + *tile * tile_rows;
  *end = p1;
  return *tile >= 0 && *first < *end;
}

// Workgroups go round-robin over the 8 XCDs; this gives each XCD a contiguous range of the work,
// so that the column tiles of a row tile meet in one L2.
__device__ inline int xcd_contiguous(int block, int blocks) {
  const int xcd = block & 7, per = blocks >> 3, rem = blocks & 7;
  return xcd * per + min(xcd, rem) + (block >> 3);
}

// The same where the work comes in units of unequal length, `tiles` workgroups each: unit u goes to
// XCD u % 8, so that no XCD gets the long ones.  -1: behind the last unit.
__device__ inline int xcd_spread(int block, int units, int tiles) {
  const int at = block >> 3, unit = (at / tiles) * 8 + (block & 7);
  return unit < units ? unit * tiles + at % tiles : -1;
}

// A row number of `order`, -1 (and reported) outside the matrix.
__device__ inline int row_at(const int *order, int r, int rows, int *err) {
  const int id = order ? order[r] : r;
  if ((unsigned)id < (unsigned)rows) return id;
  *err = 1;
  return -1;
}

// The row numbers of a tile, thread t's of row t: -1 behind the group's last row and (reported)
// outside the matrix.
template <int BM>
__device__ inline void put_row_ids(int *row_ids, int mine, int first, int end, const GroupedArgs &a) {
  const int t = threadIdx.x;
  if (t < BM) {
    const bool inside = (unsigned)mine < (unsigned)a.rows;
    if (!inside && first + t < end) *a.err = 1;
    row_ids[t] = inside && first + t < end ? mine : -1;
  }
  __syncthreads();
}

// Results of a wave's blocks, with the bias, into the rows of Y.
template <int D> struct RowsOut {
  typedef typename Type<D>::Raw Raw;
  const GroupedArgs &a;
  const int g;
  __device__ f4 bias_at(int n) const {
    f4 b = {0.f, 0.f, 0.f, 0.f};
    if (a.bias && g < a.n_groups) {
      const Raw *p = static_cast<const Raw *>(a.bias) + (long long)g * a.ld_bias + n;
#pragma unroll
      for (int e = 0; e < 4; e++) b[e] = n + e < a.n ? raw_to_float<D>(p[e]) : 0.f;
    }
    return b;
  }
  __device__ void put(int id, int n, f4 v) const {
    const f4 b = bias_at(n);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] += b[e];
    put_results<D>(a.y, (long long)id * a.ldy + n, a.n - n, v);
  }
  template <int MI, int NJ>
  __device__ __forceinline__ void put_all(const f4 (&acc)[MI][NJ], const int *ids, int n_first,
                                          unsigned short *scratch) const {
    f4 b[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) b[j] = bias_at(n_first + 16 * j + 4 * (((int)threadIdx.x >> 4) & 3));
#pragma unroll
    for (int i = 0; i < MI; i++) {
      f4 v[NJ];
#pragma unroll
      for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) v[j][e] = acc[i][j][e] + b[j][e];
      put_rows<D, NJ>(scratch, v, a.n - n_first, [&](int row) -> Raw * {
        const int id = ids[16 * i + row];
        return id < 0 ? nullptr : static_cast<Raw *>(a.y) + (long long)id * a.ldy + n_first;
      });
    }
  }
};

// ---- Y = X W + b -----------------------------------------------------------------------------------
template <int D, int BM, int BN, int WM, int WN, bool TRANS_W, int STAGES, int FLIGHT>
__global__ __launch_bounds__(64 * WM * WN, BM == 64 && D == INCAGG_DTYPE_F32 ? 4 : 2)
void grouped_rows_kernel(const GroupedArgs a) {
  typedef typename Type<D>::Raw Raw;
  constexpr int T = 64 * WM * WN, BK = Type<D>::BK, P = Type<D>::P;
  constexpr int MI = BM / WM / 16, NJ = BN / WN / 16;
  __shared__ __align__(16) unsigned short tiles[STAGES * P * (BM + BN) * BK];
  unsigned short *const xt = tiles, *const wt = tiles + STAGES * P * BM * BK;
  static_assert(WM * WN * kRowScratch<D, NJ> <= STAGES * P * (BM + BN) * BK, "space for the results");
  __shared__ int row_ids[BM];
  const int work = xcd_contiguous(blockIdx.x, gridDim.x);
  const int slot = work / a.n_tiles, n0 = (work - slot * a.n_tiles) * BN;
  int g, first, end, tile;
  if (!tile_of_slot<T>(a.ptr, a.n_groups, a.rows, BM, slot, &g, &first, &end, &tile)) return;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int row0 = (wave / WN) * (BM / WM), col0 = (wave % WN) * (BN / WN);
  static_assert(BM <= T, "a row number to a thread");
  const int my_row = a.order && tid < BM ? a.order[min(first + tid, end - 1)] : first + tid;

  f4 acc[MI][NJ] = {};
  const Raw *x = static_cast<const Raw *>(a.x);
  const Raw *w = static_cast<const Raw *>(a.w) + (long long)g * a.w_group;
  if (g < a.n_groups) {
    // (rows and columns outside the matrices repeat one inside; their results are dropped)
    RowStage<D, BM, T> xs[FLIGHT];
    RowStage<D, TRANS_W ? BN : 16, T> wr[FLIGHT];
    ColStage<D, TRANS_W ? T * 8 / BK : BN, T> wc[FLIGHT];
    if constexpr (TRANS_W)
#pragma unroll
      for (int f = 0; f < FLIGHT; f++)
        wr[f].init([&](int c) { return w + (long long)min(n0 + c, a.n - 1) * a.ldw; });
    const int n_chunks = (a.k + BK - 1) / BK;
    if constexpr (!TRANS_W)
#pragma unroll
      for (int f = 0; f < FLIGHT; f++) wc[f].init(n0, a.n);
    auto load_w = [&](int c, int f) __attribute__((always_inline)) {
      const int k0 = c * BK;
      if constexpr (TRANS_W) {
        if (k0 + BK <= a.k) wr[f].load(k0);
        else wr[f].load_tail(k0, a.k);
      } else {
        const int r0 = k0 + wc[f].row();
        if (k0 + BK <= a.k) {
          const Raw *p = w + (long long)r0 * a.ldw;
          wc[f].load(a.n, [&](int i) { return p + i * a.ldw; });
        } else {
          wc[f].load(a.n, [&](int i) { return w + (long long)min(r0 + i, a.k - 1) * a.ldw; });
          wc[f].clear_from(a.k - r0);
        }
      }
    };
    auto load_x = [&](int c, int f) __attribute__((always_inline)) {
      if (c * BK + BK <= a.k) xs[f].load(c * BK);
      else xs[f].load_tail(c * BK, a.k);
    };
    auto load = [&](int c, int f) __attribute__((always_inline)) {
      load_x(c, f);
      load_w(c, f);
    };
    auto store = [&](int c, int s, int f) __attribute__((always_inline)) {
      xs[f].settle(a.k - c * BK, a.k);
      xs[f].store(xt + s * P * BM * BK);
      if constexpr (TRANS_W) {
        wr[f].settle(a.k - c * BK, a.k);
        wr[f].store(wt + s * P * BN * BK);
      } else {
        wc[f].settle();
        wc[f].store(wt + s * P * BN * BK);
      }
    };
    // (the first weights are on their way while the row numbers arrive, which the rows wait for)
#pragma unroll
    for (int f = 0; f < FLIGHT; f++)
      if (f < n_chunks) load_w(f, f);
    put_row_ids<BM>(row_ids, my_row, first, end, a);
#pragma unroll
    for (int f = 0; f < FLIGHT; f++) {
      xs[f].init([&](int r) { return x + (long long)max(row_ids[r], 0) * a.ldx; });
      if (f < n_chunks) load_x(f, f);
    }
    if constexpr (STAGES == 2) {
      for (int c0 = 0; c0 < n_chunks; c0 += (FLIGHT > 1 ? FLIGHT : 2))
#pragma unroll
        for (int u = 0; u < (FLIGHT > 1 ? FLIGHT : 2); u++) {
          const int c = c0 + u;
          if (c >= n_chunks) break;
          // (the other buffer may still be read; this one was read before the last barrier)
          store(c, u & 1, u % FLIGHT);
          __syncthreads();
          if (c + FLIGHT < n_chunks) load(c + FLIGHT, u % FLIGHT);
          multiply<D, BM, BN>(xt + (u & 1) * P * BM * BK, wt + (u & 1) * P * BN * BK, row0, col0, acc);
        }
    } else {
      static_assert(FLIGHT == 1, "one buffer, one chunk on its way");
      for (int c = 0; c < n_chunks; c++) {
        if (c > 0) __syncthreads();
        store(c, 0, 0);
        __syncthreads();
        if (c + 1 < n_chunks) load(c + 1, 0);
        multiply<D, BM, BN>(xt, wt, row0, col0, acc);
      }
    }
  } else {
    put_row_ids<BM>(row_ids, my_row, first, end, a);
  }
  const RowsOut<D> out{a, g};
  const int lane = tid & 63;
  if constexpr (D == INCAGG_DTYPE_F32) {
    const int columns = a.n - (n0 + col0 + 4 * (lane >> 4));
    const bool finite = all_finite(acc, columns, [&](int i) __attribute__((always_inline)) {
      return row_ids[row0 + 16 * i + (lane & 15)] >= 0;
    });
    if (g < a.n_groups && __syncthreads_or(!finite)) {
      // (a value that does not split, or a result out of range: plain multiply-adds)
      for (int ij = 0; ij < MI * NJ; ij++) {
        const int id = row_ids[row0 + 16 * (ij / NJ) + (lane & 15)];
        const int n = n0 + col0 + 16 * (ij % NJ) + 4 * (lane >> 4);
        if (id < 0 || n >= a.n) continue;
        f4 v;
        for (int e = 0; e < 4; e++) {
          const int c = min(n + e, a.n - 1);
          const Raw *px = x + (long long)id * a.ldx;
          const Raw *pw = TRANS_W ? w + (long long)c * a.ldw : w + c;
          const long long step = TRANS_W ? 1 : a.ldw;
          float s = 0.f;
          for (int k = 0; k < a.k; k++) s = fmaf(px[k], pw[k * step], s);
          v[e] = s;
        }
        out.put(id, n, v);
      }
      return;
    }
    unscale(acc);
  }
  __syncthreads();                       // (the tiles are read no more)
  out.put_all(acc, row_ids + row0, n0 + col0, tiles + wave * kRowScratch<D, NJ>);
}

// ---- D_g = sum A^T B ---------------------------------------------------------------------------------
// A group's rows are cut into segments of `segment` rows; a group of one segment writes its D
// itself (an empty one zeros), the segments of a longer one leave float32 partials that a second
// launch adds up in order.  Partials of group g start at 3 ptr[g] / segment: a group of n > segment
// rows has at most 3 n / segment - 1 segments, so no two groups meet.
__device__ inline long long partial_at(const int *ptr, int g, int rows, int segment, int tile) {
  return 3ll * group_begin(ptr, g, rows) / segment + tile;
}

// Results of a wave's blocks into D_g, or into the segment's partial.
template <int D> struct TnOut {
  const TnArgs &t;
  const int g, seg;
  const bool whole;
  __device__ float *partial() const {
    const long long part = (long long)t.m * t.n + (t.sums ? t.m : 0);
    return t.partials + partial_at(t.ptr, g, t.rows, t.segment, seg) * part;
  }
  __device__ void put(int m, int n, f4 v) const {
    const long long e = (long long)m * t.n + n;
    if (whole) put_results<D>(t.d, g * t.d_group + e, t.n - n, v);
    else put_results<INCAGG_DTYPE_F32>(partial(), e, t.n - n, v);
  }
  __device__ void put_sum(int m, float s) const {
    const f4 v = {s, 0.f, 0.f, 0.f};
    if (whole) put_results<D>(t.sums, (long long)g * t.m + m, 1, v);
    else partial()[(long long)t.m * t.n + m] = s;
  }
  template <int MI, int NJ>
  __device__ __forceinline__ void put_all(const f4 (&acc)[MI][NJ], int m_first, int n_first,
                                          unsigned short *scratch) const {
    typedef typename Type<D>::Raw Raw;
    if (n_first >= t.n) return;
#pragma unroll
    for (int i = 0; i < MI; i++) {
      const int m = m_first + 16 * i;
      if (whole)
        put_rows<D, NJ>(scratch, acc[i], t.n - n_first, [&](int row) -> Raw * {
          return m + row < t.m ? static_cast<Raw *>(t.d) + g * t.d_group + (long long)(m + row) * t.n +
                                     n_first : nullptr;
        });
      else
        put_rows<INCAGG_DTYPE_F32, NJ>(scratch, acc[i], t.n - n_first, [&](int row) -> float * {
          return m + row < t.m ? partial() + (long long)(m + row) * t.n + n_first : nullptr;
        });
    }
  }
};

template <int D, int BM, int BN>
__global__ __launch_bounds__(256, 2) void grouped_tn_kernel(const TnArgs t) {
  typedef typename Type<D>::Raw Raw;
  constexpr int T = 256, BK = Type<D>::BK, P = Type<D>::P;
  constexpr int MI = BM / 32, NJ = BN / 32;
  constexpr int TILES = P * (BM + BN) * BK;
  static_assert(4 * kRowScratch<INCAGG_DTYPE_F32, NJ> <= TILES, "space for the results");
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
  const int last = first + min(end - first, t.segment);      // (first + segment may pass 2^31)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row0 = (wave >> 1) * (BM / 2), col0 = (wave & 1) * (BN / 2);
  const Raw *a = static_cast<const Raw *>(t.a), *b = static_cast<const Raw *>(t.b);
  const bool want_sums = t.sums && n0 == 0;

  f4 acc[MI][NJ] = {};
  ColStage<D, BM, T> as;
  ColStage<D, BN, T> bs;
  float sums[decltype(as)::V] = {};
  // (copies: captured as members of the argument, they would be read from memory in the loop)
  const int *const order = t.order;
  const long long lda = t.lda, ldb = t.ldb;
  const unsigned last_row = t.rows - 1u;
  const int width_a = t.m, width_b = t.n;
  as.init(m0, t.m);
  bs.init(n0, t.n);
  // row numbers of a chunk are fetched one chunk ahead of its rows
  typedef int Ids __attribute__((ext_vector_type(8)));
  Ids ia, ib;
  auto fetch_ids = [&](int r0) __attribute__((always_inline)) {
    if (!order) return;
    if (r0 + BK <= last) {
      ia = __builtin_bit_cast(Ids, *reinterpret_cast<const Pack<int, 8> *>(order + r0 + as.row()));
      ib = __builtin_bit_cast(Ids, *reinterpret_cast<const Pack<int, 8> *>(order + r0 + bs.row()));
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        ia[i] = order[min(r0 + as.row() + i, last - 1)];
        ib[i] = order[min(r0 + bs.row() + i, last - 1)];
      }
    }
  };
  auto load = [&](int r0) __attribute__((always_inline)) {
    const int ra = r0 + as.row(), rb = r0 + bs.row();
    // (rows behind the last repeat it, row numbers outside the matrix its last row: cleared below)
    if (order) {
      as.load(width_a, [&](int i) { return a + (long long)min((unsigned)ia[i], last_row) * lda; });
      bs.load(width_b, [&](int i) { return b + (long long)min((unsigned)ib[i], last_row) * ldb; });
    } else {
      const int la = last - 1 - ra, lb = last - 1 - rb;
      const Raw *pa = a + (long long)min(ra, last - 1) * lda, *pb = b + (long long)min(rb, last - 1) * ldb;
      as.load(width_a, [&](int i) { return i <= la ? pa + i * lda : pa; });
      bs.load(width_b, [&](int i) { return i <= lb ? pb + i * ldb : pb; });
    }
    if (r0 + BK > last) {
      as.clear_from(last - ra);
      bs.clear_from(last - rb);
    }
    if (order) {      // rows of no matrix: zeros, and reported
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 8; i++)
        bad |= (unsigned)ia[i] > last_row || (unsigned)ib[i] > last_row;
      if (bad) {
        *t.err = 1;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          as.clear_row(i, (unsigned)ia[i] <= last_row);
          bs.clear_row(i, (unsigned)ib[i] <= last_row);
        }
      }
    }
    if (r0 + BK < last) fetch_ids(r0 + BK);
  };
  if (first < last) {
    fetch_ids(first);
    load(first);
    for (int r0 = first; r0 < last; r0 += BK) {
      if (r0 > first) __syncthreads();
      as.settle();
      bs.settle();
      as.store(at);
      bs.store(bt);
      if (want_sums)
#pragma unroll
        for (int e = 0; e < decltype(as)::V; e++) {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < 8; i++) s += raw_to_float<D>(as.r[i][e]);
          sums[e] += s;
        }
      __syncthreads();
      if (r0 + BK < last) load(r0 + BK);
      multiply<D, BM, BN>(at, bt, row0, col0, acc);
    }
  }
  const TnOut<D> out{t, g, seg, whole};
  bool again = false;
  if constexpr (D == INCAGG_DTYPE_F32) {
    const int columns = t.n - (n0 + col0 + 4 * (lane >> 4)), left = t.m - (m0 + row0 + (lane & 15));
    again = __syncthreads_or(!all_finite(acc, columns, [&](int i) __attribute__((always_inline)) {
      return 16 * i < left;
    }));
  }
  if (again) {          // (a value that does not split, or a result out of range)
    for (int ij = 0; ij < MI * NJ; ij++) {
      const int m = m0 + row0 + 16 * (ij / NJ) + (lane & 15);
      const int n = n0 + col0 + 16 * (ij % NJ) + 4 * (lane >> 4);
      if (m >= t.m || n >= t.n) continue;
      f4 v = {0.f, 0.f, 0.f, 0.f};
      for (int r = first; r < last; r++) {
        const int id = row_at(t.order, r, t.rows, t.err);
        if (id < 0) continue;
        const float am = raw_to_float<D>(a[(long long)id * t.lda + m]);
        const Raw *pb = b + (long long)id * t.ldb;
        for (int e = 0; e < 4; e++)
          v[e] = fmaf(am, raw_to_float<D>(pb[min(n + e, t.n - 1)]), v[e]);
      }
      out.put(m, n, v);
    }
  } else {
    if constexpr (D == INCAGG_DTYPE_F32) unscale(acc);
    __syncthreads();                     // (the tiles are read no more)
    out.put_all(acc, m0 + row0, n0 + col0, tiles + wave * kRowScratch<INCAGG_DTYPE_F32, NJ>);
  }
  if (!want_sums) return;
  // column sums: threads of one column group, row groups in order
  constexpr int V = decltype(as)::V, RG = BK / 8;
  static_assert(sizeof(float) * RG * BM <= sizeof(tiles), "reduction space");
  float *red = reinterpret_cast<float *>(tiles);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < V; e++) red[(as.row() / 8) * BM + as.col() + e] = sums[e];
  __syncthreads();
  for (int c = tid; c < BM && m0 + c < t.m; c += T) {
    float s = 0.f;
    for (int r = 0; r < RG; r++) s += red[r * BM + c];
    out.put_sum(m0 + c, s);
  }
}

// ---- 16-bit types at full speed: tiles that go from memory into LDS by themselves ----------------------
// The kernels above pass every tile through registers, which lets them take any alignment and
// split float32.  For 16-bit operands whose rows are 16-byte aligned the loads write LDS directly
// (global_load_lds, 16 bytes a lane, 1 KB an instruction, in lane order), without registers or
// stores.  The LDS image of a chunk (32 values along k) keeps the layout of the matrix:
//   K-contiguous operand: [row][32 k], 64 bytes a row; piece c of row r lies at c ^ (r / 4 % 4).  A
//     fragment is one 16-byte read.
//   K-strided operand: [k][EXT columns]; the 32-byte segment s of row k lies at s ^ f(k), f(k) =
//     k % 4 + 4 (k / 8 % 2).  A fragment is two transposing reads (ds_read_b64_tr_b16: 16 lanes
//     name 4 rows x 16 columns, lane i gets column i): the 32 lanes of a read phase touch rows
//     0..3 and 8..11 of a 16-row block, which f spreads over all 64 banks.
// The permutation is applied where it is free, to the address each lane loads from (bank conflicts
// take 4 to 7 % of the LDS cycles, those of the results' way out, put_rows, included).  What lies past
// the end of the reduction is loaded
// from 16 bytes of zeros.
//
// Two buffers and one barrier a chunk.  Fragments are read AHEAD row blocks before they are
// multiplied, so AHEAD blocks before the end of chunk c everything of it is in registers: there the
// wave waits for the loads of chunk c + 1, meets the others, sends off the loads of c + 2 into the
// buffer of c and reads the first fragments of c + 1, while the matrix cores work off the last
// blocks of c.
constexpr int kDepth = 64;
__device__ const u4 g_zeros = {0u, 0u, 0u, 0u};

// The instruction has no result register, and its address registers are read when it issues.  (As
// a builtin, the compiler makes the next LDS read wait for it, whichever buffer that one reads.)
// m0: where in LDS lane 0's piece goes; put there by the compiler, which then knows what m0 holds.
__device__ inline void load_to_lds(const void *src, unsigned lds_byte) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "{m0}"(lds_byte), "v"(src) : "memory");
}

// Waits for this wave's loads into LDS; with a barrier behind it, for everybody's.
__device__ inline void loads_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ inline unsigned lds_byte(const unsigned short *p) {
  return (unsigned)(unsigned long long)(const __attribute__((address_space(3))) unsigned short *)p;
}

// Loads of one operand's chunks: wave `wave` of WAVES issues PER instructions for its rows.
template <bool STRIDED, int EXT, int WAVES> struct LdsTile {
  static constexpr int PIECES = STRIDED ? EXT / 8 : kDepth / 8;   // 16-byte pieces of an image row
  static constexpr int ROWS = 64 / PIECES;                        // image rows of an instruction
  static constexpr int PER = (STRIDED ? kDepth : EXT) / ROWS / WAVES;
  static constexpr int SIZE = EXT * kDepth;
  static_assert(PER >= 1 && (PER * ROWS * WAVES == (STRIDED ? kDepth : EXT)), "whole instructions");
  // image row that this lane loads a piece of, and which piece of the matrix's row goes there
  static __device__ int row(int wave, int i) {
    return (wave * PER + i) * ROWS + ((int)threadIdx.x & 63) / PIECES;
  }
  static __device__ int piece(int row) {
    const int at = ((int)threadIdx.x & 63) % PIECES;
    if constexpr (STRIDED) return at ^ (2 * ((row & 3) | ((row >> 3) & 1) << 2));
    else return at ^ (row & 7);
  }
};

typedef short s4 __attribute__((ext_vector_type(4)));
__device__ inline s4 read_transposed(const unsigned short *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s4 *)const_cast<unsigned short *>(p));
}

// Where this lane's part of a fragment lies: of the fragment at the operand's column (or row) 0.
template <bool STRIDED, int EXT> __device__ __forceinline__ int fragment_base() {
  const int l16 = threadIdx.x & 15, quad = (threadIdx.x >> 4) & 3;
  if constexpr (STRIDED)
    return (quad * 8 + (l16 >> 2)) * EXT + (((l16 >> 2) | (quad & 1) << 2) << 4) + (l16 & 3) * 4;
  else
    return l16 * kDepth + ((quad ^ (l16 & 7)) << 3);
}

// Fragment of the 16 rows (columns, for a strided operand) from `first` on, k = 32 kk ..
template <bool STRIDED, int EXT>
__device__ __forceinline__ u4 fragment(const unsigned short *tile, int base, int first, int kk) {
  if constexpr (STRIDED) {
    const unsigned short *p = tile + (base ^ first) + kk * 32 * EXT;    // (segment s ^ f(k))
    struct { s4 lo, hi; } r = {read_transposed(p), read_transposed(p + 4 * EXT)};
    return __builtin_bit_cast(u4, r);
  } else {
    return *reinterpret_cast<const u4 *>(tile + (base ^ (kk << 5)) + first * kDepth);
  }
}

// The pipeline over the chunks of one tile.  load(s): issues the loads of the next chunk, into
// buffer s.
template <int D, bool ROWS_STRIDED, bool COLS_STRIDED, int BM, int BN, int WM, int WN>
struct LdsPipeline {
  static constexpr int WAVES = WM * WN, MI = BM / WM / 16, NJ = BN / WN / 16;
  static constexpr int AHEAD = 2, RING = 4, STEPS = 2 * MI;
  static_assert(STEPS % RING == 0 && AHEAD < RING && MI >= NJ && NJ % AHEAD == 0, "fragment schedule");
  typedef LdsTile<ROWS_STRIDED, BM, WAVES> Rows;
  typedef LdsTile<COLS_STRIDED, BN, WAVES> Cols;
  static constexpr int CHUNK = Rows::SIZE + Cols::SIZE;         // values of a buffer
  f4 acc[MI][NJ];

  template <typename Load, typename Extra>
  __device__ __forceinline__ void run(const unsigned short *tiles, int n_chunks, int row0, int col0,
                                      Load &&load, Extra &&extra) {
    u4 a[RING], b[2][NJ];
    // (the wave's first row goes into the address, the block within the wave is a constant)
    int ra = fragment_base<ROWS_STRIDED, BM>(), ca = fragment_base<COLS_STRIDED, BN>();
    ra = ROWS_STRIDED ? ra ^ row0 : ra + row0 * kDepth;
    ca = COLS_STRIDED ? ca ^ col0 : ca + col0 * kDepth;
    const auto rows_at = [&](const unsigned short *tile, int i, int kk) __attribute__((always_inline)) {
      return fragment<ROWS_STRIDED, BM>(tile, ra, 16 * i, kk);
    };
    const auto cols_at = [&](const unsigned short *tile, int j, int kk) __attribute__((always_inline)) {
      return fragment<COLS_STRIDED, BN>(tile + Rows::SIZE, ca, 16 * j, kk);
    };
    load(0);
    loads_landed();
    __syncthreads();
    if (n_chunks > 1) load(1);
#pragma unroll
    for (int j = 0; j < NJ; j++) b[0][j] = cols_at(tiles, j, 0);
#pragma unroll
    for (int t = 0; t < AHEAD; t++) a[t] = rows_at(tiles, t, 0);
    for (int c = 0; c < n_chunks; c++) {
      const unsigned short *tile = tiles + (c & 1) * CHUNK, *after = tiles + (~c & 1) * CHUNK;
      asm volatile("" : "+v"(ra), "+v"(ca));    // (an address per block would not fit the registers)
#pragma unroll
      for (int t = 0; t < STEPS; t++) {
        const int next = t + AHEAD;
        if (t == STEPS - AHEAD) {       // (behind the last chunk: fragments are read, not used)
          loads_landed();
          __syncthreads();
          if (c + 2 < n_chunks) load(c & 1);
        }
        a[next % RING] = next < STEPS ? rows_at(tile, next % MI, next / MI)
                                      : rows_at(after, next - STEPS, 0);
        if (t >= MI - NJ && t < MI) b[1][t - (MI - NJ)] = cols_at(tile, t - (MI - NJ), 1);
        if (t >= STEPS - AHEAD)
#pragma unroll
          for (int j = 0; j < NJ / AHEAD; j++)
            b[0][(t - (STEPS - AHEAD)) * (NJ / AHEAD) + j] =
                cols_at(after, (t - (STEPS - AHEAD)) * (NJ / AHEAD) + j, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < NJ; j++)
          acc[t % MI][j] = mfma<D>(b[t / MI][j], a[t % RING], acc[t % MI][j]);
        extra(t % MI, a[t % RING]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

template <int D, int BM, int BN, int WM, int WN, bool TRANS_W>
__global__ __launch_bounds__(64 * WM * WN, 2) void grouped_rows_lds_kernel(const GroupedArgs a) {
  constexpr int T = 64 * WM * WN;
  typedef LdsPipeline<D, false, !TRANS_W, BM, BN, WM, WN> Pipe;
  typedef typename Pipe::Rows X;
  typedef typename Pipe::Cols W;
  __shared__ __align__(1024) unsigned short tiles[2 * Pipe::CHUNK];
  __shared__ int row_ids[BM];
  const int work = xcd_contiguous(blockIdx.x, gridDim.x);
  const int slot = work / a.n_tiles, n0 = (work - slot * a.n_tiles) * BN;
  int g, first, end, tile;
  if (!tile_of_slot<T>(a.ptr, a.n_groups, a.rows, BM, slot, &g, &first, &end, &tile)) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row0 = (wave / WN) * (BM / WM), col0 = (wave % WN) * (BN / WN);
  static_assert(BM <= T, "a row number to a thread");
  put_row_ids<BM>(row_ids, a.order && tid < BM ? a.order[min(first + tid, end - 1)] : first + tid,
                  first, end, a);

  Pipe pipe{};
  if (g < a.n_groups) {
    const unsigned short *x = static_cast<const unsigned short *>(a.x);
    const unsigned short *w = static_cast<const unsigned short *>(a.w) + (long long)g * a.w_group;
    // what lies outside the matrices repeats something inside; those results are dropped
    const unsigned short *px[X::PER], *pw[W::PER];
    int kx[X::PER], kw[W::PER];         // where along k the lane's piece (or row) is
#pragma unroll
    for (int i = 0; i < X::PER; i++) {
      const int r = X::row(wave, i);
      kx[i] = X::piece(r) * 8;
      px[i] = x + (long long)max(row_ids[r], 0) * a.ldx + kx[i];
    }
#pragma unroll
    for (int i = 0; i < W::PER; i++) {
      const int r = W::row(wave, i);
      if constexpr (TRANS_W) {
        kw[i] = W::piece(r) * 8;
        pw[i] = w + (long long)min(n0 + r, a.n - 1) * a.ldw + kw[i];
      } else {
        kw[i] = r;
        pw[i] = w + (long long)r * a.ldw + min(n0 + W::piece(r) * 8, a.n - 8);
      }
    }
    const long long w_step = TRANS_W ? kDepth : kDepth * a.ldw;
    const unsigned base = __builtin_amdgcn_readfirstlane(lds_byte(tiles));
    int left = a.k;                     // of the reduction, from the next chunk on
    auto load = [&](int s) __attribute__((always_inline)) {
      const unsigned to = base + s * Pipe::CHUNK * 2 + wave * X::PER * 1024;
      const unsigned wo = base + s * Pipe::CHUNK * 2 + X::SIZE * 2 + wave * W::PER * 1024;
      if (left >= kDepth) {
#pragma unroll
        for (int i = 0; i < X::PER; i++) load_to_lds(px[i], to + i * 1024);
#pragma unroll
        for (int i = 0; i < W::PER; i++) load_to_lds(pw[i], wo + i * 1024);
      } else {
#pragma unroll
        for (int i = 0; i < X::PER; i++)
          load_to_lds(kx[i] < left ? (const void *)px[i] : (const void *)&g_zeros, to + i * 1024);
#pragma unroll
        for (int i = 0; i < W::PER; i++)
          load_to_lds(kw[i] < left ? (const void *)pw[i] : (const void *)&g_zeros, wo + i * 1024);
      }
#pragma unroll
      for (int i = 0; i < X::PER; i++) px[i] += kDepth;
#pragma unroll
      for (int i = 0; i < W::PER; i++) pw[i] += w_step;
      left -= kDepth;
    };
    pipe.run(tiles, (a.k + kDepth - 1) / kDepth, row0, col0, load, [](int, u4) {});
  }
  const RowsOut<D> out{a, g};
  __syncthreads();                       // (the tiles are read no more)
  out.put_all(pipe.acc, row_ids + row0, n0 + col0, tiles + wave * kRowScratch<D, Pipe::NJ>);
}

// D_g over one segment; the column sums of A come from the matrix cores too, as one more column
// block of ones (exact products, the same float32 sums).  Row numbers come through the scalar
// cache: a vector load of them would have to be waited for, and with it all tile loads behind it.
template <int D, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void grouped_tn_lds_kernel(const TnArgs t) {
  constexpr int T = 64 * WM * WN;
  typedef LdsPipeline<D, true, true, BM, BN, WM, WN> Pipe;
  typedef typename Pipe::Rows A;
  typedef typename Pipe::Cols B;
  static_assert(A::PER * A::ROWS == B::PER * B::ROWS, "a wave loads the same rows of both");
  constexpr int WAVE_ROWS = A::PER * A::ROWS;
  __shared__ __align__(1024) unsigned short tiles[2 * Pipe::CHUNK];
  // (segments of different length: 131072 rows in 16 groups, 1024 x 2048, contiguous / spread 823 / 725 us,
  // 65536 rows in one, 2048 x 2048 1107 / 640; a unit is a row of tiles, which share their part of A)
  const int work = xcd_spread(blockIdx.x, t.slots * t.m_tiles, t.n_tiles);
  if (work < 0) return;
  const int per_slot = t.m_tiles * t.n_tiles, slot = work / per_slot, mn = work - slot * per_slot;
  const int m0 = (mn / t.n_tiles) * BM, n0 = (mn % t.n_tiles) * BN;
  int g, first, end, seg;
  const bool any = tile_of_slot<T>(t.ptr, t.n_groups, t.rows, t.segment, slot, &g, &first, &end, &seg);
  if (g >= t.n_groups || seg < 0 || (!any && seg > 0)) return;
  g = __builtin_amdgcn_readfirstlane(g);
  const int begin = group_begin(t.ptr, g, t.rows);
  const bool whole = end - begin <= t.segment;       // the group's only segment (or an empty group)
  const int last = __builtin_amdgcn_readfirstlane(first + min(end - first, t.segment));
  first = __builtin_amdgcn_readfirstlane(first);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row0 = (wave / WN) * (BM / WM), col0 = (wave % WN) * (BN / WN);
  const bool want_sums = t.sums && n0 == 0 && col0 == 0;

  // the columns each lane's pieces begin at (instructions i and i + 2: the same piece)
  constexpr int CA = A::PER < 2 ? A::PER : 2, CB = B::PER < 2 ? B::PER : 2;
  int ca[CA], cb[CB];
#pragma unroll
  for (int i = 0; i < CA; i++) ca[i] = min(m0 + A::piece(A::row(wave, i)) * 8, t.m - 8);
#pragma unroll
  for (int i = 0; i < CB; i++) cb[i] = min(n0 + B::piece(B::row(wave, i)) * 8, t.n - 8);
  const auto *order = (const __attribute__((address_space(4))) int *)t.order;
  int ids[WAVE_ROWS];                   // row numbers of the next chunk to load (-1: zeros)
  int bad = 0;
  int next_row = first + wave * WAVE_ROWS;
  auto fetch_ids = [&]() __attribute__((always_inline)) {
    if (order) {
#pragma unroll
      for (int i = 0; i < WAVE_ROWS; i++)
        ids[i] = __builtin_amdgcn_readfirstlane(order[min(next_row + i, last - 1)]);
#pragma unroll
      for (int i = 0; i < WAVE_ROWS; i++) {
        const int outside = (unsigned)ids[i] >= (unsigned)t.rows;
        bad |= outside;
        ids[i] = next_row + i < last && !outside ? ids[i] : -1;
      }
    } else {
#pragma unroll
      for (int i = 0; i < WAVE_ROWS; i++) ids[i] = next_row + i < last ? next_row + i : -1;
    }
    next_row += kDepth;
  };
  const unsigned base = __builtin_amdgcn_readfirstlane(lds_byte(tiles));
  const int n_chunks = (last - first + kDepth - 1) / kDepth;
  auto load = [&](int s) __attribute__((always_inline)) {
    const unsigned ao = base + s * Pipe::CHUNK * 2 + wave * A::PER * 1024;
    const unsigned bo = base + s * Pipe::CHUNK * 2 + A::SIZE * 2 + wave * B::PER * 1024;
    // row `of` (of this lane) among the wave's rows
    auto id_of = [&](int i, int rows, int of) __attribute__((always_inline)) {
      int id = ids[i * rows];
#pragma unroll
      for (int j = 1; j < rows; j++) id = of == j ? ids[i * rows + j] : id;
      return id;
    };
#pragma unroll
    for (int i = 0; i < A::PER; i++) {
      const int id = id_of(i, A::ROWS, lane / A::PIECES);
      const unsigned short *p = static_cast<const unsigned short *>(t.a) + id * t.lda + ca[i % CA];
      load_to_lds(id < 0 ? (const void *)&g_zeros : (const void *)p, ao + i * 1024);
    }
#pragma unroll
    for (int i = 0; i < B::PER; i++) {
      const int id = id_of(i, B::ROWS, lane / B::PIECES);
      const unsigned short *p = static_cast<const unsigned short *>(t.b) + id * t.ldb + cb[i % CB];
      load_to_lds(id < 0 ? (const void *)&g_zeros : (const void *)p, bo + i * 1024);
    }
    fetch_ids();                        // (behind the last chunk: zeros)
  };

  Pipe pipe{};
  f4 sums[Pipe::MI] = {};
  const u4 ones = D == INCAGG_DTYPE_BF16 ? u4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}
                                         : u4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
  if (first < last) {
    fetch_ids();
    if (want_sums)
      pipe.run(tiles, n_chunks, row0, col0, load,
               [&](int i, u4 a) __attribute__((always_inline)) { sums[i] = mfma<D>(ones, a, sums[i]); });
    else
      pipe.run(tiles, n_chunks, row0, col0, load, [](int, u4) {});
    if (bad) *t.err = 1;
  }
  const TnOut<D> out{t, g, seg, whole};
  __syncthreads();                       // (the tiles are read no more)
  out.put_all(pipe.acc, m0 + row0, n0 + col0,
              tiles + wave * kRowScratch<INCAGG_DTYPE_F32, Pipe::NJ>);
  if (want_sums && lane < 16)
#pragma unroll
    for (int i = 0; i < Pipe::MI; i++) {
      const int m = m0 + row0 + 16 * i + lane;
      if (m < t.m) out.put_sum(m, sums[i][0]);
    }
}

// Partials of groups that were cut into segments, added up: 32 x 4 neighbouring elements to a
// workgroup, every eighth segment to a thread (in order), the eight sums in order.
template <int D> __global__ __launch_bounds__(256) void grouped_tn_finish_kernel(const TnArgs t) {
  __shared__ f4 sums[8][32];
  const int g = blockIdx.y;
  const int begin = group_begin(t.ptr, g, t.rows), end = group_begin(t.ptr, g + 1, t.rows);
  if (end - begin <= t.segment) return;
  const int segments = (end - begin + t.segment - 1) / t.segment;
  const long long mn = (long long)t.m * t.n, part = mn + (t.sums ? t.m : 0);
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  for (long long first = blockIdx.x * 128ll; first < part; first += gridDim.x * 128ll) {
    const long long e = first + lane * 4;
    const float *p = t.partials + partial_at(t.ptr, g, t.rows, t.segment, row) * part + e;
    const int count = (int)max(0ll, min(4ll, part - e));
    f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = row; i < segments; i += 8, p += 8 * part) {
      if (count == 4) {
        const Pack<float, 4> q = *reinterpret_cast<const Pack<float, 4> *>(p);
#pragma unroll
        for (int j = 0; j < 4; j++) s[j] += q.v[j];
      } else {
        for (int j = 0; j < count; j++) s[j] += p[j];
      }
    }
    sums[row][lane] = s;
    __syncthreads();
    if (row == 0 && count > 0) {
#pragma unroll
      for (int i = 1; i < 8; i++) s += sums[i][lane];
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
    __syncthreads();
  }
}

// ---- host side ---------------------------------------------------------------------------------------
constexpr int64_t kMaxThreads = 1ll << 32;       // of a launch

template <int D, int BM, int BN, int WM, int WN, int STAGES, int FLIGHT>
static int launch_rows_tile(GroupedArgs &a, bool trans_w, hipStream_t s) {
  a.n_tiles = (a.n + BN - 1) / BN;
  const int64_t blocks = ((int64_t)a.rows / BM + a.n_groups + 1) * a.n_tiles;
  INCAGG_REQUIRE(blocks * (64 * WM * WN) < kMaxThreads, "too many rows and columns for one call");
  const dim3 grid((unsigned)blocks), block(64 * WM * WN);
  if (trans_w)
    hipLaunchKernelGGL((grouped_rows_kernel<D, BM, BN, WM, WN, true, STAGES, FLIGHT>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((grouped_rows_kernel<D, BM, BN, WM, WN, false, STAGES, FLIGHT>), grid, block, 0, s, a);
  INCAGG_HIP_TRY(hipGetLastError());
  return INCAGG_OK;
}

template <int D, int BM, int BN, int WM, int WN>
static int launch_rows_lds(GroupedArgs &a, bool trans_w, hipStream_t s) {
  a.n_tiles = (a.n + BN - 1) / BN;
  const int64_t blocks = ((int64_t)a.rows / BM + a.n_groups + 1) * a.n_tiles;
  INCAGG_REQUIRE(blocks * (64 * WM * WN) < kMaxThreads, "too many rows and columns for one call");
  const dim3 grid((unsigned)blocks), block(64 * WM * WN);
  if (trans_w)
    hipLaunchKernelGGL((grouped_rows_lds_kernel<D, BM, BN, WM, WN, true>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((grouped_rows_lds_kernel<D, BM, BN, WM, WN, false>), grid, block, 0, s, a);
  INCAGG_HIP_TRY(hipGetLastError());
  return INCAGG_OK;
}

// Rows in whole 16-byte pieces.
static bool pieces(const void *p, int64_t ld, int64_t width) {
  return aligned16(p) && ld % 8 == 0 && width % 8 == 0;
}

// Tiles by the average number of rows to a group: below one tile of rows the weights are what is
// read, and a tall tile is mostly empty.  64 groups, 1024 -> 1024 bfloat16 and 512 -> 512 float32,
// forward, us by rows of a tile (128: the LDS-loading kernel for bfloat16):
//     rows to a group      4     16     32     64    128    256    512
//     bfloat16    16    24.3   28.0   33.5   53.5   86.4    148    283
//                 64    26.1   27.4   28.3   39.1   46.0   70.1    124
//                128    35.8   36.8   37.3   40.2   58.0   60.3   92.8
//     float32     16    21.0   24.7   33.7   49.0   82.0    150    289
//                 64    31.5   30.0   30.9   39.4   47.2   66.3    113
//                128    44.0   43.1   43.6   44.2   46.9   75.8    120     (8192 rows: 941 / 881)
// The average is all the host knows: it counts groups without a row, so many groups of which few are
// used get tiles that are too low.  32768 rows in 8 groups of 8 / 64 / 512 / 2048, 512 -> 512: bfloat16
// 36 / 35 / 61 / 286 us, float32 116 / 123 / 202 / 673.
template <int D> static int launch_rows(GroupedArgs &a, bool trans_w, hipStream_t s) {
  constexpr bool F32 = D == INCAGG_DTYPE_F32;
  constexpr int STAGES = F32 ? 1 : 2;
  const int64_t average = a.rows / a.n_groups;
  if (average <= 16) return launch_rows_tile<D, 16, 64, 1, 4, 2, 4>(a, trans_w, s);
  // one column tile (128 rows / 64 rows, us: float16 23297 x 602 -> 41 16.5 / 13.9, bfloat16 60000 x
  // 100 -> 47 12.3 / 11.4, 200000 x 256 -> 64 31.3 / 31.1, float32 120000 x 128 -> 40 25.4 / 24.5)
  if (a.n <= 64) return launch_rows_tile<D, 64, 64, 2, 2, STAGES, 1>(a, trans_w, s);
  // float32 stays with 64 rows -- more workgroups that take turns between loading, splitting and
  // multiplying -- until there are a dozen 128 x 128 tiles to a CU (65304 x 256 -> 256 and 16326 x 512
  // -> 512: 73 / 65 and 82 / 70 us by 128 / 64 rows; 65536 x 1024 -> 1024: 881 / 941)
  const int64_t large = (int64_t)(a.rows / 128) * ((a.n + 127) / 128);
  if (average <= (F32 ? 768 : 64) || (F32 && large < 3000))
    return launch_rows_tile<D, 64, 128, 2, 2, STAGES, 1>(a, trans_w, s);
  if constexpr (!F32) {
    if (pieces(a.x, a.ldx, a.k) && pieces(a.w, a.ldw, trans_w ? a.k : a.n) && a.w_group % 8 == 0) {
      // 256 x 256 halves what a tile reads for its products, but leaves one workgroup to a CU: for
      // at least one round of them (128 x 128 against it, 131072 x 1024 -> 2048: 848 / 671 us,
      // 32768 x 1024 -> 1024, two rounds: 93 / 90 us)
      const int64_t tiles = ((int64_t)a.rows / 256 + a.n_groups / 2) * ((a.n + 255) / 256);
      if (a.n <= 128 || tiles < 256) return launch_rows_lds<D, 128, 128, 2, 2>(a, trans_w, s);
      return launch_rows_lds<D, 256, 256, 2, 4>(a, trans_w, s);
    }
  }
  return launch_rows_tile<D, 128, 128, 2, 2, STAGES, 1>(a, trans_w, s);
}

// Whether the weight gradient runs in 256 x 256 tiles where the operands' alignment allows it.
static bool tn_large_tiles(int64_t m, int64_t n, int dtype) {
  return dtype != INCAGG_DTYPE_F32 && m > 128 && n > 128;
}

// Rows of a segment: enough segments to fill the chip (one workgroup to a CU of 256 x 256 tiles,
// two of 128 x 128), at least 256 rows.  Shorter ones even out groups of different sizes, but every
// one of a longer group costs a partial written and read (float32, 16326 rows, 256 x 256, 128 / 256 /
// 512 rows: 46 / 41 / 49 us).  A group ends inside a segment, which makes up to one more for each.
// Where a group has many segments (`even`) those would be the few workgroups over a full round that
// cost another one: there they are taken off (without / with, 60000 rows in 5 groups, 512 x 512
// bfloat16 113 / 73 us; 65304 rows in 5 groups, 256 x 256 float32 132 / 93).  Where it has few, short
// last segments make room early (20000 rows in 8 groups, 1024 x 1024 float16 144 / 164).
struct Segments {
  int rows;
  bool even;
};
static Segments tn_segments(int64_t rows, int64_t n_groups, int64_t m, int64_t n, int dtype) {
  const bool large = tn_large_tiles(m, n, dtype);
  const int64_t tile = large ? 256 : 128, tiles = ((m + tile - 1) / tile) * ((n + tile - 1) / tile);
  const int64_t wanted = std::max<int64_t>(1, (large ? 256 : 512) / tiles);
  const bool even = n_groups * 8 <= wanted && rows >= 256 * wanted;
  const int64_t count = even ? wanted - n_groups : wanted;
  const int64_t s = std::max<int64_t>(256, (rows + count - 1) / count);
  return {(int)((s + 63) / 64 * 64), even};
}

// Adds up the partials of groups that were cut into segments.
template <int D> static int tn_finish(TnArgs &t, hipStream_t s) {
  if (t.rows <= t.segment) return INCAGG_OK;
  const int64_t part = (int64_t)t.m * t.n + (t.sums ? t.m : 0);
  hipLaunchKernelGGL(grouped_tn_finish_kernel<D>,
                     dim3((unsigned)std::min<int64_t>((part + 127) / 128, 512), (unsigned)t.n_groups),
                     dim3(256), 0, s, t);
  INCAGG_HIP_TRY(hipGetLastError());
  return INCAGG_OK;
}

template <int D, int BM, int BN> static int launch_tn_tile(TnArgs &t, hipStream_t s) {
  t.m_tiles = (t.m + BM - 1) / BM;
  t.n_tiles = (t.n + BN - 1) / BN;
  const int64_t blocks = ((int64_t)t.rows / t.segment + t.n_groups) * t.m_tiles * t.n_tiles;
  INCAGG_REQUIRE(blocks * 256 < kMaxThreads, "too many rows and columns for one call");
  hipLaunchKernelGGL((grouped_tn_kernel<D, BM, BN>), dim3((unsigned)blocks), dim3(256), 0, s, t);
  INCAGG_HIP_TRY(hipGetLastError());
  return tn_finish<D>(t, s);
}

template <int D, int BM, int BN, int WM, int WN>
static int launch_tn_lds(TnArgs &t, hipStream_t s) {
  t.m_tiles = (t.m + BM - 1) / BM;
  t.n_tiles = (t.n + BN - 1) / BN;
  t.slots = t.rows / t.segment + t.n_groups;
  const int64_t blocks = ((int64_t)t.slots * t.m_tiles + 7) / 8 * 8 * t.n_tiles;
  INCAGG_REQUIRE(blocks * (64 * WM * WN) < kMaxThreads, "too many rows and columns for one call");
  hipLaunchKernelGGL((grouped_tn_lds_kernel<D, BM, BN, WM, WN>), dim3((unsigned)blocks),
                     dim3(64 * WM * WN), 0, s, t);
  INCAGG_HIP_TRY(hipGetLastError());
  return tn_finish<D>(t, s);
}

template <int D> static int launch_tn(TnArgs &t, bool even, hipStream_t s) {
  if constexpr (D != INCAGG_DTYPE_F32) {
    if (tn_large_tiles(t.m, t.n, D) && pieces(t.a, t.lda, t.m) && pieces(t.b, t.ldb, t.n))
      return launch_tn_lds<D, 256, 256, 2, 4>(t, s);
  }
  if (t.n <= 64) return t.m <= 64 ? launch_tn_tile<D, 64, 64>(t, s) : launch_tn_tile<D, 128, 64>(t, s);
  // 128 x 128 tiles load and split less for a product, 64 x 128 leave twice the workgroups to hide
  // what they wait for.  float32, us by 128 / 64: 16326 rows, 256 x 256 46 / 41, even segments: 65304
  // rows, 256 x 256 93 / 110, 100000 rows, 300 x 200 154 / 188; 65536 rows, 1024 x 1024 1114 / 1195, 40000
  // rows in 40 groups, 512 x 512 226 / 210; one column of tiles, 128064 rows, 256 x 100, 83 / 100.
  // 16-bit types always take the narrower: float16 30000 rows, 300 x 601 250 / 74; bfloat16 30000
  // rows, 256 x 100 57 / 23.
  if constexpr (D == INCAGG_DTYPE_F32) {
    const int64_t tiles = (int64_t)((t.m + 127) / 128) * ((t.n + 127) / 128);
    if (t.m > 64 && (t.n <= 128 || even || (t.rows / t.segment + t.n_groups) * tiles >= 800))
      return launch_tn_tile<D, 128, 128>(t, s);
  }
  return launch_tn_tile<D, 64, 128>(t, s);
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
  const int64_t segment = tn_segments(rows, n_groups, m, n, dtype).rows;
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
  const Segments segments = tn_segments(rows, n_groups, m, n, dtype);
  t.segment = segments.rows;
  t.a = a; t.b = b; t.d = d; t.sums = sums; t.lda = lda; t.ldb = ldb; t.d_group = d_group;
  t.ptr = ptr; t.order = order; t.n_groups = (int)n_groups; t.rows = (int)rows;
  t.m = (int)m; t.n = (int)n;
  rc = error_flag_address(&t.err);
  if (rc) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case INCAGG_DTYPE_F32: return launch_tn<INCAGG_DTYPE_F32>(t, segments.even, s);
    case INCAGG_DTYPE_BF16: return launch_tn<INCAGG_DTYPE_BF16>(t, segments.even, s);
    default: return launch_tn<INCAGG_DTYPE_F16>(t, segments.even, s);
  }
}
