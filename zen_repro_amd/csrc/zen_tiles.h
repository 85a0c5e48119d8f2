// Matrix products in tiles, for zen_product.hip and zen_orthogonal.hip.
//
//   D[i, j] = sum over k of A[i, k] B[k, j],   A and B in 16 bits, sums in fp32 (MFMA 32x32x16)
//
// A workgroup owns a tile of D and walks k in steps of 64.  A step's pieces of A and B come straight into LDS (buffer
// loads with an LDS destination, 16 bytes a lane) into buffers that go round, so the loads of the steps ahead are in flight while
// one is multiplied.  Each operand may be stored with k contiguous (rows of k) or with k as the stride (rows of i or j):
// the first is read from LDS 16 bytes a lane, the second by transposing reads (ds_read_b64_tr_b16), so no operand is ever
// transposed in memory.  The range check of the buffer loads puts zeros where the tile hangs over the operand's end.
//
// What bounds it: with 256 x 256 tiles a step's products take a compute unit 2048 cycles, of some 2900 (8192^3, k contiguous:
// matrix cores busy 71 % of the cycles, LDS 20 %, and a clock that the power limit holds at 1.5 to 1.9 GHz: 1200 to 1310
// TFLOP/s; without the loads, 1550).  What mattered most: reads, loads and products in an order of our own, one by one (the
// compiler's: 1.79 against 1.50 million cycles at that size), and reads of LDS without bank conflicts.
//
// LDS layout: a row of 64 k is eight 16-byte pieces; piece c of row r lies in place c ^ key(r).  With k as the stride a row
// holds the tile's i or j, and piece c of row k lies in place(k, c).  Both spread what lanes read at the same time (32 rows at one c;
// four rows of k at two or four neighbouring pieces) over all banks: no conflicts were counted.  The loads' LDS destination is one run
// of lanes, so the order is in the addresses they read from.
#pragma once

#include "zen_common.h"

namespace zen {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kTileK = 64;
constexpr int64_t kMostLd = 1 << 21;  // a step's addresses, 256 rows at most, stay below 2^30
constexpr int kMostList = 32;  // matrices of separate addresses to a launch
constexpr int64_t kMostThreads = 0xffffffffll;  // of a launch: the runtime counts them in 32 bits

struct MatOperand {
  const uint16_t *p[2];  // the matrix, and what its rounding to 16 bits left over (itself where there is nothing: never null)
  int64_t ld;            // elements from row to row
  int64_t batch;         // elements from matrix to matrix
};

struct MatSize {
  int m, n, k;
  int tiles_m, tiles_n;
  int batch;
  int parts;       // 1: A B; 3: A B + A B' + A' B with the left-overs A', B'
  int splits;      // > 1: the steps of a tile are shared among so many workgroups, whose sums go to `partial`
  float *partial;  // and are joined by a launch of their own
};

// Addresses of a stack's matrices: base + b * stride, or a list.
struct MatList {
  char *base;
  int64_t stride;  // bytes
  int listed;
  char *at[kMostList];
  __device__ __forceinline__ char *of(int b) const { return listed ? at[b] : base + (int64_t)b * stride; }
};

template <int BM_, int BN_, int WM_, int WN_, int STAGES>
struct TileShape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;       // tile, waves down and across
  static constexpr int W = WM * WN, threads = W * 64;
  static constexpr int TM = BM / WM, TN = BN / WN;                   // a wave's part
  static constexpr int FM = TM / 32, FN = TN / 32;                   // its MFMA blocks
  static constexpr int stages = STAGES;                              // buffers that go round
  static constexpr int stage_halves = (BM + BN) * kTileK;
  static constexpr int wave_sums = TM * TN;
  static constexpr bool whole_steps = FM * FN <= 4;                  // read a step ahead, not a quarter
};

#define ZEN_LDS __attribute__((address_space(3)))

// One operand's share of loads and reads. R: the tile's rows (i or j); KC: k is contiguous.
template <int R, bool KC, int W>
struct TileOperand {
  static constexpr int loads = R / 8 / W;  // 1 KiB each, per wave and step
  static_assert(R / 8 % W == 0, "a step's loads are shared evenly");
  static constexpr int row_lanes = KC ? 8 : R / 8;    // lanes to a row of the piece
  static constexpr int rows = 64 / row_lanes;         // rows to a load
  static_assert(KC || (W * rows) % 4 == 0, "the swizzle is the same in every load of a wave");
  const char *first[2];   // of the tile in the matrix, and in what its rounding left over
  const char *base;       // of the step that is aimed at next
  int64_t step;           // bytes from step to step
  uint32_t records, full, tail;  // bytes there are from `base` on; in the first step; (k as the stride) in the last one
  uint32_t voffset, vlast, vnow, soffset;
  __amdgpu_buffer_rsrc_t source;

  // k contiguous: piece c of row r lies in place c ^ key(r)
  static __device__ __forceinline__ int key(int r) { return ((r >> 1) & 3) | ((r >> 2) & 4); }

  // k as the stride: where piece `chunk` of row k of the step lies
  static __device__ __forceinline__ int place(int k, int chunk) { return chunk ^ (R >= 128 ? (k & 3) << 2 : (k & 2) << 1); }

  // r0: first row (i or j) of the tile; rows_all: rows there are; k: the operand's k.  What a step reaches lies within 2^30
  // bytes (kMostLd), so 32 bits do for everything but the addresses.
  __device__ __forceinline__ void start(const MatOperand &o, int z, int64_t r0, int64_t rows_all, int k, int wave, int lane) {
    const int row = wave * rows + lane / row_lanes;
    const int slot = lane % row_lanes;
    const int chunk = KC ? slot ^ key(row) : place(row, slot);
    const int64_t ld = o.ld, from = z * o.batch + (KC ? r0 * ld : r0);
    first[0] = reinterpret_cast<const char *>(o.p[0] + from);
    first[1] = reinterpret_cast<const char *>(o.p[1] + from);
    const int rest = (k - 1) % kTileK + 1;  // k of the last step
    voffset = vlast = (uint32_t)((row * ld + chunk * 8) * 2);
    if (KC) {
      const int64_t lines = rows_all - r0 < R ? rows_all - r0 : R;
      full = (uint32_t)(((lines - 1) * ld + ((k + 7) & ~7)) * 2);  // whole pieces: k is a multiple of 8, or ld has room
      tail = 0;
      step = kTileK * 2;
      if (chunk * 8 >= rest) vlast = 0x80000000u;
    } else {
      const int64_t line = (rows_all - r0 + 1) & ~1ll;  // whole words: the address is a multiple of 16
      const int64_t most = line < ld ? line : ld;
      full = (uint32_t)(((kTileK - 1) * ld + most) * 2);
      tail = (uint32_t)(((rest - 1) * ld + most) * 2);
      step = kTileK * ld * 2;
    }
    soffset = (uint32_t)(W * rows * ld * 2);
  }

  // The next step aimed at is step `at`, of `low`'s matrix.
  __device__ __forceinline__ void begin(bool low, int at) {
    base = first[low] + at * step;
    records = KC ? full - at * (uint32_t)(kTileK * 2) : full;
  }

  // What the loads of the step read (the operand's last step?): nothing where `there` is false, zeros arrive.
  __device__ __forceinline__ void aim(bool last, bool there) {
    const uint32_t bytes = KC ? records : last ? tail : full;
    // all lanes' are the same, and the loads want them in scalar registers: where the compiler has come to keep them in others it
    // would loop over the lanes' values at every load
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    const uint64_t low = (uint32_t)__builtin_amdgcn_readfirstlane((int)at), high = (uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32));
    source = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(high << 32 | low), 0,
                                               __builtin_amdgcn_readfirstlane((int)(there ? bytes : 0u)), 0x00027000);
    vnow = KC && last ? vlast : voffset;
    base += step;
    records -= kTileK * 2;
  }

  // Load q of them into `lds` (this operand's part of a buffer).
  __device__ __forceinline__ void load(uint16_t *lds, int q, int wave) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(source, (ZEN_LDS void *)(lds + (q * W + wave) * 512), 16, (int)vnow,
                                             (int)(q * soffset), 0, 0);
  }

  // The block of 32 rows from row r0 of the tile (a multiple of 32) and k from kk * 16, as an MFMA operand.
  static __device__ __forceinline__ short8v read(const uint16_t *lds, int r0, int kk, int lane) {
    if (KC) {
      const int r = r0 + (lane & 31);
      const int chunk = (kk * 2 + (lane >> 5)) ^ key(lane);  // r0 is a multiple of 32
      return *reinterpret_cast<const short8v *>(lds + r * kTileK + chunk * 8);
    }
    // sixteen lanes turn four rows of sixteen: lane j gives the address of four elements of row j / 4
    const int j = lane & 15;
    const int krow = kk * 16 + (lane >> 5) * 8 + (j >> 2);
    const int slot = place(krow, (r0 >> 3) + ((lane >> 4) & 1) * 2 + ((j & 3) >> 1));  // the same four rows on
    const uint16_t *at = lds + krow * R + slot * 8 + (j & 1) * 4;
    const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ZEN_LDS short4v *)(at));
    const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ZEN_LDS short4v *)(at + 4 * R));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// All but the newest LOADS of the wave's loads into LDS have arrived, it has got what it read from there, and so have all waves of
// the workgroup.  (A fence would wait for all loads.)
template <int LOADS>
__device__ __forceinline__ void arrived() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x70 | (LOADS & 15) | (LOADS >> 4) << 14);  // vmcnt(LOADS) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <bool BF>
__device__ __forceinline__ float16v mfma(short8v a, short8v b, float16v c) {
  if (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// Row and column of tile t of the lower triangle, counted row by row.
__device__ __forceinline__ void triangle(int t, int &i, int &j) {
  i = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
  while ((int64_t)i * (i + 1) / 2 > t) --i;
  while ((int64_t)(i + 1) * (i + 2) / 2 <= t) ++i;
  j = t - (int)((int64_t)i * (i + 1) / 2);
}

// Number of a tile among the launch's, for what is kept by tiles.
template <bool SYM>
__device__ __forceinline__ int tile_number(const MatSize &s, int b, int ti, int tj) {
  return SYM ? b * (s.tiles_m * (s.tiles_m + 1) / 2) + ti * (ti + 1) / 2 + tj : (b * s.tiles_m + ti) * s.tiles_n + tj;
}

// The launch's tiles: of the whole matrix, or of its lower triangle (SYM), each in so many shares.  Workgroups go round the eight dies, whose
// L2s are apart: the tiles are dealt so that a die's are neighbours, four tile rows by all columns at a time.
template <bool SYM>
__device__ __forceinline__ void tile_of(const MatSize &s, int shares, int &share, int &b, int &ti, int &tj) {
  const int per = SYM ? s.tiles_m * (s.tiles_m + 1) / 2 : s.tiles_m * s.tiles_n;
  const int all = per * s.batch * shares;
  int t = (int)blockIdx.x;
  const int die = t & 7, most = all >> 3, rest = all & 7;
  t = die * most + (die < rest ? die : rest) + (t >> 3);
  share = t % shares;
  t /= shares;
  b = t / per;
  t -= b * per;
  if (SYM) {
    triangle(t, ti, tj);
    return;
  }
  constexpr int kGroup = 4;
  const int group = t / (kGroup * s.tiles_n), first = group * kGroup;
  const int rows = s.tiles_m - first < kGroup ? s.tiles_m - first : kGroup;
  t -= group * kGroup * s.tiles_n;
  ti = first + t % rows;
  tj = t / rows;
}

// ---------------------------------------------------------------- what becomes of a tile

__device__ __forceinline__ float load_value(const char *p, int64_t i, int dtype) {
  if (dtype == ZEN_F32) return reinterpret_cast<const float *>(p)[i];
  if (dtype == ZEN_BF16) return (float)reinterpret_cast<const __bf16 *>(p)[i];
  return (float)reinterpret_cast<const _Float16 *>(p)[i];
}

__device__ __forceinline__ void store_value(char *p, int64_t i, int dtype, float v) {
  if (dtype == ZEN_F32) reinterpret_cast<float *>(p)[i] = v;
  else if (dtype == ZEN_BF16) reinterpret_cast<__bf16 *>(p)[i] = (__bf16)v;
  else reinterpret_cast<_Float16 *>(p)[i] = (_Float16)v;
}

typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float8v __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float8v widen(half8v v) { return __builtin_convertvector(v, float8v); }

__device__ __forceinline__ float8v load_eight(const char *p, int64_t i, int dtype) {
  if (dtype == ZEN_F32) return *reinterpret_cast<const float8v *>(p + i * 4);
  if (dtype == ZEN_BF16) return __builtin_convertvector(*reinterpret_cast<const bf8 *>(p + i * 2), float8v);
  return widen(*reinterpret_cast<const half8v *>(p + i * 2));
}

// `of(e)`-th elements for e below N, all on their way together: no branch but the one on the type, which stands around them.
template <int N, class T, class At>
__device__ __forceinline__ void load_these(const char *p, float (&v)[N], At of) {
  T raw[N];
#pragma unroll
  for (int e = 0; e < N; ++e) raw[e] = reinterpret_cast<const T *>(p)[of(e)];
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (float)raw[e];
}

template <int N, class At>
__device__ __forceinline__ void load_values(const char *p, int dtype, float (&v)[N], At of) {
  if (dtype == ZEN_F32) load_these<N, float>(p, v, of);
  else if (dtype == ZEN_BF16) load_these<N, __bf16>(p, v, of);
  else load_these<N, _Float16>(p, v, of);
}

// Elements j to j + 7 of a line of n a stride apart, zeros behind its end.
__device__ __forceinline__ float8v load_line(const char *p, int64_t line, int64_t stride, int j, int n, int dtype) {
  float v[8];
  load_values(p, dtype, v, [&](int e) { return line + (j + e < n ? j + e : n - 1) * stride; });
  float8v out;
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = j + e < n ? v[e] : 0.f;
  return out;
}

__device__ __forceinline__ void store_eight(char *p, int64_t i, int dtype, float8v v) {
  if (dtype == ZEN_F32) *reinterpret_cast<float8v *>(p + i * 4) = v;
  else if (dtype == ZEN_BF16) *reinterpret_cast<bf8 *>(p + i * 2) = __builtin_convertvector(v, bf8);
  else *reinterpret_cast<half8v *>(p + i * 2) = __builtin_convertvector(v, half8v);
}

// The wave's order of its own LDS operations is the program's; this holds the compiler to it.
__device__ __forceinline__ void lds_in_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// 32 rows of a wave's sums on their way out, through LDS: written as the MFMA layout has them, read eight neighbours a lane,
// of a row or (for a mirror image) of a column.  Rows of COLS + 4: neighbouring rows begin in different banks.
template <int COLS>
struct Stage {
  static constexpr int row = COLS + 4;
  static constexpr int floats = 32 * row;
  static constexpr int turns = 32 * COLS / 512;  // eight a lane

  static __device__ __forceinline__ void of_row(int turn, int lane, int &i, int &j) {
    const int at = turn * 64 + lane;
    i = at / (COLS / 8);
    j = at % (COLS / 8) * 8;
  }
  static __device__ __forceinline__ float8v row_sums(const float *sums, int i, int j) {
    const float4v a = *reinterpret_cast<const float4v *>(sums + i * row + j), b = *reinterpret_cast<const float4v *>(sums + i * row + j + 4);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ void put_row(float *sums, int i, int j, float8v v) {
    *reinterpret_cast<float4v *>(sums + i * row + j) = __builtin_shufflevector(v, v, 0, 1, 2, 3);
    *reinterpret_cast<float4v *>(sums + i * row + j + 4) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ void of_column(int turn, int lane, int &i, int &j) {
    const int at = turn * 64 + lane;
    i = (at & 3) * 8;
    j = at >> 2;
  }
  static __device__ __forceinline__ float8v column_sums(const float *sums, int i, int j) {
    float8v v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = sums[(i + e) * row + j];
    return v;
  }
};

// What goes out to a caller's matrix: out = gain * (alpha * acc + beta * (X + X')) + keep * res.
struct OutEpilogue {
  float alpha, beta, gain, keep;
  const _Float16 *x, *x_low;  // null: none (and no mirror image where there is one)
  int64_t x_ld, x_batch;
  const float *row_low;       // with x: what rounding left over of the left operand's diagonal, a row's times alpha joins beta (null: none)
  int64_t low_batch;
  int rows, cols;
  MatList out, res;             // res: listed < 0 for none
  int64_t out_rs, out_cs, res_rs, res_cs;
  int out_type, res_type;
  int lines;                    // 1: rows of out and res are contiguous and begin at multiples of 16 bytes; 2: columns
                                // do (and there is no mirror image); 0: neither

  __device__ __forceinline__ float beta_of(int z, int i) const {
    return row_low ? fmaf(alpha, row_low[z * low_batch + i], beta) : beta;
  }

  template <int COLS, int AT>
  __device__ __forceinline__ void block(int z, int i0, int j0, float *sums, bool mirror, int lane) const {
    using T = Stage<COLS>;
    if (i0 >= rows || j0 >= cols) return;
    char *o = out.of(z);
    const char *r = res.listed >= 0 ? res.of(z) : nullptr;
    if (lines && i0 + 32 <= rows && j0 + COLS <= cols) {
#pragma unroll
      for (int turn = 0; turn < T::turns; ++turn) {
        int di, dj;
        T::of_row(turn, lane, di, dj);
        float8v v = alpha * T::row_sums(sums, di, dj);
        const int i = i0 + di, j = j0 + dj;
        if (x) {
          const int64_t at = z * x_batch + (int64_t)i * x_ld + j;
          v += beta_of(z, i) * (widen(*reinterpret_cast<const half8v *>(x + at)) + widen(*reinterpret_cast<const half8v *>(x_low + at)));
        }
        v *= gain;
        if (lines == 2) {
          T::put_row(sums, di, dj, v);
          continue;
        }
        if (r) v += keep * load_eight(r, i * res_rs + j, res_type);
        store_eight(o, i * out_rs + j, out_type, v);
      }
      if (lines == 2) {
        lds_in_order();
#pragma unroll
        for (int turn = 0; turn < T::turns; ++turn) {
          int i, j;
          T::of_column(turn, lane, i, j);
          float8v v = T::column_sums(sums, i, j);
          i += i0;
          j += j0;
          if (r) v += keep * load_eight(r, j * res_cs + i, res_type);
          store_eight(o, j * out_cs + i, out_type, v);
        }
        return;
      }
      if (!mirror) return;
#pragma unroll 1
      for (int turn = 0; turn < T::turns; ++turn) {
        int i, j;
        T::of_column(turn, lane, i, j);
        float8v v = gain * alpha * T::column_sums(sums, i, j);
        i += i0;
        j += j0;
        if (r) v += keep * load_eight(r, j * res_rs + i, res_type);
        store_eight(o, j * out_rs + i, out_type, v);
      }
      return;
    }
    // one by one: the tile hangs over the matrix, or its rows are not lines
    const int turns = mirror ? 2 : 1;
    for (int turn = 0; turn < turns; ++turn) {
      const bool down = (out_rs < out_cs) != (turn == 1);  // neighbouring lanes are neighbours of a column
      for (int base = lane; base < 32 * COLS; base += 64 * AT) {
        float v[AT], read[AT];
        int i[AT], j[AT];
        bool there[AT];
#pragma unroll
        for (int u = 0; u < AT; ++u) {  // no branches: what lies beyond the matrix reads its last row or column
          const int at = base + u * 64;
          const int di = down ? at & 31 : at / COLS, dj = down ? at >> 5 : at % COLS;
          there[u] = i0 + di < rows && j0 + dj < cols;
          i[u] = i0 + di < rows ? i0 + di : rows - 1;
          j[u] = j0 + dj < cols ? j0 + dj : cols - 1;
          v[u] = alpha * sums[di * T::row + dj];
        }
        if (x) {
          const auto from = [&](int u) { return z * x_batch + (int64_t)i[u] * x_ld + j[u]; };
          float low[AT];
          load_these<AT, _Float16>(reinterpret_cast<const char *>(x), read, from);
          load_these<AT, _Float16>(reinterpret_cast<const char *>(x_low), low, from);
#pragma unroll
          for (int u = 0; u < AT; ++u) v[u] += beta_of(z, i[u]) * (read[u] + low[u]);
        }
#pragma unroll
        for (int u = 0; u < AT; ++u) v[u] *= gain;
        if (r) {
          load_values(r, res_type, read, [&](int u) { return (turn ? j[u] : i[u]) * res_rs + (turn ? i[u] : j[u]) * res_cs; });
#pragma unroll
          for (int u = 0; u < AT; ++u) v[u] += keep * read[u];
        }
#pragma unroll
        for (int u = 0; u < AT; ++u)
          if (there[u]) store_value(o, (turn ? j[u] : i[u]) * out_rs + (turn ? i[u] : j[u]) * out_cs, out_type, v[u]);
      }
    }
  }
};

// What goes back to a workspace, of the three products of a step:
//   kGram    d = alpha acc
//   kSquare  d = alpha acc + beta c + diag on the diagonal, where acc is c c
//   kApply   d = alpha acc + beta (c + c'), its transpose t beside it, where acc is P c
// in 16 bits, for kApply in twice 16.  Rows and columns are multiples of 64.
// HALVES: every operand has its left-over (c', d', t') in 16 bits.  Otherwise the diagonals of what kGram and kSquare write are kept
// whole: their entries are often nearly equal, so that rounding takes all of them the same way and scales the whole product (384
// x 6000: results off by 1.4e-3, 0.6e-3 with whole diagonals).  What their rounding leaves over goes to `low` and is made good where
// the matrix is used, for a number an element.
enum Keep { kGram, kSquare, kApply };

template <Keep WHAT, bool HALVES>
struct KeepEpilogue {
  float alpha, beta, diag;
  int rows, cols;
  int diag_n;  // the diagonal's length
  const _Float16 *c, *c_low;
  _Float16 *d, *d_low, *t, *t_low;
  int64_t ld, batch, t_ld, t_batch;  // c lies as d does
  float *low;             // kGram, kSquare: of d's diagonal
  const float *from_low;  // kSquare: of c's diagonal; kApply: of P's
  int64_t low_batch;      // of both

  template <bool LOW>
  static __device__ __forceinline__ void store(_Float16 *p, _Float16 *low, int64_t at, float8v v) {
    const half8v h = __builtin_convertvector(v, half8v);
    *reinterpret_cast<half8v *>(p + at) = h;
    if constexpr (LOW) *reinterpret_cast<half8v *>(low + at) = __builtin_convertvector(v - widen(h), half8v);
  }

  template <int COLS, int AT>
  __device__ __forceinline__ void block(int z, int i0, int j0, float *sums, bool mirror, int lane) const {
    using T = Stage<COLS>;
    constexpr bool kWhole = !HALVES && WHAT != kApply;
    if (i0 >= rows || j0 >= cols) return;
    const bool turned = mirror || WHAT == kApply;
    const float *l = HALVES || WHAT == kGram ? nullptr : from_low + z * low_batch;
    float8v across = {};
    if constexpr (!HALVES && WHAT == kSquare) {
      int di, dj;
      T::of_row(0, lane, di, dj);  // a lane's columns are the same in every turn
      across = *reinterpret_cast<const float8v *>(l + j0 + dj);
    }
#pragma unroll
    for (int turn = 0; turn < T::turns; ++turn) {
      int di, dj;
      T::of_row(turn, lane, di, dj);
      const int i = i0 + di, j = j0 + dj;
      const int64_t at = z * batch + (int64_t)i * ld + j;
      const bool crossed = i >= j && i < j + 8;  // by the diagonal
      float8v v = T::row_sums(sums, di, dj);
      if constexpr (WHAT != kGram) {
        float8v own = widen(*reinterpret_cast<const half8v *>(c + at));
        float times = beta;
        if constexpr (!HALVES && WHAT == kApply) times = fmaf(alpha, l[i], beta);  // (P + l) c for a diagonal l
        if constexpr (!HALVES && WHAT == kSquare) {  // (c + l)(c + l): l l is beyond fp32's last bit
          const float mine = l[i];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = fmaf(own[e], mine + across[e], v[e]);
            own[e] += i == j + e ? mine : 0.f;
          }
        }
        if constexpr (HALVES || WHAT == kApply) own += widen(*reinterpret_cast<const half8v *>(c_low + at));
        v = alpha * v + times * own;
      } else {
        v *= alpha;
      }
      if constexpr (WHAT == kSquare) {
        if (diag != 0.f && crossed && i < diag_n) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += i == j + e ? diag : 0.f;
        }
      }
      store<HALVES || WHAT == kApply>(d, d_low, at, v);
      if (kWhole && crossed) {
        float left = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) left += i == j + e ? v[e] - (float)(_Float16)v[e] : 0.f;
        low[z * low_batch + i] = left;
      }
      if (turned) T::put_row(sums, di, dj, v);
    }
    if (!turned) return;
    lds_in_order();
    _Float16 *to = mirror ? d : t, *to_low = mirror ? d_low : t_low;
    const int64_t to_ld = mirror ? ld : t_ld, from = z * (mirror ? batch : t_batch);
#pragma unroll
    for (int turn = 0; turn < T::turns; ++turn) {
      int di, dj;
      T::of_column(turn, lane, di, dj);
      store<HALVES>(to, to_low, from + (int64_t)(j0 + dj) * to_ld + i0 + di, T::column_sums(sums, di, dj));
    }
  }
};

// LDS of a wave's epilogue, in halves.
template <class S>
constexpr int epilogue_cols() { return S::TN % 64 ? 32 : 64; }
template <class S>
constexpr int epilogue_halves() { return 2 * Stage<epilogue_cols<S>()>::floats; }

// ROWS times 32 rows of a wave's part of the tile, from row i0 and column j0 on.
template <class S, int ROWS, class Epilogue>
__device__ __forceinline__ void finish(const Epilogue &e, int z, int i0, int j0, const float16v (&acc)[ROWS][S::FN], bool mirror,
                                       uint16_t *lds, int lane) {
  constexpr int kCols = epilogue_cols<S>();
  // elements on their way together where they go one by one: many where the code is laid out few times
  constexpr int kAtOnce = ROWS * S::TN / kCols <= 2 ? 8 : 2;
  float *sums = reinterpret_cast<float *>(lds);
#pragma unroll
  for (int a = 0; a < ROWS; ++a)
#pragma unroll
    for (int c = 0; c < S::TN; c += kCols) {
      // of a 32 x 32 block a lane holds row lane & 31: four times four neighbours, eight columns apart
#pragma unroll
      for (int b = 0; b < kCols / 32; ++b)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float16v &f = acc[a][c / 32 + b];
          *reinterpret_cast<float4v *>(sums + (lane & 31) * Stage<kCols>::row + b * 32 + q * 8 + (lane >> 5) * 4) =
              float4v{f[q * 4], f[q * 4 + 1], f[q * 4 + 2], f[q * 4 + 3]};
        }
      lds_in_order();
      e.template block<kCols, kAtOnce>(z, i0 + a * 32, j0 + c, sums, mirror, lane);
      lds_in_order();
    }
}

template <class S, bool AK, bool BK, bool BF, bool SYM, class Epilogue>
__global__ __launch_bounds__(S::threads, S::W > 4 || S::stages * S::stage_halves <= 40960 ? 2 : 1) void k_tiles(MatSize size, MatOperand a, MatOperand b, Epilogue epilogue) {
  static_assert(S::W * epilogue_halves<S>() <= S::stages * S::stage_halves, "the epilogue fits the buffers");
  __shared__ __attribute__((aligned(1024))) uint16_t s_buf[S::stages * S::stage_halves];
  int z, ti, tj, share;
  tile_of<SYM>(size, size.splits, share, z, ti, tj);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / S::WN, wn = wave % S::WN;
  using OpA = TileOperand<S::BM, AK, S::W>;
  using OpB = TileOperand<S::BN, BK, S::W>;
  OpA la;
  OpB lb;
  const int steps = (size.k + kTileK - 1) / kTileK;
  // this workgroup's steps of all parts
  const int begin = (int)((int64_t)steps * size.parts * share / size.splits);
  const int all = (int)((int64_t)steps * size.parts * (share + 1) / size.splits) - begin;
  la.start(a, z, (int64_t)ti * S::BM, size.m, size.k, wave, lane);
  lb.start(b, z, (int64_t)tj * S::BN, size.n, size.k, wave, lane);
  int at = begin % (steps ? steps : 1), part = begin / (steps ? steps : 1);  // what is loaded next: step of a part
  int left = all;
  la.begin(part == 2, at);
  lb.begin(part == 1, at);

  auto aim = [&]() {
    const bool there = left-- > 0, last = at + 1 == steps;
    la.aim(last, there);
    lb.aim(last, there);
    ++at;
    if (last) {
      at = 0;
      ++part;
      la.begin(part == 2, 0);
      lb.begin(part == 1, 0);
    }
  };
  constexpr int kLoads = OpA::loads + OpB::loads;
  auto load = [&](uint16_t *buf, int l) {
    if (l < OpA::loads) la.load(buf, l, wave);
    else lb.load(buf + S::BM * kTileK, l - OpA::loads, wave);
  };

  float16v acc[S::FM][S::FN];
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) acc[i][j] = float16v{};

  // Reads of LDS and loads into it lie one by one between the products, in the order written here (a row of loads would hold the
  // wave up for as long as the address unit takes over them; the compiler would move reads to where they are used).
  constexpr int kProducts = S::FM * S::FN, kReads = S::FM + S::FN, kQuarters = kTileK / 16, kAhead = (S::stages - 2) * kLoads;
  constexpr int kSets = S::whole_steps ? 2 * kQuarters : 2;
  short8v fa[kSets][S::FM], fb[kSets][S::FN];
  auto read = [&](const uint16_t *buf, int kk, int set, int r) {
    if (r < S::FN) fb[set][r] = OpB::read(buf + S::BM * kTileK, wn * S::TN + r * 32, kk, lane);
    else fa[set][r - S::FN] = OpA::read(buf, wm * S::TM + (r - S::FN) * 32, kk, lane);
  };
  // The products of `set`; between them the reads of quarter kk into set `to`, and loads first..last - 1.  The compiler lets a
  // transposing read wait for all loads into LDS in front of it: with one of those the loads come behind the reads.
  constexpr bool kPlain = AK && BK;
  constexpr int kReadUp = kPlain ? kProducts : (kReads + 1) / 2;  // products that reads lie between
  constexpr int kLoadFrom = kPlain ? 0 : kReadUp < kProducts ? kReadUp : kProducts - 1;
  auto quarter = [&](int set, const uint16_t *from, int kk, int to, uint16_t *into, int first, int last) {
#pragma unroll
    for (int p = 0; p < kProducts; ++p) {
#pragma unroll
      for (int r = kReads * p / kReadUp; r < kReads * (p + 1) / kReadUp; ++r)
        if (r < kReads) read(from, kk, to, r);
      const int l0 = p < kLoadFrom ? 0 : (last - first) * (p - kLoadFrom) / (kProducts - kLoadFrom);
      const int l1 = p < kLoadFrom ? 0 : (last - first) * (p - kLoadFrom + 1) / (kProducts - kLoadFrom);
#pragma unroll
      for (int l = first + l0; l < first + l1; ++l) load(into, l);
      const int i = p / S::FN, j = p % S::FN;
      acc[i][j] = mfma<BF>(fb[set][j], fa[set][i], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // How many of a step's loads follow its barrier at once: with two buffers all, they are needed at the next one; with more the
  // rest lie in the three quarters behind.
  constexpr int kAtOnce = S::whole_steps || S::stages == 2 || !kPlain ? kLoads : kLoads / 4;
  if (all > 0) {
#pragma unroll
    for (int p = 0; p < S::stages; ++p) {
      aim();
#pragma unroll
      for (int l = 0; l < kLoads; ++l)
        if (p + 1 < S::stages || l < kAtOnce) load(s_buf + p * S::stage_halves, l);
    }
    arrived<kAhead + kAtOnce>();
    // step t's buffer, the next one's, and the one that is being loaded
    int now = 0, next = S::stage_halves, into = (S::stages - 1) * S::stage_halves;
    auto round = [&]() {
      into = now;
      now = next;
      next = next + S::stage_halves == S::stages * S::stage_halves ? 0 : next + S::stage_halves;
    };
    if constexpr (S::whole_steps) {
      // A step's products are too few to cover a quarter's reads: all of the next step is read while one is multiplied.  In front
      // of that lies the step's one barrier: every wave has read this step whole, so its buffer is loaded again, and the next
      // one has arrived.
#pragma unroll
      for (int kk = 0; kk < kQuarters; ++kk)
#pragma unroll
        for (int r = 0; r < kReads; ++r) read(s_buf, kk, kk, r);
      for (int t = 0; t < all; t += 2) {  // an odd number: one step of zeros behind them
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          arrived<kAhead>();
          aim();
#pragma unroll
          for (int kk = 0; kk < kQuarters; ++kk)
            quarter(u * kQuarters + kk, s_buf + next, kk, (u ^ 1) * kQuarters + kk, s_buf + now,
                    kPlain ? kLoads * kk / kQuarters : 0,
                    kPlain ? kLoads * (kk + 1) / kQuarters : kk + 1 == kQuarters ? kLoads : 0);
          round();
        }
      }
    } else {
      // Fragments of 16 k are read while those before them are multiplied, also across the steps: a step's last quarter is
      // multiplied while the first of the next one is read.  In front of that lies the step's one barrier: every wave has
      // read all of the step's buffer, so it is loaded again, and the next one has arrived.
#pragma unroll
      for (int r = 0; r < kReads; ++r) read(s_buf, 0, 0, r);
      for (int t = 0; t < all; ++t) {  // behind the last step zeros are loaded, and not multiplied
#pragma unroll
        for (int kk = 0; kk + 1 < kQuarters; ++kk)
          quarter(kk & 1, s_buf + now, kk + 1, ~kk & 1, s_buf + into, kAtOnce + (kLoads - kAtOnce) * kk / 3,
                  kAtOnce + (kLoads - kAtOnce) * (kk + 1) / 3);
        arrived<kAhead>();
        aim();
        quarter(1, s_buf + next, 0, 0, s_buf + now, 0, kAtOnce);
        round();
      }
    }
  }

  arrived<0>();  // the buffers are free: nothing is on its way into them
  if (size.splits > 1) {  // a lane's sums as they are, one line a wave and register
    float4v *to = reinterpret_cast<float4v *>(size.partial + ((int64_t)tile_number<SYM>(size, z, ti, tj) * size.splits + share) * (S::BM * S::BN) +
                                              wave * S::wave_sums) + lane;
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
      for (int j = 0; j < S::FN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float16v &f = acc[i][j];
          to[((i * S::FN + j) * 4 + q) * 64] = float4v{f[q * 4], f[q * 4 + 1], f[q * 4 + 2], f[q * 4 + 3]};
        }
    return;
  }
  finish<S, S::FM>(epilogue, z, ti * S::BM + wm * S::TM, tj * S::BN + wn * S::TN, acc, SYM && ti != tj, s_buf + wave * epilogue_halves<S>(), lane);
}

// The sums of a tile's shares, in their order, and what becomes of them: a workgroup of one wave for every 32 rows of a wave's part.
template <class S, bool SYM, class Epilogue>
__global__ __launch_bounds__(64) void k_join(MatSize size, Epilogue epilogue) {
  __shared__ __attribute__((aligned(16))) uint16_t s_sums[epilogue_halves<S>()];
  int z, ti, tj, part;
  tile_of<SYM>(size, S::W * S::FM, part, z, ti, tj);
  const int wave = part / S::FM, rows = part % S::FM, lane = threadIdx.x;
  const float4v *from = reinterpret_cast<const float4v *>(size.partial + (int64_t)tile_number<SYM>(size, z, ti, tj) * size.splits * (S::BM * S::BN) +
                                                          wave * S::wave_sums + rows * 32 * S::TN) + lane;
  float16v acc[1][S::FN];
#pragma unroll
  for (int j = 0; j < S::FN; ++j) acc[0][j] = float16v{};
#pragma unroll 4
  for (int share = 0; share < size.splits; ++share, from += S::BM * S::BN / 4) {
#pragma unroll
    for (int j = 0; j < S::FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4v f = from[(j * 4 + q) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[0][j][q * 4 + e] += f[e];
      }
  }
  finish<S, 1>(epilogue, z, ti * S::BM + wave / S::WN * S::TM + rows * 32, tj * S::BN + wave % S::WN * S::TN, acc, SYM && ti != tj, s_sums, lane);
}

template <class S, bool AK, bool BK, bool BF, bool SYM, class Epilogue>
inline int launch_tiles(MatSize size, const MatOperand &a, const MatOperand &b, const Epilogue &e, hipStream_t stream) {
  static_assert(!SYM || S::BM == S::BN, "a triangle of square tiles");
  size.tiles_m = (size.m + S::BM - 1) / S::BM;
  size.tiles_n = (size.n + S::BN - 1) / S::BN;
  const int64_t tiles = (SYM ? (int64_t)size.tiles_m * (size.tiles_m + 1) / 2 : (int64_t)size.tiles_m * size.tiles_n) * size.batch;
  const int64_t joined = size.splits > 1 ? S::W * S::FM * 64 : 0;
  if (tiles > kMostThreads / (size.splits * S::threads + joined)) return fail(ZEN_EINVAL, "matrix product: too many tiles");
  k_tiles<S, AK, BK, BF, SYM, Epilogue><<<dim3((unsigned)(tiles * size.splits)), dim3(S::threads), 0, stream>>>(size, a, b, e);
  ZEN_LAUNCH_CHECK("k_tiles");
  if (size.splits > 1) {
    k_join<S, SYM, Epilogue><<<dim3((unsigned)(tiles * S::W * S::FM)), dim3(64), 0, stream>>>(size, e);
    ZEN_LAUNCH_CHECK("k_join");
  }
  return ZEN_OK;
}

// ---------------------------------------------------------------- which tiles

// What a step of 64 k costs a compute unit, in us: measured with products from one tile to some rounds of tiles (256 x 256 x 4096 to
// 4096^3, k 1024 and 4096).  Large tiles read LDS and L2 least for their sums (4096^3: 124 us with 256, 130 with 128, 251
// with 64); small ones fill the card where there are few (1024 x 1024 x 4096: 79, 32 and 20 us).  With a tile on every unit the
// L2s bound the small ones (12 to 16 TB/s).  A launch costs some us apart from its steps, and so does joining the shares of
// tiles that are split.
struct TileCost {
  int side;
  int at_once;           // workgroups that a compute unit holds
  float lone, one, all;  // us a step: a workgroup by itself; one on every unit; at_once on every unit
  float launch;          // us, with the epilogue
  bool k_only;           // operands with k contiguous only
};
constexpr TileCost kTileCosts[] = {
    {256, 1, 1.10f, 1.85f, 1.85f, 9.f, false}, {192, 1, 0.75f, 1.20f, 1.20f, 7.f, true},
    {128, 2, 0.95f, 0.95f, 1.05f, 6.f, false}, {128, 1, 0.37f, 0.64f, 0.64f, 5.f, false}, {64, 2, 0.17f, 0.25f, 0.48f, 4.f, false}};
constexpr int kMostSplits = 24;

struct TilePlan {
  int side, at_once, splits;
  size_t partial_bytes;
};

// What the *_path calls say of it (include/zen_hip.h).
inline int path_of(const TilePlan &p) { return p.side | p.at_once << 10 | p.splits << 12; }

inline TilePlan plan_tiles(int64_t m, int64_t n, int64_t k, int parts, int64_t batch, bool sym, bool by_k) {
  const int64_t steps = ceil_div(k, kTileK) * parts;
  TilePlan best = {64, 2, 1, 0};
  double least = 1e30;
  for (const TileCost &c : kTileCosts) {
    if (c.k_only && !by_k) continue;
    const int64_t down = ceil_div(m, c.side), across = ceil_div(n, c.side);
    const int64_t tiles = (sym ? down * (down + 1) / 2 : down * across) * batch;
    for (int splits = 1; splits <= kMostSplits && (splits == 1 || (tiles * splits <= 512 && steps / splits >= 4)); ++splits) {
      const int64_t groups = tiles * splits;
      // whole rounds, and a last one of so many a unit
      const int64_t slots = 256 * c.at_once, whole = groups <= 256 ? 0 : groups / slots, rest = groups - whole * slots;
      const double last = rest == 0 ? 0.0 : rest <= 256 ? c.lone + (c.one - c.lone) * rest / 256.0 : c.all;
      const double bytes = splits > 1 ? 4.0 * groups * c.side * c.side : 0.0;
      const double us = (whole * c.all + last) * (double)ceil_div(steps, splits) + c.launch + (splits > 1 ? 4.0 + bytes / 2e6 : 0.0);
      if (us < least) {
        least = us;
        best = {c.side, c.at_once, splits, (size_t)bytes};
      }
    }
  }
  return best;
}

using Tile256 = TileShape<256, 256, 2, 4, 2>;
using Tile192 = TileShape<192, 192, 2, 2, 3>;
using Tile128 = TileShape<128, 128, 2, 2, 2>;      // two workgroups to a compute unit
using Tile128Deep = TileShape<128, 128, 2, 2, 4>;  // one: where there are no more, they spread over all units, loads further ahead
using Tile64 = TileShape<64, 64, 2, 2, 4>;

// The product as planned; partial: plan.partial_bytes.
template <bool AK, bool BK, bool BF, bool SYM, class Epilogue>
inline int run_tiles(const TilePlan &plan, float *partial, MatSize size, const MatOperand &a, const MatOperand &b, const Epilogue &e,
                     hipStream_t stream) {
  size.splits = plan.splits;
  size.partial = partial;
  if (plan.side == 256) return launch_tiles<Tile256, AK, BK, BF, SYM>(size, a, b, e, stream);
  if constexpr (AK && BK)
    if (plan.side == 192) return launch_tiles<Tile192, AK, BK, BF, SYM>(size, a, b, e, stream);
  if (plan.side == 128 && plan.at_once == 1) return launch_tiles<Tile128Deep, AK, BK, BF, SYM>(size, a, b, e, stream);
  if (plan.side == 128) return launch_tiles<Tile128, AK, BK, BF, SYM>(size, a, b, e, stream);
  return launch_tiles<Tile64, AK, BK, BF, SYM>(size, a, b, e, stream);
}

// Matrices of 16-bit values laid out for the tiles: `rows` x `cols` at any strides become rows of `ld` elements, zeros beyond `cols`
// (zen_pack.hip).
struct PackArgs {
  MatList in;
  int64_t rs, cs;
  int rows, cols;
  int batch;
  uint16_t *out;
  int64_t ld, out_batch;
};
int pack_matrices(const PackArgs *args, int count, hipStream_t stream);  // one or two of them, one launch

}  // namespace zen
