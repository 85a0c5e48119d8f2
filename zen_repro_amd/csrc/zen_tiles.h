// Matrix products in tiles, for zen_product.hip and zen_orthogonal.hip.
//
//   D[i, j] = sum over k of A[i, k] B[k, j],   A and B in 16 bits, sums in fp32 (MFMA 16x16x32)
//
// A workgroup owns a tile of D and walks k in steps of 64.  A step's pieces of A and B come straight into LDS (buffer
// loads with an LDS destination, 16 bytes a lane); two buffers take turns, so a step's loads are in flight while the step before
// it is multiplied.  Each operand may be stored with k contiguous (rows of k) or with k as the stride (rows of i or j):
// the first is read from LDS 16 bytes a lane, the second by transposing reads (ds_read_b64_tr_b16), so no operand is ever
// transposed in memory.  The range check of the buffer loads puts zeros where the tile hangs over the operand's end.
//
// LDS layout: a row of 64 k is eight 16-byte pieces; the piece k / 8 of row r lies in place (k / 8) ^ (r & 7), which
// spreads the eight rows that eight lanes read at once over all banks.  With k as the stride a row holds the tile's i or j,
// and piece c of row k lies in place c ^ ((k & 3) << 1): the four rows that sixteen lanes of a transposing read take lie
// in different banks.  The loads' LDS destination is one run of lanes, so the swizzle is in the addresses they read from.
#pragma once

#include "zen_common.h"

namespace zen {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr int kTileK = 64;
constexpr int64_t kMostLd = 1 << 21;  // a step's addresses, 256 rows at most, stay below 2^30
constexpr int kMostList = 32;  // matrices of separate addresses to a launch

struct MatOperand {
  const uint16_t *p[2];  // the matrix, and (split products) what its rounding to 16 bits left over
  int64_t ld;            // elements from row to row
  int64_t batch;         // elements from matrix to matrix
};

struct MatSize {
  int m, n, k;
  int tiles_m, tiles_n;
  int batch;
  int parts;  // 1: A B; 3: A B + A B' + A' B with the left-overs A', B'
};

// Addresses of a stack's matrices: base + b * stride, or a list.
struct MatList {
  char *base;
  int64_t stride;  // bytes
  int listed;
  char *at[kMostList];
  __device__ __forceinline__ char *of(int b) const { return listed ? at[b] : base + (int64_t)b * stride; }
};

template <int BM_, int BN_, int WM_, int WN_>
struct TileShape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;       // tile, waves down and across
  static constexpr int W = WM * WN, threads = W * 64;
  static constexpr int TM = BM / WM, TN = BN / WN;                   // a wave's part
  static constexpr int FM = TM / 16, FN = TN / 16;                   // its MFMA blocks
  static constexpr int stage_bytes = (BM + BN) * kTileK * 2;
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
  const char *base;      // of the next step
  int64_t left;          // bytes of the operand from there on
  int64_t step;          // bytes to the next step
  uint32_t voffset, soffset;
  int tail_chunk;        // KC: this lane's first k within the step

  // r0: first row (i or j) of the tile; rows_all: rows there are; k: the operand's k
  __device__ __forceinline__ void start(const uint16_t *p, int64_t ld, int64_t r0, int64_t rows_all, int k, int wave, int lane) {
    const int row = wave * rows + lane / row_lanes;
    const int slot = lane % row_lanes;
    if (KC) {
      const int chunk = slot ^ (row & 7);
      tail_chunk = chunk * 8;
      base = reinterpret_cast<const char *>(p + r0 * ld);
      left = ((rows_all - r0 - 1) * ld + ((k + 7) & ~7)) * 2;  // whole pieces: k is a multiple of 8, or ld has room
      voffset = (uint32_t)((row * ld + chunk * 8) * 2);
      step = kTileK * 2;
    } else {
      const int chunk = slot ^ ((row & 3) << 1);
      tail_chunk = 0;
      base = reinterpret_cast<const char *>(p + r0);
      left = (((int64_t)k - 1) * ld + ((rows_all - r0 + 1) & ~1ll)) * 2;  // whole words: the address is a multiple of 16
      voffset = (uint32_t)((row * ld + chunk * 8) * 2);
      step = kTileK * ld * 2;
    }
    soffset = (uint32_t)(W * rows * ld * 2);
  }

  // The loads of the step at `base`, whose first k is k0 of k, into `lds` (this operand's part of a buffer).
  __device__ __forceinline__ void load(uint16_t *lds, int k0, int k, int wave) {
    const int64_t most = 0x7fff0000ll;  // the addresses of a tile end below (kMostLd)
    const uint32_t records = left <= 0 ? 0u : (uint32_t)(left < most ? left : most);
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, (int)records, 0x00027000);
    const uint32_t vo = KC && k0 + kTileK > k && k0 + tail_chunk >= k ? 0x80000000u : voffset;
#pragma unroll
    for (int q = 0; q < loads; ++q)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (ZEN_LDS void *)(lds + (q * W + wave) * 512), 16, (int)vo,
                                               (int)(q * soffset), 0, 0);
    base += step;
    left -= step;
  }

  // The block of sixteen rows from row r0 of the tile (a multiple of 16) and k from kk * 32, as an MFMA operand.
  static __device__ __forceinline__ short8v read(const uint16_t *lds, int r0, int kk, int lane) {
    if (KC) {
      const int r = r0 + (lane & 15);
      const int chunk = (kk * 4 + (lane >> 4)) ^ (lane & 7);
      return *reinterpret_cast<const short8v *>(lds + r * kTileK + chunk * 8);
    }
    const int j = lane & 15;
    const int krow = kk * 32 + (lane >> 4) * 8 + (j >> 2);
    const int slot = ((r0 >> 3) ^ ((j >> 2) << 1)) + ((j & 3) >> 1);
    const uint16_t *at = lds + krow * R + slot * 8 + (j & 1) * 4;
    const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ZEN_LDS short4v *)(at));
    const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ZEN_LDS short4v *)(at + 4 * R));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

template <bool BF>
__device__ __forceinline__ float4v mfma(short8v a, short8v b, float4v c) {
  if (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// Row and column of tile t of the lower triangle, counted row by row.
__device__ __forceinline__ void triangle(int t, int &i, int &j) {
  i = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
  while ((int64_t)i * (i + 1) / 2 > t) --i;
  while ((int64_t)(i + 1) * (i + 2) / 2 <= t) ++i;
  j = t - (int)((int64_t)i * (i + 1) / 2);
}

// The launch's tiles: of the whole matrix, or of its lower triangle (SYM).  Workgroups go round the eight dies, whose
// L2s are apart: the tiles are dealt so that a die's are neighbours, four tile rows by all columns at a time.
template <bool SYM>
__device__ __forceinline__ void tile_of(const MatSize &s, int &b, int &ti, int &tj) {
  const int per = SYM ? s.tiles_m * (s.tiles_m + 1) / 2 : s.tiles_m * s.tiles_n;
  const int all = per * s.batch;
  int t = (int)blockIdx.x;
  const int die = t & 7, most = all >> 3, rest = all & 7;
  t = die * most + (die < rest ? die : rest) + (t >> 3);
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

template <class S, bool AK, bool BK, bool BF, bool SYM, class Epilogue>
__global__ __launch_bounds__(S::threads, 2) void k_tiles(MatSize size, MatOperand a, MatOperand b, Epilogue epilogue) {
  __shared__ __attribute__((aligned(1024))) uint16_t s_buf[S::stage_bytes];
  int z, ti, tj;
  tile_of<SYM>(size, z, ti, tj);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / S::WN, wn = wave % S::WN;
  using OpA = TileOperand<S::BM, AK, S::W>;
  using OpB = TileOperand<S::BN, BK, S::W>;
  OpA la;
  OpB lb;
  const int steps = (size.k + kTileK - 1) / kTileK, all = steps * size.parts;
  int at = 0, part = 0;  // what is loaded next: step of a part

  auto next = [&](uint16_t *buf) {
    if (at == 0) {
      la.start(a.p[part == 2] + z * a.batch, a.ld, (int64_t)ti * S::BM, size.m, size.k, wave, lane);
      lb.start(b.p[part == 1] + z * b.batch, b.ld, (int64_t)tj * S::BN, size.n, size.k, wave, lane);
    }
    la.load(buf, at * kTileK, size.k, wave);
    lb.load(buf + S::BM * kTileK, at * kTileK, size.k, wave);
    if (++at == steps) {
      at = 0;
      ++part;
    }
  };

  float4v acc[S::FM][S::FN];
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) acc[i][j] = float4v{0.f, 0.f, 0.f, 0.f};

  auto multiply = [&](const uint16_t *buf) {
#pragma unroll
    for (int kk = 0; kk < kTileK / 32; ++kk) {
      __builtin_amdgcn_sched_barrier(0);
      short8v fa[S::FM], fb[S::FN];
#pragma unroll
      for (int i = 0; i < S::FM; ++i) fa[i] = OpA::read(buf, wm * S::TM + i * 16, kk, lane);
#pragma unroll
      for (int j = 0; j < S::FN; ++j) fb[j] = OpB::read(buf + S::BM * kTileK, wn * S::TN + j * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int j = 0; j < S::FN; ++j) acc[i][j] = mfma<BF>(fb[j], fa[i], acc[i][j]);
    }
  };

  // A buffer is loaded again only behind the barrier that every wave reaches after its reads of it.
  if (all > 0) next(s_buf);
  int turn = 0;
  for (int t = 0; t < all; ++t) {
    __builtin_amdgcn_s_waitcnt(0xf70);  // vmcnt(0): this wave's loads are in LDS
    __syncthreads();
    if (t + 1 < all) next(s_buf + (turn ^ (S::stage_bytes / 2)));
    multiply(s_buf + turn);
    turn ^= S::stage_bytes / 2;
  }

  // A lane holds four neighbours of a row: row lane & 15 of a block, columns (lane >> 4) * 4 and on.
  const int row0 = ti * S::BM + wm * S::TM + (lane & 15), col0 = tj * S::BN + wn * S::TN + (lane >> 4) * 4;
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) epilogue.put(z, row0 + i * 16, col0 + j * 16, acc[i][j], SYM && ti != tj);
}

template <class S, bool AK, bool BK, bool BF, bool SYM, class Epilogue>
inline int launch_tiles(MatSize size, const MatOperand &a, const MatOperand &b, const Epilogue &e, hipStream_t stream) {
  size.tiles_m = (size.m + S::BM - 1) / S::BM;
  size.tiles_n = (size.n + S::BN - 1) / S::BN;
  const int64_t per = SYM ? (int64_t)size.tiles_m * (size.tiles_m + 1) / 2 : (int64_t)size.tiles_m * size.tiles_n;
  const int64_t blocks = per * size.batch;
  if (blocks > 0x7fffffffll) return fail(ZEN_EINVAL, "matrix product: too many tiles");
  k_tiles<S, AK, BK, BF, SYM, Epilogue><<<dim3((unsigned)blocks), dim3(S::threads), 0, stream>>>(size, a, b, e);
  ZEN_LAUNCH_CHECK("k_tiles");
  return ZEN_OK;
}

// ---------------------------------------------------------------- values of three types

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

// What goes out to a caller's matrix: out = gain * (alpha * acc + beta * (X + X')) + keep * res.
struct OutEpilogue {
  float alpha, beta, gain, keep;
  const _Float16 *x, *x_low;  // null: none
  int64_t x_ld, x_batch;
  int rows, cols;
  MatList out, res;             // res: listed < 0 for none
  int64_t out_rs, out_cs, res_rs, res_cs;
  int out_type, res_type;

  __device__ __forceinline__ void one(char *o, const char *r, int i, int j, float v) const {
    if (res.listed >= 0) v = gain * v + keep * load_value(r, i * res_rs + j * res_cs, res_type);
    else v *= gain;
    store_value(o, i * out_rs + j * out_cs, out_type, v);
  }

  __device__ __forceinline__ void put(int z, int i, int j, float4v acc, bool mirror) const {
    if (i >= rows) return;
    char *o = out.of(z);
    const char *r = res.listed >= 0 ? res.of(z) : nullptr;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (j + e >= cols) break;
      float v = alpha * acc[e];
      if (x) {
        const int64_t at = z * x_batch + (int64_t)i * x_ld + j + e;
        v += beta * ((float)x[at] + (float)x_low[at]);
      }
      one(o, r, i, j + e, v);
      if (mirror) one(o, r, j + e, i, v);
    }
  }
};

// What goes back to a workspace: d = alpha * acc + beta * (c + c') + diag on the diagonal, in one or two times 16 bits.
struct KeepEpilogue {
  float alpha, beta, diag;
  int diag_n;  // the diagonal's length
  const _Float16 *c, *c_low;
  _Float16 *d, *d_low;
  int64_t c_ld, c_batch, d_ld, d_batch;

  __device__ __forceinline__ void put(int z, int i, int j, float4v acc, bool mirror) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v = alpha * acc[e];
      if (c) {
        const int64_t at = z * c_batch + (int64_t)i * c_ld + j + e;
        v += beta * ((float)c[at] + (c_low ? (float)c_low[at] : 0.f));
      }
      if (i == j + e && i < diag_n) v += diag;
      const _Float16 h = (_Float16)v, l = (_Float16)(v - (float)h);
      const int64_t at = z * d_batch + (int64_t)i * d_ld + j + e, to = z * d_batch + (int64_t)(j + e) * d_ld + i;
      d[at] = h;
      if (d_low) d_low[at] = l;
      if (mirror) {
        d[to] = h;
        if (d_low) d_low[to] = l;
      }
    }
  }
};

// Matrices laid out for the tiles: `rows` x `cols` values at any strides become 16-bit rows of `ld` elements, zeros beyond
// `cols` and from `rows` to `rows_all` (zen_pack.hip).  Raw: the 16 bits as they are; else value * scale[matrix], in fp16 and, with
// `low`, what that rounding left over in fp16 again.
struct PackArgs {
  MatList in;
  int64_t rs, cs;
  int dtype;
  int rows, cols, rows_all;
  int batch;
  uint16_t *out, *low;
  int64_t ld, out_batch;
  const double *squares;  // null: raw.  Else `shares` sums of squares a matrix, and scale = unit / (root of their sum + eps)
  int shares;
  double eps;
  float unit;
};
int pack_matrices(const PackArgs &args, hipStream_t stream);

}  // namespace zen
