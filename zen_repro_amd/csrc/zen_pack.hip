// Matrices at any strides, laid out in rows of 16 bits for zen_tiles.h (see PackArgs there).  Bound by memory: one read, one
// or two writes.  A workgroup takes 64 x 64 elements; the reads go along whichever stride is the shorter, the writes along
// the rows, with LDS in between.
#include "zen_tiles.h"

namespace zen {
namespace {

constexpr int kSide = 64;

__global__ __launch_bounds__(256) void k_pack(PackArgs p) {
  __shared__ uint32_t s_tile[kSide][kSide + 1];
  __shared__ double s_sum[4];
  const int z = blockIdx.z, i0 = blockIdx.y * kSide, j0 = blockIdx.x * kSide;
  const int tid = threadIdx.x;
  double scale = 1.0;
  if (p.squares) {
    double sum = 0.0;
    for (int i = tid; i < p.shares; i += 256) sum += p.squares[(int64_t)z * p.shares + i];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
    __syncthreads();
    sum = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    const double norm = sqrt(sum) + p.eps;
    scale = norm == 0.0 ? 0.0 : (double)p.unit / norm;  // nothing but zeros, and eps is zero
  }
  const char *in = p.in.of(z);
  const bool across = p.cs <= p.rs;  // neighbours in memory are neighbours of a row
#pragma unroll
  for (int q = 0; q < kSide * kSide / 256; ++q) {
    const int at = q * 256 + tid, fast = at & 63, slow = at >> 6;
    const int i = across ? slow : fast, j = across ? fast : slow;
    uint32_t v = 0;
    if (i0 + i < p.rows && j0 + j < p.cols) {
      const int64_t from = (i0 + i) * p.rs + (j0 + j) * p.cs;
      v = p.squares ? __float_as_uint(load_value(in, from, p.dtype)) : (uint32_t)reinterpret_cast<const uint16_t *>(in)[from];
    }
    s_tile[i][j] = v;
  }
  __syncthreads();
  const int64_t from = (int64_t)z * p.out_batch;
  const auto write = [&](uint16_t *out, uint16_t *low, int64_t ld, int row0, int rows, int col0, bool turned) {
#pragma unroll
    for (int q = 0; q < kSide * kSide / 512; ++q) {  // two columns a lane
      const int at = q * 256 + tid, j = (at & 31) * 2, i = at >> 5;
      if (row0 + i >= rows || col0 + j >= ld) continue;
      uint32_t word = 0, rest = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t raw = turned ? s_tile[j + e][i] : s_tile[i][j + e];
        if (!p.squares) {
          word |= raw << (16 * e);
          continue;
        }
        const float v = (float)((double)__uint_as_float(raw) * scale);  // in fp64: a tiny update's scale is beyond fp32
        const _Float16 h = (_Float16)v, l = (_Float16)(v - (float)h);
        word |= (uint32_t)__builtin_bit_cast(uint16_t, h) << (16 * e);
        rest |= (uint32_t)__builtin_bit_cast(uint16_t, l) << (16 * e);
      }
      const int64_t to = from + (int64_t)(row0 + i) * ld + col0 + j;  // ld is even
      *reinterpret_cast<uint32_t *>(out + to) = word;
      if (low) *reinterpret_cast<uint32_t *>(low + to) = rest;
    }
  };
  write(p.out, p.low, p.ld, i0, p.rows_all, j0, false);
  if (p.turned) write(p.turned, p.turned_low, p.rows_all, j0, (int)p.ld, i0, true);
}

}  // namespace

int pack_matrices(const PackArgs &p, hipStream_t stream) {
  const int64_t across = ceil_div(p.ld, kSide), down = ceil_div(p.rows_all, kSide);
  if (across > 0x7fffffffll || down > 65535 || p.batch > 65535) return fail(ZEN_EINVAL, "matrix product: too many rows");
  k_pack<<<dim3((unsigned)across, (unsigned)down, (unsigned)p.batch), dim3(256), 0, stream>>>(p);
  ZEN_LAUNCH_CHECK("k_pack");
  return ZEN_OK;
}

}  // namespace zen
