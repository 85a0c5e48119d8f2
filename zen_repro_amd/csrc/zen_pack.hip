// Matrices at any strides, laid out in rows for zen_tiles.h (see PackArgs there).  Bound by memory: one read, one write.  A
// workgroup takes 64 x 64 elements; the reads go along whichever stride is the shorter, the writes along the rows, with
// LDS in between.
#include "zen_tiles.h"

namespace zen {
namespace {

constexpr int kSide = 64;

__global__ __launch_bounds__(256) void k_pack(PackArgs p) {
  __shared__ uint16_t s_tile[kSide][kSide + 2];  // a row is 33 words: columns lie in different banks
  const int z = blockIdx.z, i0 = blockIdx.y * kSide, j0 = blockIdx.x * kSide, tid = threadIdx.x;
  const uint16_t *in = reinterpret_cast<const uint16_t *>(p.in.of(z));
  const bool across = p.cs <= p.rs;  // neighbours in memory are neighbours of a row
#pragma unroll
  for (int q = 0; q < kSide * kSide / 256; ++q) {
    const int at = q * 256 + tid, fast = at & 63, slow = at >> 6;
    const int i = across ? slow : fast, j = across ? fast : slow;
    s_tile[i][j] = i0 + i < p.rows && j0 + j < p.cols ? in[(i0 + i) * p.rs + (j0 + j) * p.cs] : 0;
  }
  __syncthreads();
  uint16_t *out = p.out + (int64_t)z * p.out_batch;
#pragma unroll
  for (int q = 0; q < kSide * kSide / 512; ++q) {  // two columns a lane
    const int at = q * 256 + tid, j = (at & 31) * 2, i = at >> 5;
    if (i0 + i < p.rows && j0 + j < p.ld)  // ld is even
      *reinterpret_cast<uint32_t *>(out + (int64_t)(i0 + i) * p.ld + j0 + j) = *reinterpret_cast<const uint32_t *>(&s_tile[i][j]);
  }
}

}  // namespace

int pack_matrices(const PackArgs &p, hipStream_t stream) {
  const int64_t across = ceil_div(p.ld, kSide), down = ceil_div(p.rows, kSide);
  if (across > 0x7fffffffll || down > 65535 || p.batch > 65535) return fail(ZEN_EINVAL, "matrix product: too many rows");
  k_pack<<<dim3((unsigned)across, (unsigned)down, (unsigned)p.batch), dim3(256), 0, stream>>>(p);
  ZEN_LAUNCH_CHECK("k_pack");
  return ZEN_OK;
}

}  // namespace zen
