// Matrices at any strides, laid out in rows for zen_tiles.h (see PackArgs there).  Bound by memory: one read, one write.  A
// workgroup takes 64 x 64 elements; the reads go along whichever stride is the shorter, the writes along the rows, with
// LDS in between.
#include "zen_tiles.h"

namespace zen {
namespace {

constexpr int kSide = 64;

struct Two {
  PackArgs of[2];
  int64_t blocks[2], across[2], down[2];
};

__global__ __launch_bounds__(256) void k_pack(Two two) {
  __shared__ uint16_t s_tile[kSide][kSide + 2];  // a row is 33 words: columns lie in different banks
  const int which = (int64_t)blockIdx.x >= two.blocks[0];
  const PackArgs &p = two.of[which];
  int64_t at_block = (int64_t)blockIdx.x - (which ? two.blocks[0] : 0);
  const int tid = threadIdx.x, j0 = (int)(at_block % two.across[which]) * kSide;
  at_block /= two.across[which];
  const int i0 = (int)(at_block % two.down[which]) * kSide, z = (int)(at_block / two.down[which]);
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

int pack_matrices(const PackArgs *args, int count, hipStream_t stream) {
  Two two = {};
  for (int i = 0; i < count; ++i) {
    two.of[i] = args[i];
    two.across[i] = ceil_div(args[i].ld, kSide);
    two.down[i] = ceil_div(args[i].rows, kSide);
    if (two.down[i] > 0x7fffffffll / two.across[i]) return fail(ZEN_EINVAL, "matrix product: too many rows");
    two.blocks[i] = two.across[i] * two.down[i] * args[i].batch;
  }
  if (two.blocks[0] + two.blocks[1] > 0x7fffffffll) return fail(ZEN_EINVAL, "matrix product: too many rows");
  k_pack<<<dim3((unsigned)(two.blocks[0] + two.blocks[1])), dim3(256), 0, stream>>>(two);
  ZEN_LAUNCH_CHECK("k_pack");
  return ZEN_OK;
}

}  // namespace zen
