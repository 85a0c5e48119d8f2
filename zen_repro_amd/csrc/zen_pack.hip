// Matrices at any strides, laid out in rows for zen_tiles.h (see PackArgs there).  Bound by memory: one read, one write.  A
// workgroup takes 64 x 64 elements; the reads go along whichever stride is the shorter, the writes along the rows, with
// LDS in between.  No branch stands around a read, so a lane's sixteen are on their way together (208 workgroups: 5.9 us, 7.9 with
// branches).
#include "zen_tiles.h"

namespace zen {
namespace {

constexpr int kSide = 64;

struct Two {
  PackArgs of[2];
  uint32_t blocks[2], across[2], down[2];  // workgroups: 31 bits in all
};

__global__ __launch_bounds__(256) void k_pack(Two two) {
  __shared__ uint16_t s_tile[kSide][kSide + 2];  // a row is 33 words: columns lie in different banks
  const int which = blockIdx.x >= two.blocks[0];
  const PackArgs &p = two.of[which];
  const uint32_t at_block = blockIdx.x - (which ? two.blocks[0] : 0), line = at_block / two.across[which];
  const int tid = threadIdx.x, j0 = (int)(at_block - line * two.across[which]) * kSide;
  const int z = (int)(line / two.down[which]), i0 = (int)(line - z * two.down[which]) * kSide;
  const uint16_t *in = reinterpret_cast<const uint16_t *>(p.in.of(z));
  const bool across = p.cs <= p.rs;  // neighbours in memory are neighbours of a row
  uint16_t v[kSide * kSide / 256];
#pragma unroll
  for (int q = 0; q < kSide * kSide / 256; ++q) {  // all on their way together: what lies beyond the matrix reads its last row or column
    const int at = q * 256 + tid, fast = at & 63, slow = at >> 6;
    const int i = i0 + (across ? slow : fast), j = j0 + (across ? fast : slow);
    v[q] = in[(i < p.rows ? i : p.rows - 1) * p.rs + (j < p.cols ? j : p.cols - 1) * p.cs];
  }
#pragma unroll
  for (int q = 0; q < kSide * kSide / 256; ++q) {
    const int at = q * 256 + tid, fast = at & 63, slow = at >> 6;
    const int i = across ? slow : fast, j = across ? fast : slow;
    s_tile[i][j] = i0 + i < p.rows && j0 + j < p.cols ? v[q] : 0;
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
  int64_t all = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t across = ceil_div(args[i].ld, kSide), down = ceil_div(args[i].rows, kSide);
    if (down * args[i].batch > 0x7fffffffll / across) return fail(ZEN_EINVAL, "matrix product: too many rows");
    two.of[i] = args[i];
    two.across[i] = (uint32_t)across;
    two.down[i] = (uint32_t)down;
    two.blocks[i] = (uint32_t)(across * down * args[i].batch);
    all += two.blocks[i];
  }
  if (all > kMostThreads / 256) return fail(ZEN_EINVAL, "matrix product: too many rows");
  k_pack<<<dim3((unsigned)all), dim3(256), 0, stream>>>(two);
  ZEN_LAUNCH_CHECK("k_pack");
  return ZEN_OK;
}

}  // namespace zen
