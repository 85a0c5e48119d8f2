// Momentum and update of an optimiser step, from a dense gradient or from ascending lists:
//   m' = mu m + g,   u = nesterov ? g + mu m' : m'
// One pass: the momentum is read and written once, the update written once.  Bound by memory.
//
// Lists: a wave owns kTile neighbouring elements.  A first launch walks the lists' indices, checks them and writes down where
// each tile's entries begin in each list; the second one adds a tile's entries in LDS, one list after the other (the LDS
// operations of a wave keep their order, so sums are taken in the order of the lists and repeat bit for bit), while
// the momentum is on its way.
#include "zen_tiles.h"

namespace zen {
namespace {

constexpr int kBlock = 256;
constexpr int kTile = 1024;            // elements to a wave: 4 KiB of LDS, so a compute unit holds 32 waves (2048: 454 instead of 406 us at
                                       // 200 M elements and 20 M entries)
constexpr int kPer = kTile / 64;       // to a lane
constexpr int kMarkPer = 4;            // entries to a lane of the marking launch
constexpr int kMarkGap = 8;            // more tiles than that between two entries are marked by the whole wave

// Eight neighbours, 16 bytes at a time.
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&out)[8]) {
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
  constexpr int per = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8 / per; ++i) {
    const vec v = __builtin_nontemporal_load(reinterpret_cast<const vec *>(p) + i);
#pragma unroll
    for (int e = 0; e < per; ++e) out[i * per + e] = (float)v[e];
  }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&in)[8]) {
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
  constexpr int per = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8 / per; ++i) {
    vec v;
#pragma unroll
    for (int e = 0; e < per; ++e) v[e] = (T)in[i * per + e];
    __builtin_nontemporal_store(v, reinterpret_cast<vec *>(p) + i);
  }
}

__device__ __forceinline__ void moved(float &m, float g, float mu, bool nesterov, float &u) {
  m = fmaf(mu, m, g);
  u = nesterov ? fmaf(mu, m, g) : m;
}

template <typename M, typename G, typename U, bool WIDE>
__global__ __launch_bounds__(kBlock) void k_momentum(M *momentum, const G *grad, int64_t n, float mu, bool nesterov, U *update) {
  const int64_t first = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * 8;
  if (WIDE && first + 8 <= n) {
    float m[8], g[8], u[8];
    load8(momentum + first, m);
    load8(grad + first, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) moved(m[e], g[e], mu, nesterov, u[e]);
    store8(momentum + first, m);
    store8(update + first, u);
    return;
  }
  for (int e = 0; e < 8; ++e) {
    const int64_t i = WIDE ? first + e : (int64_t)blockIdx.x * kBlock * 8 + e * kBlock + threadIdx.x;
    if (i >= n) break;
    float m = (float)momentum[i], u;
    moved(m, (float)grad[i], mu, nesterov, u);
    momentum[i] = (M)m;
    update[i] = (U)u;
  }
}

struct Lists {
  const void *idx[ZEN_MOMENTUM_LISTS_MOST], *val[ZEN_MOMENTUM_LISTS_MOST];
  const int64_t *count[ZEN_MOMENTUM_LISTS_MOST];
  uint32_t length[ZEN_MOMENTUM_LISTS_MOST];
  uint32_t first_block[ZEN_MOMENTUM_LISTS_MOST];  // of the marking launch
  int n;
};

// An entry writes its place down for the tiles behind the entry before it, up to its own; the place behind the last one for
// the rest (marks[list][tile], tiles + 1 of them).
template <typename I>
__global__ __launch_bounds__(kBlock) void k_marks(Lists lists, int64_t n, uint32_t tiles, uint32_t *__restrict__ marks,
                                                  int32_t *status) {
  int l = 0;  // the block's list
#pragma unroll
  for (int d = ZEN_MOMENTUM_LISTS_MOST / 2; d > 0; d >>= 1)
    if (l + d < lists.n && lists.first_block[l + d] <= blockIdx.x) l += d;
  const I *idx = static_cast<const I *>(lists.idx[l]);
  uint32_t length = lists.length[l];
  if (lists.count[l]) {
    const int64_t c = *lists.count[l];
    length = c < 0 ? 0u : c < (int64_t)length ? (uint32_t)c : length;
  }
  marks += (size_t)l * (tiles + 1);
  const uint32_t first = (blockIdx.x - lists.first_block[l]) * (kBlock * kMarkPer) + threadIdx.x;
  int64_t prev[kMarkPer], cur[kMarkPer];
#pragma unroll
  for (int u = 0; u < kMarkPer; ++u) {
    const uint32_t at = first + u * kBlock;
    prev[u] = at > 0 && at <= length ? (int64_t)idx[at - 1] : -1;
    cur[u] = at < length ? (int64_t)idx[at] : (int64_t)tiles * kTile;
  }
  bool any = false;
#pragma unroll
  for (int u = 0; u < kMarkPer; ++u) {
    const uint32_t at = first + u * kBlock;
    uint32_t from = 0, to = 0;
    const bool bad = at < length && (cur[u] >= n || cur[u] <= prev[u] || cur[u] < 0);
    any |= bad;
    if (at <= length && !bad && prev[u] >= -1 && prev[u] < n) {
      from = at > 0 ? (uint32_t)(prev[u] / kTile) + 1u : 0u;
      to = (uint32_t)(cur[u] / kTile) + 1u;
    }
    if (to > from && to - from <= kMarkGap)
      for (uint32_t t = from; t < to; ++t) marks[t] = at;
    uint64_t wide = __ballot(to > from && to - from > kMarkGap);
    while (wide) {
      const int who = __ffsll((unsigned long long)wide) - 1;
      wide &= wide - 1;
      const uint32_t f = (uint32_t)__shfl((int)from, who), e = (uint32_t)__shfl((int)to, who), a = (uint32_t)__shfl((int)at, who);
      for (uint32_t t = f + (threadIdx.x & 63); t < e; t += 64) marks[t] = a;
    }
  }
  if (__ballot(any) && (threadIdx.x & 63) == 0) atomicOr(status, ZEN_STAT_BAD_INDEX);
}

template <typename M, typename U, bool WIDE>
__global__ __launch_bounds__(kBlock) void k_momentum_lists(M *momentum, Lists lists, int idx64, int val_type, int64_t n,
                                                           uint32_t tiles, const uint32_t *__restrict__ marks, float mu,
                                                           bool nesterov, U *update, const int32_t *status) {
  __shared__ float s_sum[kBlock / 64][kTile];
  if (*status) return;  // a list that is none, or the call that made the lists said so of them all
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t tile = blockIdx.x * (kBlock / 64) + (uint32_t)wave;
  if (tile >= tiles) return;
  float *sum = s_sum[wave];
  const int64_t first = (int64_t)tile * kTile;
  const int64_t left = n - first;
  const bool whole = WIDE && left >= kTile;
  float m[kPer / 8][8];
  if (whole) {
#pragma unroll
    for (int i = 0; i < kPer / 8; ++i) load8(momentum + first + i * 512 + lane * 8, m[i]);
  }
  // where the tile's entries lie in list `lane`, and how many there are up to it
  uint32_t begin = 0, count = 0;
  if (lane < lists.n) {
    const uint32_t *at = marks + (size_t)lane * (tiles + 1) + tile;
    begin = at[0];
    count = at[1] - begin;
  }
  uint32_t upto = count;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t below = (uint32_t)__shfl_up((int)upto, d);
    if (lane >= d) upto += below;
  }
  const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
  if (total) {
#pragma unroll
    for (int i = 0; i < kPer / 4; ++i) reinterpret_cast<float4v *>(sum)[i * 64 + lane] = float4v{0.f, 0.f, 0.f, 0.f};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint32_t offset = begin - (upto - count);  // an entry's number to its place in the list
    for (uint32_t base = 0; base < total; base += 64) {
      const uint32_t e = base + (uint32_t)lane;
      // its list: the lanes whose lists end at or before it come first
      int l = 0;
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) {
        const uint32_t end = (uint32_t)__shfl((int)upto, l + d - 1);
        if (end <= e) l += d;
      }
      l = l > 63 ? 63 : l;
      const uint32_t at = e + (uint32_t)__shfl((int)offset, l);
      uint32_t off = kTile;
      float v = 0.f;
      if (e < total) {
        const int64_t i = idx64 ? static_cast<const int64_t *>(lists.idx[l])[at] : (int64_t)static_cast<const int32_t *>(lists.idx[l])[at];
        v = load_value(static_cast<const char *>(lists.val[l]), at, val_type);
        off = (uint32_t)(i - first);
      }
      const int last = __builtin_amdgcn_readlane(l, (int)(total - base < 64 ? total - base - 1 : 63));
      for (int p = __builtin_amdgcn_readlane(l, 0); p <= last; ++p)
        if (l == p && off < kTile) __hip_atomic_fetch_add(&sum[off], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  if (whole) {
#pragma unroll
    for (int i = 0; i < kPer / 8; ++i) {
      float g[8] = {}, u[8];
      if (total) {
        const float4v *s = reinterpret_cast<const float4v *>(sum + i * 512 + lane * 8);
        const float4v a = s[0], b = s[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = a[e], g[e + 4] = b[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) moved(m[i][e], g[e], mu, nesterov, u[e]);
      store8(momentum + first + i * 512 + lane * 8, m[i]);
      store8(update + first + i * 512 + lane * 8, u);
    }
    return;
  }
  for (int i = lane; i < kTile && i < left; i += 64) {
    float one = (float)momentum[first + i], u;
    moved(one, total ? sum[i] : 0.f, mu, nesterov, u);
    momentum[first + i] = (M)one;
    update[first + i] = (U)u;
  }
}

bool aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

uint32_t tiles_of(int64_t n) { return (uint32_t)((n + kTile - 1) / kTile); }

template <typename M, typename G, typename U>
int dense(void *momentum, const void *grad, int64_t n, float mu, int nesterov, void *update, hipStream_t s) {
  const int64_t blocks = ceil_div(n, kBlock * 8);
  if (blocks > kMostThreads / kBlock) return fail(ZEN_EINVAL, "zen_momentum: too many elements");
  M *m = static_cast<M *>(momentum);
  const G *g = static_cast<const G *>(grad);
  U *u = static_cast<U *>(update);
  if (aligned(m) && aligned(g) && aligned(u))
    k_momentum<M, G, U, true><<<dim3((unsigned)blocks), dim3(kBlock), 0, s>>>(m, g, n, mu, nesterov != 0, u);
  else
    k_momentum<M, G, U, false><<<dim3((unsigned)blocks), dim3(kBlock), 0, s>>>(m, g, n, mu, nesterov != 0, u);
  ZEN_LAUNCH_CHECK("k_momentum");
  return ZEN_OK;
}

template <typename M, typename G>
int dense(void *momentum, const void *grad, int64_t n, float mu, int nesterov, void *update, int type, hipStream_t s) {
  if (type == ZEN_F32) return dense<M, G, float>(momentum, grad, n, mu, nesterov, update, s);
  if (type == ZEN_BF16) return dense<M, G, __bf16>(momentum, grad, n, mu, nesterov, update, s);
  return dense<M, G, _Float16>(momentum, grad, n, mu, nesterov, update, s);
}

template <typename M>
int dense(void *momentum, const void *grad, int grad_type, int64_t n, float mu, int nesterov, void *update, int type, hipStream_t s) {
  if (grad_type == ZEN_F32) return dense<M, float>(momentum, grad, n, mu, nesterov, update, type, s);
  if (grad_type == ZEN_BF16) return dense<M, __bf16>(momentum, grad, n, mu, nesterov, update, type, s);
  return dense<M, _Float16>(momentum, grad, n, mu, nesterov, update, type, s);
}

template <typename M, typename U>
int from_lists(void *momentum, const Lists &lists, int idx64, int val_type, int64_t n, const uint32_t *marks, float mu,
               int nesterov, void *update, const int32_t *status, hipStream_t s) {
  const uint32_t tiles = tiles_of(n);
  const dim3 grid((tiles + kBlock / 64 - 1) / (kBlock / 64));
  M *m = static_cast<M *>(momentum);
  U *u = static_cast<U *>(update);
  if (aligned(m) && aligned(u))
    k_momentum_lists<M, U, true><<<grid, dim3(kBlock), 0, s>>>(m, lists, idx64, val_type, n, tiles, marks, mu, nesterov != 0, u, status);
  else
    k_momentum_lists<M, U, false><<<grid, dim3(kBlock), 0, s>>>(m, lists, idx64, val_type, n, tiles, marks, mu, nesterov != 0, u, status);
  ZEN_LAUNCH_CHECK("k_momentum_lists");
  return ZEN_OK;
}

template <typename M>
int from_lists(void *momentum, const Lists &lists, int idx64, int val_type, int64_t n, const uint32_t *marks, float mu,
               int nesterov, void *update, int type, const int32_t *status, hipStream_t s) {
  if (type == ZEN_F32) return from_lists<M, float>(momentum, lists, idx64, val_type, n, marks, mu, nesterov, update, status, s);
  if (type == ZEN_BF16) return from_lists<M, __bf16>(momentum, lists, idx64, val_type, n, marks, mu, nesterov, update, status, s);
  return from_lists<M, _Float16>(momentum, lists, idx64, val_type, n, marks, mu, nesterov, update, status, s);
}

bool known(int type) { return type == ZEN_F32 || type == ZEN_BF16 || type == ZEN_F16; }

}  // namespace
}  // namespace zen

extern "C" {

int zen_momentum(void *momentum, int momentum_dtype, const void *grad, int grad_dtype, int64_t n, float mu, int nesterov,
                 void *update, int update_dtype, void *stream) {
  using namespace zen;
  if (n < 0) return fail(ZEN_EINVAL, "zen_momentum: negative size");
  if ((momentum_dtype != ZEN_F32 && momentum_dtype != ZEN_BF16) || !known(grad_dtype) || !known(update_dtype))
    return fail(ZEN_EINVAL, "zen_momentum: momentum is fp32 or bf16, gradient and update fp32, bf16 or fp16");
  if (n == 0) return ZEN_OK;
  if (!momentum || !grad || !update) return fail(ZEN_EINVAL, "zen_momentum: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (momentum_dtype == ZEN_F32) return dense<float>(momentum, grad, grad_dtype, n, mu, nesterov, update, update_dtype, s);
  return dense<__bf16>(momentum, grad, grad_dtype, n, mu, nesterov, update, update_dtype, s);
}

size_t zen_momentum_lists_workspace(int64_t n, int lists) {
  if (n <= 0 || n > 0x7fffffffll || lists < 1 || lists > ZEN_MOMENTUM_LISTS_MOST) return 0;
  return (size_t)lists * (zen::tiles_of(n) + 1) * sizeof(uint32_t);
}

int zen_momentum_lists(void *momentum, int momentum_dtype, const void *const *idx, int idx64, const void *const *val,
                       int val_dtype, const int64_t *lengths, const int64_t *const *counts, int lists, int64_t n, float mu,
                       int nesterov, void *update, int update_dtype, void *workspace, size_t workspace_bytes,
                       int32_t *status, void *stream) {
  using namespace zen;
  if (n < 0 || n > 0x7fffffffll) return fail(ZEN_EINVAL, "zen_momentum_lists: need 0 <= n < 2^31");
  if (lists < 1 || lists > ZEN_MOMENTUM_LISTS_MOST) return fail(ZEN_EINVAL, "zen_momentum_lists: 1 to 64 lists");
  if ((momentum_dtype != ZEN_F32 && momentum_dtype != ZEN_BF16) || !known(val_dtype) || !known(update_dtype))
    return fail(ZEN_EINVAL, "zen_momentum_lists: momentum is fp32 or bf16, values and update fp32, bf16 or fp16");
  if (!idx || !val || !lengths || !status) return fail(ZEN_EINVAL, "zen_momentum_lists: null pointer");
  Lists all = {};
  all.n = lists;
  uint64_t blocks = 0;
  for (int l = 0; l < lists; ++l) {
    if (lengths[l] < 0 || lengths[l] > 0x7fffffffll) return fail(ZEN_EINVAL, "zen_momentum_lists: a list's length is out of range");
    if (lengths[l] > 0 && (!idx[l] || !val[l])) return fail(ZEN_EINVAL, "zen_momentum_lists: null pointer");
    all.idx[l] = idx[l];
    all.val[l] = val[l];
    all.count[l] = counts ? counts[l] : nullptr;
    all.length[l] = (uint32_t)lengths[l];
    all.first_block[l] = (uint32_t)blocks;
    blocks += (uint64_t)lengths[l] / (kBlock * kMarkPer) + 1;  // one more than the entries: the place behind the last one
  }
  if (blocks > (uint64_t)kMostThreads / kBlock) return fail(ZEN_EINVAL, "zen_momentum_lists: too many entries");
  if (n == 0) {
    for (int l = 0; l < lists; ++l)
      if (lengths[l] > 0) return fail(ZEN_EINVAL, "zen_momentum_lists: entries for no elements");
    return ZEN_OK;
  }
  if (!momentum || !update || !workspace) return fail(ZEN_EINVAL, "zen_momentum_lists: null pointer");
  if (workspace_bytes < zen_momentum_lists_workspace(n, lists)) return fail(ZEN_EWORKSPACE, "zen_momentum_lists: workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint32_t *marks = static_cast<uint32_t *>(workspace);
  if (idx64) k_marks<int64_t><<<dim3((unsigned)blocks), dim3(kBlock), 0, s>>>(all, n, tiles_of(n), marks, status);
  else k_marks<int32_t><<<dim3((unsigned)blocks), dim3(kBlock), 0, s>>>(all, n, tiles_of(n), marks, status);
  ZEN_LAUNCH_CHECK("k_marks");
  if (momentum_dtype == ZEN_F32)
    return from_lists<float>(momentum, all, idx64, val_dtype, n, marks, mu, nesterov, update, update_dtype, status, s);
  return from_lists<__bf16>(momentum, all, idx64, val_dtype, n, marks, mu, nesterov, update, update_dtype, status, s);
}

}  // extern "C"
