// Updates made orthogonal by Newton-Schulz steps:  X <- a X + (b A + c A A) X,  A = X X^T,  from X = U / (|U| + eps).
//
// A step is three products (zen_tiles.h).  A and A A are symmetric: the tiles of the lower triangle are computed and
// mirrored.  X is kept with rows <= columns (a tall update is turned when it is laid out, its result when it goes out), and its
// transpose beside it: every operand is then read along k, the quickest way (4096 x 4096: 118 us a product against 141 us
// with a transposing read, for 7 us of writing).
// Bound by the matrix instructions: 3 m m n + m m m flops a step.
//
// Everything is held as fp16 times a unit of 2^10: a value of 1 is far from fp16's limits and what rounding leaves over is far
// from its denormals (coefficients that can take values beyond 63 get smaller units, see Units).  Why fp16 and not bf16:
// entries stay below 2 or so, range is not needed, and the iteration amplifies rounding (errors against 64 bits, Gaussian
// update 1024 x 1024: bf16 2e-2, fp16 1e-3).  Where a direction starts small it grows by `a` a step, and so does the noise
// that rounding X adds to it; so X is carried on as two fp16 (22 bits) and only the products see 11 of them.  The last two
// steps are written as X + (b A + c A A + (a - 1) I) X: there the singular values are near 1, the bracket is near zero, and
// so is what rounding it does.  The diagonals of A and of the bracket are kept whole (KeepEpilogue).  Before its own
// rounding a result is then off by 0.24 to 1.24e-3 from 64 rows on (64 x 64 to 1024 x 4096; a single strong direction does
// best, a square Gaussian update worst, and the more rows the better), which is less than rounding it to bf16 does, 1.66e-3.
// With `precise` (results of fp32 and fp16) the products see 22 bits of every operand too: A B + A B' + A' B, what is left
// out is below 2^-22; off by half to twice what products in fp32 are (twice: one strong direction, whose fellows grow out
// of X's 22 bits).
#include <cmath>

#include "zen_tiles.h"

namespace zen {
namespace {

constexpr double kUnit = 1024.0, kMostHalf = 65504.0;
constexpr int kSquareBlock = 256;
constexpr int kMostShares = 1024;  // workgroups to a matrix' sum of squares

// Sums of squares in fp64 (an fp32 square overflows from 2^64 on), one a workgroup, in a fixed order.  `slow` lines of `fast`
// values; wide: a line is contiguous and begins at a multiple of 16 bytes.  Bound by the read.
__global__ __launch_bounds__(kSquareBlock) void k_squares(MatList in, int64_t slow_stride, int64_t fast_stride, int dtype, int slow,
                                                          int fast, int wide, int shares, double *__restrict__ sums) {
  __shared__ double s_sum[kSquareBlock / 64];
  const int share = blockIdx.x, z = blockIdx.y;
  const char *p = in.of(z);
  const int64_t pieces = (fast + 7) / 8, all = pieces * slow;
  const int64_t first = all * share / shares, last = all * (share + 1) / shares;
  double even = 0.0, odd = 0.0;
#pragma unroll 2
  for (int64_t at = first + threadIdx.x; at < last; at += kSquareBlock) {
    const int64_t i = at / pieces;
    const int j = (int)(at - i * pieces) * 8;
    const float8v v = wide && j + 8 <= fast ? load_eight(p, i * slow_stride + j, dtype) : load_line(p, i * slow_stride, fast_stride, j, fast, dtype);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      even = fma((double)v[e], (double)v[e], even);
      odd = fma((double)v[e + 1], (double)v[e + 1], odd);
    }
  }
  double sum = even + odd;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all_waves = 0.0;
    for (int w = 0; w < kSquareBlock / 64; ++w) all_waves += s_sum[w];
    sums[(int64_t)z * shares + share] = all_waves;
  }
}

constexpr int kLaySide = 64;

// X = U / (|U| + eps) and its transpose, in fp16 and what that leaves over, in whole steps of the products with zeros behind the
// matrix' own (fp64: a tiny update's scale is beyond fp32).  A workgroup takes 64 lines of 64 neighbours: one of the two goes out as
// it was read, the other through LDS.  Bound by memory: one read, three or four writes.
struct LayOut {
  MatList in;
  int64_t slow_stride, fast_stride;
  int dtype, slow, fast, wide;
  _Float16 *along, *along_low;  // lines as they lie in memory, of along_ld; null low: not kept
  _Float16 *across, *across_low;
  int64_t along_ld, across_ld, batch;
  const double *squares;
  int shares;
  double eps;
};

__device__ __forceinline__ void put_halves(_Float16 *hi, _Float16 *low, int64_t at, float8v v) {
  const half8v h = __builtin_convertvector(v, half8v);
  *reinterpret_cast<half8v *>(hi + at) = h;
  if (low) *reinterpret_cast<half8v *>(low + at) = __builtin_convertvector(v - widen(h), half8v);
}

__global__ __launch_bounds__(256) void k_lay_out(LayOut p) {
  __shared__ float s_tile[kLaySide][kLaySide + 1];
  __shared__ double s_sum[4];
  const int z = blockIdx.z, f0 = blockIdx.x * kLaySide, s0 = blockIdx.y * kLaySide, tid = threadIdx.x;
  const char *in = p.in.of(z);
  float8v v[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int s = s0 + q * 32 + tid / 8, f = f0 + tid % 8 * 8;
    const int64_t line = (s < p.slow ? s : p.slow - 1) * p.slow_stride;
    v[q] = p.wide && f + 8 <= p.fast ? load_eight(in, line + f, p.dtype) : load_line(in, line, p.fast_stride, f, p.fast, p.dtype);
    if (s >= p.slow) v[q] = float8v{};
  }
  double sum = 0.0;
  for (int i = tid; i < p.shares; i += 256) sum += p.squares[(int64_t)z * p.shares + i];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
  __syncthreads();
  const double norm = sqrt((s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3])) + p.eps;
  const double scale = norm == 0.0 ? 0.0 : kUnit / norm;  // nothing but zeros, and eps is zero
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int s = q * 32 + tid / 8, f = tid % 8 * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[q][e] = (float)((double)v[q][e] * scale);
      s_tile[s][f + e] = v[q][e];
    }
    put_halves(p.along, p.along_low, z * p.batch + (s0 + s) * p.along_ld + f0 + f, v[q]);
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int f = q * 32 + tid / 8, s = tid % 8 * 8;
    float8v w;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = s_tile[s + e][f];
    put_halves(p.across, p.across_low, z * p.batch + (f0 + f) * p.across_ld + s0 + s, w);
  }
}

// A chunk's buffers: `batch` matrices at once.  Rows and columns are whole steps of the products; what lies behind the
// matrix' own is zero and stays so.
struct Room {
  int64_t m, n;
  int batch;
  _Float16 *x, *x_low;              // X, carried on in place
  _Float16 *turned[2], *turned_low[2];  // its transpose, for the products: they take turns
  _Float16 *a, *a_low, *b, *b_low;
  float *a_diag, *b_diag;  // what rounding their diagonals left over, where they have no low halves
  double *squares;
  float *partial;  // sums of tiles that are split
  TilePlan gram, square, apply;
  size_t bytes;
};

// What a step's matrices are held times, powers of two: an entry is at most its matrix' largest singular value, X's begin at
// one at most, and a step takes an s from [0, top] to p(s) = s (a + b s^2 + c s^4) and X X^T's s^2 to the bracket's value.
struct Units {
  double x, a, b;  // of X before the step, A and the bracket
};

double unit_of(double most) {
  double unit = kUnit;
  while (unit * most > kMostHalf * 0.98) unit *= 0.5;  // (roundings on the way are far less than a fiftieth)
  return unit;
}

// The largest |f| on [0, end], from its values at both ends and at the roots of its derivative r0 + r1 y + r2 y^2 in between.
template <class F>
double most_of(F f, double end, double r0, double r1, double r2) {
  double most = fmax(fabs(f(0.0)), fabs(f(end)));
  const auto look = [&](double y) {
    if (y > 0 && y < end) most = fmax(most, fabs(f(y)));
  };
  if (r2 == 0.0) {
    if (r1 != 0.0) look(-r0 / r1);
  } else if (const double d = r1 * r1 - 4 * r2 * r0; d >= 0) {
    const double q = -0.5 * (r1 + copysign(sqrt(d), r1));  // no cancellation
    look(q / r2);
    if (q != 0.0) look(r0 / q);
  }
  return most;
}

// Of the step that begins with singular values up to `top`, which becomes the next one's.  Without an answer where a unit would be below
// one (coefficients that are not finite among them): values around one would come too near to fp16's denormals.
bool units_of(double a, double b, double c, bool near, double &top, Units &u) {
  const double end = top * top;
  const double shift = near ? a - 1.0 : 0.0;
  const double bracket = most_of([&](double y) { return shift + y * (b + c * y); }, end, b, 2 * c, 0.0);
  if (!(top < kMostHalf / 2 && end < kMostHalf / 2 && bracket < kMostHalf / 2 && std::isfinite(a))) return false;
  u = {unit_of(top), unit_of(end), unit_of(bracket)};
  top = most_of([&](double y) { return sqrt(y) * (a + y * (b + c * y)); }, end, a, 3 * b, 5 * c);
  return true;
}

bool holds(const zen_orthogonal_args &p) {
  double top = 1.0;
  Units u;
  for (int step = 0; step < p.steps; ++step)
    if (!units_of(p.a, p.b, p.c, step >= p.steps - 2, top, u)) return false;
  return true;
}

int shares_of(int64_t rows, int64_t cols) {
  const int64_t want = rows * cols / 4096 + 1;
  return (int)(want < kMostShares ? want : kMostShares);
}

int chunk_of(int64_t m, int64_t n, int64_t count, bool precise) {
  // enough matrices at once to fill the card, in no more room than 2 GiB (and the split sums') where one matrix does
  const int64_t bytes = 2 * (precise ? 6 * m * n + 4 * m * m : 4 * m * n + 2 * m * m);
  int64_t most = (1ll << 31) / bytes;
  if (most < 1) most = 1;
  if (most > kMostList) most = kMostList;
  return (int)(count < most ? count : most);
}

Room room_for(int64_t rows, int64_t cols, int64_t count, bool precise, void *at) {
  Room r = {};
  const int64_t small = rows < cols ? rows : cols, large = rows < cols ? cols : rows;
  r.m = ceil_div(small, kTileK) * kTileK;
  r.n = ceil_div(large, kTileK) * kTileK;
  r.batch = chunk_of(r.m, r.n, count, precise);
  Carver cv(at);
  const size_t xs = (size_t)r.batch * r.m * r.n, as = (size_t)r.batch * r.m * r.m;
  r.x = cv.take<_Float16>(xs);
  r.x_low = cv.take<_Float16>(xs);
  r.turned[0] = cv.take<_Float16>(xs);
  r.turned[1] = cv.take<_Float16>(xs);
  r.a = cv.take<_Float16>(as);
  r.b = cv.take<_Float16>(as);
  if (precise) {
    r.turned_low[0] = cv.take<_Float16>(xs);
    r.turned_low[1] = cv.take<_Float16>(xs);
    r.a_low = cv.take<_Float16>(as);
    r.b_low = cv.take<_Float16>(as);
  } else {
    r.a_diag = cv.take<float>((size_t)r.batch * r.m);
    r.b_diag = cv.take<float>((size_t)r.batch * r.m);
  }
  r.squares = cv.take<double>((size_t)r.batch * shares_of(rows, cols));
  const int parts = precise ? 3 : 1;
  r.gram = plan_tiles(r.m, r.m, r.n, parts, r.batch, true, true);
  r.square = plan_tiles(r.m, r.m, r.m, parts, r.batch, true, true);
  r.apply = plan_tiles(r.m, r.n, r.m, parts, r.batch, false, true);
  size_t partial = r.gram.partial_bytes > r.square.partial_bytes ? r.gram.partial_bytes : r.square.partial_bytes;
  partial = partial > r.apply.partial_bytes ? partial : r.apply.partial_bytes;
  r.partial = cv.take<float>(partial / sizeof(float));
  r.bytes = cv.used;
  return r;
}

MatOperand operand(const _Float16 *p, const _Float16 *low, int64_t ld, int64_t batch) {
  return {{reinterpret_cast<const uint16_t *>(p), reinterpret_cast<const uint16_t *>(low ? low : p)}, ld, batch};
}

template <bool HALVES>
int chunk(const zen_orthogonal_args &p, const Room &r, int64_t first, int batch, hipStream_t s) {
  const bool turn = p.rows > p.cols;
  const int small = (int)(turn ? p.cols : p.rows), large = (int)(turn ? p.rows : p.cols);
  const int shares = shares_of(p.rows, p.cols);
  MatList in = {}, out = {};
  in.listed = out.listed = 1;
  for (int i = 0; i < batch; ++i) {
    in.at[i] = static_cast<char *>(const_cast<void *>(p.updates[first + i]));
    out.at[i] = static_cast<char *>(p.outs[first + i]);
  }
  const int64_t rs = turn ? p.update_cs : p.update_rs, cs = turn ? p.update_rs : p.update_cs;
  const bool across = cs <= rs;  // memory goes along X's rows
  const int slow = across ? small : large, fast = across ? large : small;
  const int64_t slow_stride = across ? rs : cs, fast_stride = across ? cs : rs;
  int wide = fast_stride == 1 && slow_stride * (p.update_dtype == ZEN_F32 ? 4 : 2) % 16 == 0;
  for (int i = 0; i < batch; ++i) wide &= (reinterpret_cast<uintptr_t>(in.at[i]) & 15u) == 0;
  k_squares<<<dim3((unsigned)shares, (unsigned)batch), dim3(kSquareBlock), 0, s>>>(in, slow_stride, fast_stride, p.update_dtype, slow,
                                                                                  fast, wide, shares, r.squares);
  ZEN_LAUNCH_CHECK("k_squares");
  LayOut lay = {in, slow_stride, fast_stride, p.update_dtype, slow, fast, wide, r.x, r.x_low, r.turned[0], r.turned_low[0],
                r.n, r.m, r.m * r.n, r.squares, shares, p.eps};
  if (!across) {
    lay.along = r.turned[0];
    lay.along_low = r.turned_low[0];
    lay.along_ld = r.m;
    lay.across = r.x;
    lay.across_low = r.x_low;
    lay.across_ld = r.n;
  }
  k_lay_out<<<dim3((unsigned)(lay.along_ld / kLaySide), (unsigned)(lay.across_ld / kLaySide), (unsigned)batch), dim3(256), 0, s>>>(lay);
  ZEN_LAUNCH_CHECK("k_lay_out");

  const int parts = HALVES ? 3 : 1;
  const int m = (int)r.m, n = (int)r.n;
  const int64_t mm = r.m * r.m, mn = r.m * r.n;
  const MatSize gram = {m, m, n, 0, 0, batch, parts, 1, nullptr}, square = {m, m, m, 0, 0, batch, parts, 1, nullptr},
                apply = {m, n, m, 0, 0, batch, parts, 1, nullptr};
  double top = 1.0;
  Units u, next;
  units_of(p.a, p.b, p.c, p.steps <= 2, top, next);
  for (int step = 0; step < p.steps; ++step) {
    const int at = step & 1;
    const bool near = step >= p.steps - 2;
    u = next;
    if (step + 1 < p.steps) units_of(p.a, p.b, p.c, step + 1 >= p.steps - 2, top, next);
    const MatOperand x = operand(r.x, HALVES ? r.x_low : nullptr, r.n, mn);
    const MatOperand xt = operand(r.turned[at], r.turned_low[at], r.m, mn);
    const MatOperand a = operand(r.a, r.a_low, r.m, mm), b = operand(r.b, r.b_low, r.m, mm);
    KeepEpilogue<kGram, HALVES> g = {};
    g.alpha = (float)(u.a / (u.x * u.x));
    g.rows = g.cols = m;
    g.d = r.a;
    g.d_low = r.a_low;
    g.ld = r.m;
    g.batch = mm;
    g.low = r.a_diag;
    g.low_batch = r.m;
    if (const int rc = run_tiles<true, true, false, true>(r.gram, r.partial, gram, x, x, g, s)) return rc;
    KeepEpilogue<kSquare, HALVES> q = {};
    q.alpha = (float)(p.c * (u.b / (u.a * u.a)));
    q.beta = (float)(p.b * (u.b / u.a));
    q.rows = q.cols = m;
    q.diag = near ? (float)((p.a - 1.f) * u.b) : 0.f;
    q.diag_n = small;
    q.c = r.a;
    q.c_low = r.a_low;
    q.d = r.b;
    q.d_low = r.b_low;
    q.ld = r.m;
    q.batch = mm;
    q.low = r.b_diag;
    q.from_low = r.a_diag;
    q.low_batch = r.m;
    if (const int rc = run_tiles<true, true, false, true>(r.square, r.partial, square, a, a, q, s)) return rc;
    if (step + 1 < p.steps) {
      KeepEpilogue<kApply, HALVES> e = {};
      e.alpha = (float)(next.x / (u.b * u.x));
      e.beta = (float)((near ? 1.f : p.a) * (next.x / u.x));
      e.rows = m;
      e.cols = n;
      e.c = e.d = r.x;
      e.c_low = e.d_low = r.x_low;
      e.ld = r.n;
      e.batch = e.t_batch = mn;
      e.t = r.turned[at ^ 1];
      e.t_low = r.turned_low[at ^ 1];
      e.t_ld = r.m;
      e.from_low = r.b_diag;
      e.low_batch = r.m;
      if (const int rc = run_tiles<true, true, false, false>(r.apply, r.partial, apply, b, xt, e, s)) return rc;
      continue;
    }
    OutEpilogue o = {};
    o.alpha = (float)(1.0 / (u.b * u.x));
    o.beta = (float)((near ? 1.f : p.a) / u.x);
    o.gain = p.weights ? -p.gain : 1.f;
    o.keep = p.keep;
    o.x = r.x;
    o.x_low = r.x_low;
    o.x_ld = r.n;
    o.x_batch = mn;
    o.row_low = r.b_diag;
    o.low_batch = r.m;
    o.rows = small;
    o.cols = large;
    o.out = out;
    o.out_rs = turn ? p.out_cs : p.out_rs;
    o.out_cs = turn ? p.out_rs : p.out_cs;
    o.out_type = p.out_dtype;
    const int64_t size = p.out_dtype == ZEN_F32 ? 4 : 2;
    o.lines = o.out_cs == 1 && o.out_rs * size % 16 == 0 ? 1 : o.out_rs == 1 && o.out_cs * size % 16 == 0 ? 2 : 0;
    for (int i = 0; i < batch; ++i)
      if (reinterpret_cast<uintptr_t>(out.at[i]) & 15u) o.lines = 0;
    o.res.listed = -1;
    if (p.weights) {
      o.res = o.out;
      o.res_rs = o.out_rs;
      o.res_cs = o.out_cs;
      o.res_type = o.out_type;
    }
    if (const int rc = run_tiles<true, true, false, false>(r.apply, r.partial, apply, b, xt, o, s)) return rc;
  }
  return ZEN_OK;
}

constexpr int64_t kMostSide = kMostLd;

}  // namespace
}  // namespace zen

extern "C" {

size_t zen_orthogonal_workspace(int64_t rows, int64_t cols, int64_t count, int precise) {
  using namespace zen;
  if (rows <= 0 || cols <= 0 || count <= 0 || rows > kMostSide || cols > kMostSide) return 0;
  return room_for(rows, cols, count, precise != 0, nullptr).bytes;
}

int zen_orthogonal_path(int64_t rows, int64_t cols, int64_t count, int precise, int product) {
  using namespace zen;
  if (rows <= 0 || cols <= 0 || count <= 0 || rows > kMostSide || cols > kMostSide || product < 0 || product > 2)
    return fail(ZEN_EINVAL, "zen_orthogonal_path: a size is out of range");
  const Room r = room_for(rows, cols, count, precise != 0, nullptr);
  return path_of(product == 0 ? r.gram : product == 1 ? r.square : r.apply);
}

int zen_orthogonal(const zen_orthogonal_args *p) {
  using namespace zen;
  if (!p) return fail(ZEN_EINVAL, "zen_orthogonal: null pointer");
  const auto known = [](int t) { return t == ZEN_F32 || t == ZEN_BF16 || t == ZEN_F16; };
  if (!known(p->update_dtype) || !known(p->out_dtype)) return fail(ZEN_EINVAL, "zen_orthogonal: types are fp32, bf16 or fp16");
  if (p->rows < 0 || p->cols < 0 || p->count < 0) return fail(ZEN_EINVAL, "zen_orthogonal: a size is out of range");
  if (p->rows > kMostSide || p->cols > kMostSide) return fail(ZEN_EINVAL, "zen_orthogonal: a side is at most 2^21");
  if (p->steps < 1) return fail(ZEN_EINVAL, "zen_orthogonal: at least one step");
  if (!(p->eps >= 0)) return fail(ZEN_EINVAL, "zen_orthogonal: eps is not negative");
  if (p->update_rs < 0 || p->update_cs < 0 || p->out_rs < 0 || p->out_cs < 0) return fail(ZEN_EINVAL, "zen_orthogonal: negative stride");
  if (p->rows == 0 || p->cols == 0 || p->count == 0) return ZEN_OK;
  if (!p->updates || !p->outs || !p->workspace) return fail(ZEN_EINVAL, "zen_orthogonal: null pointer");
  for (int64_t i = 0; i < p->count; ++i)
    if (!p->updates[i] || !p->outs[i]) return fail(ZEN_EINVAL, "zen_orthogonal: null pointer");
  const Room r = room_for(p->rows, p->cols, p->count, p->precise != 0, p->workspace);
  if (p->workspace_bytes < r.bytes) return fail(ZEN_EWORKSPACE, "zen_orthogonal: workspace too small");
  if (!holds(*p)) return fail(ZEN_EINVAL, "zen_orthogonal: in so many steps these coefficients can take values beyond fp16's range");
  for (int64_t first = 0; first < p->count; first += r.batch) {
    const int64_t rest = p->count - first;
    const int batch = (int)(rest < r.batch ? rest : r.batch);
    hipStream_t s = static_cast<hipStream_t>(p->stream);
    if (const int rc = p->precise ? chunk<true>(*p, r, first, batch, s) : chunk<false>(*p, r, first, batch, s)) return rc;
  }
  return ZEN_OK;
}

}  // extern "C"
