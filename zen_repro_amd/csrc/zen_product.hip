// out = alpha a b + beta c for matrices in 16 bits (zen_tiles.h has the product itself).
#include "zen_tiles.h"

namespace zen {
namespace {

// How an operand is read: its `rows` (of a, or columns of b) and k.
struct Side {
  const void *p;
  int64_t row, along, batch;  // strides of rows, of k, of matrices
  int64_t rows, k;
  bool contiguous;  // read with k contiguous
  bool packed;
  int64_t ld;       // of the layout that is read
};

Side side(const void *p, int64_t row, int64_t along, int64_t batch, int64_t rows, int64_t k, int64_t batches) {
  Side s = {p, row, along, batch, rows, k, true, false, 0};
  const bool at = (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (batches <= 1 || batch % 8 == 0);
  const bool by_k = (along == 1 || k == 1) && row % 8 == 0 && row >= k && k % 8 == 0;
  const bool by_row = (row == 1 || rows == 1) && along % 8 == 0 && along >= rows;
  if (at && by_k && row <= kMostLd) {
    s.ld = row;
  } else if (at && by_row && along <= kMostLd) {
    s.contiguous = false;
    s.ld = along;
  } else {
    s.packed = true;
    s.ld = (int64_t)align_up((size_t)k, 8);
  }
  return s;
}

size_t room(const Side &s, int64_t batches) {
  return s.packed ? align_up((size_t)s.rows * s.ld * batches * 2, 256) : 0;
}

// How the operand is laid out, if it is; the side is then read from there.
bool lay_out(Side &s, int64_t batches, Carver &cv, PackArgs &p) {
  if (!s.packed) return false;
  p = {};
  p.in.base = static_cast<char *>(const_cast<void *>(s.p));
  p.in.stride = s.batch * 2;
  p.rs = s.row;
  p.cs = s.along;
  p.rows = (int)s.rows;
  p.cols = (int)s.k;
  p.batch = (int)batches;
  p.out = cv.take<uint16_t>((size_t)s.rows * s.ld * batches);
  p.ld = s.ld;
  p.out_batch = s.rows * s.ld;
  s.p = p.out;
  s.batch = p.out_batch;
  return true;
}

constexpr int64_t kMostStack = 65535;

bool known(int type) { return type == ZEN_F32 || type == ZEN_BF16 || type == ZEN_F16; }
int64_t size_of(int type) { return type == ZEN_F32 ? 4 : 2; }

template <bool AK, bool BK>
int go(const TilePlan &plan, float *partial, const MatSize &size, const MatOperand &a, const MatOperand &b, const OutEpilogue &e, bool bf,
       bool sym, hipStream_t s) {
  if (bf)
    return sym ? run_tiles<AK, BK, true, true>(plan, partial, size, a, b, e, s) : run_tiles<AK, BK, true, false>(plan, partial, size, a, b, e, s);
  return sym ? run_tiles<AK, BK, false, true>(plan, partial, size, a, b, e, s) : run_tiles<AK, BK, false, false>(plan, partial, size, a, b, e, s);
}

int lines(const void *p, int64_t rs, int64_t cs, int64_t batch, int type, int64_t batches, bool symmetric) {
  const int64_t size = size_of(type);
  if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0 || (batches > 1 && batch * size % 16 != 0)) return 0;
  return cs == 1 && rs * size % 16 == 0 ? 1 : rs == 1 && cs * size % 16 == 0 && !symmetric ? 2 : 0;
}

int check(const zen_product_args *p) {
  if (!p) return fail(ZEN_EINVAL, "zen_product: null pointer");
  const int64_t most = 0x7fffffffll - 1024;
  if (p->m < 0 || p->n < 0 || p->k < 0 || p->batch < 0 || p->m > most || p->n > most)
    return fail(ZEN_EINVAL, "zen_product: a size is out of range");
  if (p->k > kMostLd) return fail(ZEN_EINVAL, "zen_product: k is at most 2^21");
  if (p->batch > kMostStack) return fail(ZEN_EINVAL, "zen_product: at most 65535 matrices");
  if (p->dtype != ZEN_BF16 && p->dtype != ZEN_F16) return fail(ZEN_EINVAL, "zen_product: a and b are bf16 or fp16");
  if (!known(p->out_dtype) || (p->c && !known(p->c_dtype))) return fail(ZEN_EINVAL, "zen_product: c and out are fp32, bf16 or fp16");
  if (p->symmetric && p->m != p->n) return fail(ZEN_EINVAL, "zen_product: a symmetric result is square");
  if (p->a_rs < 0 || p->a_cs < 0 || p->b_rs < 0 || p->b_cs < 0 || p->c_rs < 0 || p->c_cs < 0 || p->out_rs < 0 || p->out_cs < 0)
    return fail(ZEN_EINVAL, "zen_product: negative stride");
  return ZEN_OK;
}

Side side_a(const zen_product_args &p) { return side(p.a, p.a_rs, p.a_cs, p.a_batch, p.m, p.k, p.batch); }
Side side_b(const zen_product_args &p) { return side(p.b, p.b_cs, p.b_rs, p.b_batch, p.n, p.k, p.batch); }
TilePlan plan(const zen_product_args &p, const Side &a, const Side &b) {
  return plan_tiles(p.m, p.n, p.k, 1, p.batch, p.symmetric != 0, a.contiguous && b.contiguous);
}

}  // namespace
}  // namespace zen

extern "C" {

size_t zen_product_workspace(const zen_product_args *p) {
  using namespace zen;
  if (check(p) != ZEN_OK || p->m == 0 || p->n == 0 || p->batch == 0 || p->k == 0) return 0;
  const Side a = side_a(*p), b = side_b(*p);
  return room(a, p->batch) + room(b, p->batch) + plan(*p, a, b).partial_bytes;
}

int zen_product_path(const zen_product_args *p) {
  using namespace zen;
  if (const int rc = check(p)) return rc;
  const Side a = side_a(*p), b = side_b(*p);
  return path_of(plan(*p, a, b)) | (a.contiguous ? 0 : 1 << 20) | (b.contiguous ? 0 : 1 << 21) | (a.packed ? 1 << 22 : 0) |
         (b.packed ? 1 << 23 : 0);
}

int zen_product(const zen_product_args *p) {
  using namespace zen;
  if (const int rc = check(p)) return rc;
  if (p->m == 0 || p->n == 0 || p->batch == 0) return ZEN_OK;
  if (!p->out || (p->k > 0 && (!p->a || !p->b))) return fail(ZEN_EINVAL, "zen_product: null pointer");
  const size_t need = zen_product_workspace(p);
  if (need && !p->workspace) return fail(ZEN_EINVAL, "zen_product: null pointer");
  if (p->workspace_bytes < need) return fail(ZEN_EWORKSPACE, "zen_product: workspace too small");
  hipStream_t s = static_cast<hipStream_t>(p->stream);
  Side sa = side_a(*p), sb = side_b(*p);
  const TilePlan how = plan(*p, sa, sb);
  Carver cv(p->workspace);
  if (p->k > 0) {
    PackArgs pack[2];
    int packs = lay_out(sa, p->batch, cv, pack[0]) ? 1 : 0;
    packs += lay_out(sb, p->batch, cv, pack[packs]) ? 1 : 0;
    if (packs)
      if (const int rc = pack_matrices(pack, packs, s)) return rc;
  }
  const MatSize size = {(int)p->m, (int)p->n, (int)p->k, 0, 0, (int)p->batch, 1, 1, nullptr};
  float *partial = reinterpret_cast<float *>(cv.base + cv.used);
  const uint16_t *pa = static_cast<const uint16_t *>(sa.p), *pb = static_cast<const uint16_t *>(sb.p);
  const MatOperand a = {{pa, pa}, sa.ld, sa.batch}, b = {{pb, pb}, sb.ld, sb.batch};
  const bool bf = p->dtype == ZEN_BF16, sym = p->symmetric != 0;
  OutEpilogue e = {};
  e.alpha = p->alpha;
  e.gain = 1.f;
  e.keep = p->beta;
  e.rows = (int)p->m;
  e.cols = (int)p->n;
  e.out.base = static_cast<char *>(p->out);
  e.out.stride = p->out_batch * size_of(p->out_dtype);
  e.out_rs = p->out_rs;
  e.out_cs = p->out_cs;
  e.out_type = p->out_dtype;
  e.lines = lines(p->out, p->out_rs, p->out_cs, p->out_batch, p->out_dtype, p->batch, sym);
  e.res.listed = -1;
  if (p->c) {
    if (lines(p->c, p->c_rs, p->c_cs, p->c_batch, p->c_dtype, p->batch, sym) != e.lines) e.lines = 0;
    e.res.listed = 0;
    e.res.base = static_cast<char *>(const_cast<void *>(p->c));
    e.res.stride = p->c_batch * size_of(p->c_dtype);
    e.res_rs = p->c_rs;
    e.res_cs = p->c_cs;
    e.res_type = p->c_dtype;
  }
  if (sa.contiguous)
    return sb.contiguous ? go<true, true>(how, partial, size, a, b, e, bf, sym, s) : go<true, false>(how, partial, size, a, b, e, bf, sym, s);
  return sb.contiguous ? go<false, true>(how, partial, size, a, b, e, bf, sym, s) : go<false, false>(how, partial, size, a, b, e, bf, sym, s);
}

}  // extern "C"
