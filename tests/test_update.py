"""The operators behind the exchange: momentum (dense and from lists), products, orthogonalisation, the optimiser.
Values are compared with the formulas in 64 bits; every tolerance counts roundings (u = half a step of the type,
fp32 2^-24, fp16 2^-11, bf16 2^-8)."""
import ctypes
import math

import pytest
import torch

import zen_repro_amd as zen
from zen_repro_amd import _lib

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
MU = float(torch.tensor(0.95, dtype=F32))  # what the kernels compute with


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def within(got, want, room, what=""):
    """|got - want| <= room, element by element; want and room in 64 bits."""
    off = (got.double() - want).abs()
    worst = (off - room).max().item() if off.numel() else 0.0
    assert worst <= 0.0, f"{what}: {worst:.3g} beyond the tolerance, at {int((off - room).argmax())}"


# --------------------------------------------------------------- host refusals


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def test_momentum_refusals_of_the_library(L):
    one = ctypes.c_void_p(256)  # never dereferenced: validation comes first
    assert L.zen_momentum(one, 0, one, 0, -1, 0.9, 1, one, 0, None) == _lib.EINVAL
    assert L.zen_momentum(one, 2, one, 0, 8, 0.9, 1, one, 0, None) == _lib.EINVAL   # fp16 momentum
    assert L.zen_momentum(one, 0, one, 3, 8, 0.9, 1, one, 0, None) == _lib.EINVAL
    assert L.zen_momentum(one, 0, one, 0, 8, 0.9, 1, None, 0, None) == _lib.EINVAL
    assert L.zen_momentum(None, 0, None, 0, 0, 0.9, 1, None, 0, None) == _lib.OK    # nothing to do
    ptrs, sizes = (ctypes.c_void_p * 65)(*[256] * 65), (ctypes.c_int64 * 65)(*[4] * 65)

    def lists(n=100, count=1, length=4, ws=1 << 20, val=0, mom=0, status=one):
        sizes[0] = length
        return L.zen_momentum_lists(one, mom, ptrs, 0, ptrs, val, sizes, None, count, n, 0.9, 1, one, 0, one, ws, status, None)

    assert lists(count=0) == lists(count=65) == _lib.EINVAL
    assert lists(n=1 << 31) == lists(n=-1) == lists(length=-1) == lists(length=1 << 31) == _lib.EINVAL
    assert lists(val=7) == lists(mom=2) == lists(status=None) == lists(n=0) == _lib.EINVAL
    assert lists(ws=4) == _lib.EWORKSPACE
    assert lists(n=0, length=0) == _lib.OK
    assert L.zen_momentum_lists_workspace(0, 1) == L.zen_momentum_lists_workspace(100, 65) == 0


def product_args(**more):
    p = _lib.ProductArgs(a=256, a_rs=64, a_cs=1, b=256, b_rs=64, b_cs=1, dtype=1, out=256, out_dtype=1, out_rs=64, out_cs=1,
                         m=64, n=64, k=64, batch=1, alpha=1, beta=1)
    for key, value in more.items():
        setattr(p, key, value)
    return ctypes.byref(p)


def test_product_refusals_of_the_library(L):
    for bad in (dict(m=-1), dict(k=1 << 31), dict(k=(1 << 21) + 8, a_rs=1 << 22), dict(dtype=0), dict(out_dtype=3), dict(c=256, c_dtype=9), dict(symmetric=1, n=32),
                dict(a_rs=-64), dict(out=None), dict(b=None), dict(batch=1 << 20)):
        assert L.zen_product(product_args(**bad)) == _lib.EINVAL, bad
    assert L.zen_product(None) == _lib.EINVAL
    assert L.zen_product_workspace(product_args()) == 0                       # read as it lies
    assert L.zen_product_workspace(product_args(a=258)) > 0                   # laid out first
    assert L.zen_product(product_args(a=258, workspace=256, workspace_bytes=16)) == _lib.EWORKSPACE
    assert L.zen_product(product_args(a=258)) == _lib.EINVAL                  # no workspace
    assert L.zen_product(product_args(m=0)) == L.zen_product(product_args(batch=0)) == _lib.OK


def test_orthogonal_refusals_of_the_library(L):
    ptrs = (ctypes.c_void_p * 2)(256, 256)

    def call(**more):
        p = _lib.OrthogonalArgs(updates=ptrs, update_dtype=1, update_rs=64, update_cs=1, outs=ptrs, out_dtype=1, out_rs=64,
                                out_cs=1, rows=64, cols=64, count=1, steps=5, a=3, b=-4, c=2, eps=1e-7, workspace=256,
                                workspace_bytes=1 << 30)
        for key, value in more.items():
            setattr(p, key, value)
        return L.zen_orthogonal(ctypes.byref(p))

    for bad in (dict(steps=0), dict(update_dtype=5), dict(out_dtype=-1), dict(rows=-1), dict(cols=1 << 22), dict(eps=-1.0),
                dict(eps=math.nan), dict(update_rs=-1), dict(workspace=None), dict(updates=(ctypes.c_void_p * 1)(None))):
        assert call(**bad) == _lib.EINVAL, bad
    assert call(workspace_bytes=100) == _lib.EWORKSPACE
    assert call(rows=0) == call(count=0) == _lib.OK
    assert L.zen_orthogonal(None) == _lib.EINVAL
    assert L.zen_orthogonal_workspace(64, 64, 1, 1) > L.zen_orthogonal_workspace(64, 64, 1, 0) > 0
    assert L.zen_orthogonal_workspace(0, 64, 1, 0) == L.zen_orthogonal_workspace(64, 64, 0, 0) == 0


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(8, 8)
    for call in (lambda: zen.momentum_update(x, x), lambda: zen.momentum_update_sparse(x, x.int(), x),
                 lambda: zen.product(x, x), lambda: zen.orthogonalize(x), lambda: zen.orthogonal_step(x, x, 0.1)):
        with pytest.raises(TypeError):
            call()


def test_muon_takes_matrices():
    with pytest.raises(ValueError):
        zen.Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError):
        zen.Muon([torch.nn.Parameter(torch.zeros(4, 4))], lr=-1)
    with pytest.raises(TypeError):
        zen.Muon([torch.nn.Parameter(torch.zeros(4, 4))], precision=torch.float64)


def test_muon_keeps_its_momentum_in_fp32():
    params = [torch.nn.Parameter(torch.zeros(4, 4, dtype=BF16)) for _ in range(2)]
    opt = zen.Muon(params)
    opt.state[params[1]]["momentum"] = torch.full((4, 4), 1.0 + 2.0 ** -20)
    other = zen.Muon([torch.nn.Parameter(torch.zeros(4, 4, dtype=BF16)) for _ in range(2)])
    other.load_state_dict(opt.state_dict())
    got = other.state[other.param_groups[0]["params"][1]]["momentum"]
    assert got.dtype == F32 and torch.equal(got, opt.state[params[1]]["momentum"])


# -------------------------------------------------------------------- momentum


def momentum_in_64_bits(m, g, nesterov):
    """(m', u) and how much of them is subject to rounding."""
    new = MU * m.double() + g
    u = g + MU * new if nesterov else new
    return new, u, g.abs() + MU * new.abs()


def momentum_check(before, momentum, update, g, nesterov, sum_room=0.0):
    new, u, size = momentum_in_64_bits(before, g, nesterov)
    # m' is one rounded fma of g (itself off by sum_room) and its store another; u the same of the unrounded m'
    room = U[F32] * new.abs() + sum_room
    within(momentum, new, room * (1 + 2.0 ** -20) + (U[BF16] * new.abs() if momentum.dtype == BF16 else 0) + 1e-38, "momentum")
    room_u = sum_room + MU * room + U[F32] * size if nesterov else room
    within(update, u, room_u * (1 + 2.0 ** -6) + (U[update.dtype] * u.abs() + 2.0 ** -24 if update.dtype != F32 else 0) + 1e-38,
           "update")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 7, 8, 255, 2047, 2048, 2049, 100003])
@pytest.mark.parametrize("state,grad,out", [(F32, F32, BF16), (F32, BF16, BF16), (BF16, BF16, F32), (F32, F16, F16),
                                            (BF16, F32, F16)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_momentum(n, state, grad, out, nesterov):
    before, g = normal(n, 1, state), normal(n, 2, grad)
    m = before.clone()
    u = zen.momentum_update(m, g, 0.95, nesterov, dtype=out)
    assert u.dtype == out and u.shape == (n,)
    momentum_check(before, m, u, g.double(), nesterov)


@pytest.mark.gpu
def test_momentum_at_odd_addresses_into_the_gradient_and_in_shape():
    base = normal(4099, 3)
    for shift in (1, 2, 3):
        before, g = base[shift:shift + 3000].clone(), normal(3001, 4, BF16)[1:]
        room = torch.full((3010,), 7.0, device="cuda")
        m = room[shift:shift + 3000]
        m.copy_(before)
        u = zen.momentum_update(m, g, 0.95, out=g.new_empty(3000))
        momentum_check(before, m, u, g.double(), True)
        assert (room[:shift] == 7).all() and (room[shift + 3000:] == 7).all()
    m, g = normal((3, 5, 11), 5), normal((3, 5, 11), 6)
    before, was = m.clone(), g.clone()
    u = zen.momentum_update(m, g, 0.95, out=g)
    assert u is g and u.shape == (3, 5, 11)
    momentum_check(before, m, u, was.double(), True)
    empty = torch.empty(0, device="cuda")
    assert zen.momentum_update(empty, empty.clone()).numel() == 0


def some_lists(n, lengths, seed, idx=torch.int32, val=F32, shared=0):
    """Ascending lists; `shared` indices are in all of them."""
    g = torch.Generator().manual_seed(seed)
    common = torch.randperm(n, generator=g)[:shared]
    out = []
    for k in lengths:
        own = torch.cat([common, torch.randperm(n, generator=g)])[:k]
        out.append((torch.unique(own).to(idx).cuda(), None))
    return [(i, normal(i.numel(), seed + 1 + p, val)) for p, (i, _) in enumerate(out)]


def dense_of(lists, n):
    g = torch.zeros(n, dtype=torch.float64, device="cuda")
    size = torch.zeros(n, dtype=torch.float64, device="cuda")
    for i, v in lists:
        g.index_add_(0, i.long(), v.double())
        size.index_add_(0, i.long(), v.double().abs())
    return g, size


@pytest.mark.gpu
@pytest.mark.parametrize("n,lengths,shared", [
    (1, [1], 0), (1, [0], 0), (5, [3, 0, 5], 2), (2048, [2048], 0), (2049, [1, 2, 2049], 1), (70001, [0], 0), (70001, [1], 0),
    (70001, [70001, 70001, 3], 0), (300007, [3000] * 16, 100), (300007, [100, 0, 40000, 1] * 16, 7), (4096, [64, 64, 65], 64),
    (1 << 21, [1, 0, 2, 5000], 0)])
@pytest.mark.parametrize("idx,val,state,out", [(torch.int32, F32, F32, BF16), (torch.int64, BF16, F32, F32),
                                               (torch.int64, F32, BF16, F16)])
def test_momentum_from_lists(n, lengths, shared, idx, val, state, out):
    lists = some_lists(n, lengths, 10, idx, val, shared)
    for nesterov in (True, False):
        before = normal(n, 11, state)
        m = before.clone()
        u, status = zen.momentum_update_sparse(m, [i for i, _ in lists], [v for _, v in lists], 0.95, nesterov, dtype=out)
        assert status.item() == 0
        g, size = dense_of(lists, n)
        momentum_check(before, m, u, g, nesterov, sum_room=len(lengths) * U[F32] * size)
        again = before.clone()  # sums are taken in the order of the lists
        v, _ = zen.momentum_update_sparse(again, [i for i, _ in lists], [v for _, v in lists], 0.95, nesterov, dtype=out)
        assert torch.equal(again, m) and torch.equal(u, v)


@pytest.mark.gpu
def test_momentum_from_lists_order_of_sums_and_odd_addresses():
    n = 5000
    idx = torch.arange(0, n, 7, dtype=torch.int32, device="cuda")
    lists = [normal(idx.numel(), 20 + p, F32, 10.0 ** p) for p in range(5)]
    room = torch.zeros(n + 3, device="cuda")
    for shift in (0, 1):
        m = room[shift:shift + n].zero_()
        zen.momentum_update_sparse(m, [idx] * 5, lists, 0.5, False)
        want = torch.zeros(idx.numel(), device="cuda")
        for v in lists:
            want = want + v
        assert torch.equal(m[idx.long()], want)
        assert room[n + shift:].eq(0).all()


@pytest.mark.gpu
def test_momentum_counts_on_the_device():
    n = 100000
    lists = some_lists(n, [5000, 3000, 10], 30)
    kept = [4000, 0, 10]
    want = dense_of([(i[:c], v[:c]) for (i, v), c in zip(lists, kept)], n)
    for (i, v), c in zip(lists, kept):
        i[c:] = -5
        v[c:] = math.nan
    counts = torch.tensor(kept, device="cuda")
    for given in (counts, [counts[0:1], counts[1:2], None]):
        before = normal(n, 31)
        m = before.clone()
        u, status = zen.momentum_update_sparse(m, [i for i, _ in lists], [v for _, v in lists], counts=given)
        assert status.item() == 0
        momentum_check(before, m, u, want[0], True, 3 * U[F32] * want[1])
    # a count beyond the list's length, and one below zero, are held to it
    i, v = lists[2]
    for c, used in ((99, 10), (-3, 0)):
        m = torch.zeros(n, device="cuda")
        _, status = zen.momentum_update_sparse(m, i, v, counts=torch.tensor([c], device="cuda"))
        assert status.item() == 0 and int((m != 0).sum()) == used


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [[-1, 5], [5, 5], [9, 3], [3, 4000], [0, 1 << 30], [-(1 << 31), 7]])
def test_momentum_lists_that_are_none(bad):
    n = 4000
    before = normal(n, 40)
    m = before.clone()
    good = torch.arange(10, dtype=torch.int32, device="cuda")
    wrong = torch.tensor(bad, dtype=torch.int32, device="cuda")
    _, status = zen.momentum_update_sparse(m, [good, wrong], [normal(10, 41), normal(2, 42)])
    assert status.item() & _lib.STAT_BAD_INDEX and torch.equal(m, before)


@pytest.mark.gpu
def test_momentum_refusals():
    m, g = torch.zeros(64, device="cuda"), torch.ones(64, device="cuda")
    i = torch.arange(64, dtype=torch.int32, device="cuda")
    for call, error in [
            (lambda: zen.momentum_update(m, g[:32]), ValueError), (lambda: zen.momentum_update(m.half(), g), TypeError),
            (lambda: zen.momentum_update(m, g.double()), TypeError), (lambda: zen.momentum_update(m, m), ValueError),
            (lambda: zen.momentum_update(m, g, out=m), ValueError), (lambda: zen.momentum_update(m, g, -1.0), ValueError),
            (lambda: zen.momentum_update(m, g, math.nan), ValueError),
            (lambda: zen.momentum_update(m, g, out=g.half(), dtype=F32), TypeError),
            (lambda: zen.momentum_update(m[::2], g[::2]), RuntimeError),
            (lambda: zen.momentum_update(m[:60], g[:60], out=g[4:]), ValueError),
            (lambda: zen.momentum_update(m, g.requires_grad_()), RuntimeError),
            (lambda: zen.momentum_update_sparse(m, [i], []), ValueError),
            (lambda: zen.momentum_update_sparse(m, [i] * 65, [g.detach()] * 65), ValueError),
            (lambda: zen.momentum_update_sparse(m, i.short(), g.detach()), TypeError),
            (lambda: zen.momentum_update_sparse(m, i, g.detach()[:5]), ValueError),
            (lambda: zen.momentum_update_sparse(m, i, g.detach(), counts=torch.zeros(2, dtype=torch.int64, device="cuda")), ValueError),
            (lambda: zen.momentum_update_sparse(m, i, g.detach(), counts=torch.zeros(1, device="cuda")), TypeError),
            (lambda: zen.momentum_update_sparse(m, i, m), ValueError),
            (lambda: zen.momentum_update_sparse(m[:0], i, g.detach()), ValueError)]:
        with pytest.raises(error):
            call()
    assert m.eq(0).all()


# --------------------------------------------------------------------- product


def product_check(out, a, b, residual, alpha, beta):
    k = a.shape[-1]
    want = alpha * (a.double() @ b.double())
    size = abs(alpha) * (a.double().abs() @ b.double().abs())
    # k products summed in fp32 in any order, and the scaling by alpha (itself rounded to fp32)
    room = 1.01 * (k + 4) * U[F32] * size
    if residual is not None:
        want = want + beta * residual.double()
        room = room + 4 * U[F32] * (abs(beta) * residual.double().abs() + size)
    if out.dtype != F32:
        room = room * (1 + U[out.dtype]) + U[out.dtype] * want.abs() + (2.0 ** -25 if out.dtype == F16 else 0)
    within(out, want, room + 1e-37, "product")


SIZES = [(1, 1, 1), (1, 5, 3), (16, 16, 64), (64, 64, 64), (65, 63, 72), (128, 128, 128), (130, 250, 40), (257, 511, 1023),
         (300, 129, 8), (640, 384, 512), (33, 700, 2056)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("a_turned", [False, True])
@pytest.mark.parametrize("b_turned", [False, True])
def test_product(m, n, k, dtype, a_turned, b_turned):
    a = normal((k, m), 50, dtype).t() if a_turned else normal((m, k), 50, dtype)
    b = normal((n, k), 51, dtype).t() if b_turned else normal((k, n), 51, dtype)
    product_check(zen.product(a, b), a, b, None, 1.0, 0.0)
    c = normal((m, n), 52, F32)
    out = zen.product(a, b, residual=c, alpha=0.25, beta=-1.5)
    assert out.dtype == F32
    product_check(out, a, b, c, 0.25, -1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [
    (4200, 4100, 328), (2100, 4200, 72), (2000, 1500, 136), (1900, 1930, 2056),   # large tiles to small ones, one to some rounds
    (512, 520, 4104), (70, 60, 8200), (1024, 300, 2056), (129, 129, 1000)])       # the steps of few tiles are shared
@pytest.mark.parametrize("a_turned,b_turned", [(False, True), (False, False), (True, False)])
def test_product_of_every_tile(m, n, k, a_turned, b_turned):
    a = normal((k, m), 53, BF16).t() if a_turned else normal((m, k), 53, BF16)
    b = normal((n, k), 54, BF16).t() if b_turned else normal((k, n), 54, BF16)
    c = normal((m, n), 55, F16)
    product_check(zen.product(a, b, residual=c, alpha=0.5, beta=3.0), a, b, c, 0.5, 3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(4100, 200), (3000, 136), (1000, 4104), (260, 2056)])
def test_product_symmetric_of_every_tile(m, k):
    a = normal((m, k), 56, F16)
    out = zen.product(a, a.t(), symmetric=True, dtype=F32)
    product_check(out, a, a.t(), None, 1.0, 0.0)
    assert torch.equal(out, out.t())
    out = zen.product(a, a.t(), symmetric=True)
    assert out.dtype == F16 and torch.equal(out, out.t())
    product_check(out, a, a.t(), None, 1.0, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("out", [BF16, F16, F32])
@pytest.mark.parametrize("res", [BF16, F16, F32])
def test_product_strides_types_and_the_residual_in_place(out, res):
    m, n, k = 200, 136, 96
    a = normal((m, 3 * k + 5), 60, BF16)[:, 5:5 + k]         # odd addresses: laid out first
    b = normal((2 * k, 2 * n), 61, BF16)[::2, ::2]            # no neighbours either way
    c = normal((n, m), 62, res).t()
    room = torch.full((m + 2, 2 * n), 3.0, device="cuda", dtype=out)
    o = room[1:-1, 1::2]
    assert zen.product(a, b, residual=c, alpha=0.1, beta=0.5, out=o) is o
    product_check(o, a, b, c, 0.1, 0.5)
    assert (room[0] == 3).all() and (room[-1] == 3).all() and (room[:, ::2] == 3).all()
    if out == res:
        own = c.clone()
        before = own.clone()
        zen.product(a, b, residual=own, out=own)
        product_check(own, a, b, before, 1.0, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_product_turned_results_and_residuals_that_are_one_row(dtype):
    m, n, k = 200, 328, 136
    a, b = normal((m, k), 63, BF16), normal((k, n), 64, BF16)
    c = normal((n, m), 65, dtype).t()
    for residual in (None, c, normal((1, n), 66, dtype).expand(m, n), normal((m, 1), 67, dtype).expand(m, n)):
        for out in (torch.empty(n, m, device="cuda", dtype=dtype).t(), torch.empty(m, n, device="cuda", dtype=dtype)):
            zen.product(a, b, residual=residual, beta=2.0, out=out)
            product_check(out, a, b, residual, 1.0, 2.0)
    own = c.clone()
    assert own.stride() == c.stride()
    zen.product(a, b, residual=own, out=own)
    product_check(own, a, b, c, 1.0, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [64, 200, 203])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_product_symmetric_into_its_residual(m, dtype):
    a, c = normal((m, 72), 68, F16), normal((m, m), 69, dtype)
    own = c.clone()
    zen.product(a, a.t(), residual=own, alpha=0.5, beta=-1.0, symmetric=True, out=own)
    product_check(own, a, a.t(), c, 0.5, -1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("stack,m,n,k", [(1, 64, 64, 64), (3, 100, 72, 200), (5, 129, 257, 64), (7, 8, 8, 8)])
def test_product_of_stacks(stack, m, n, k, turned):
    a, b = normal((stack, m, k), 70, F16), normal((stack, n, k), 71, F16).transpose(1, 2)
    if turned:
        b = b.contiguous()
    c = normal((stack, m, n), 72, F16)
    product_check(zen.product(a, b, residual=c, beta=2.0), a, b.contiguous(), c, 1.0, 2.0)
    one = a[:1].expand(stack, m, k)  # one matrix for all
    product_check(zen.product(one, b), one.contiguous(), b.contiguous(), None, 1.0, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(1, 8), (64, 64), (129, 40), (300, 1000), (513, 264)])
@pytest.mark.parametrize("turned", [False, True])
def test_product_symmetric(m, k, turned):
    a = normal((k, m), 80, BF16).t() if turned else normal((m, k), 80, BF16)
    c = normal((m, m), 81, F32)
    out = zen.product(a, a.t(), symmetric=True, dtype=F32)
    product_check(out, a, a.t(), None, 1.0, 0.0)
    assert torch.equal(out, out.t())
    product_check(zen.product(a, a.t(), residual=c, symmetric=True, alpha=0.5), a, a.t(), c, 0.5, 1.0)
    s = normal((2, m, m), 82, F16)
    s = s + s.transpose(1, 2)
    product_check(zen.product(s, s, symmetric=True), s, s, None, 1.0, 0.0)


@pytest.mark.gpu
def test_product_of_nothing_and_of_values_that_are_none():
    a, b = normal((0, 8), 90, BF16), normal((8, 5), 91, BF16)
    assert zen.product(a, b).shape == (0, 5)
    c = normal((4, 5), 92, F32)
    assert torch.equal(zen.product(a.new_empty(4, 0), a.new_empty(0, 5), residual=c, beta=2.0), 2 * c)
    a, b = normal((130, 72), 93, BF16), normal((72, 140), 94, BF16)
    a[3, 5] = math.inf
    b[7, 9] = math.nan
    out = zen.product(a, b, dtype=F32)
    want = a.float().cpu() @ b.float().cpu()
    assert torch.equal(out.isfinite().cpu(), want.isfinite()) and torch.equal(out.isnan().cpu(), want.isnan())
    # rows that a tile reads beyond its matrix are another's: they must not come in
    big = torch.full((300, 72), math.nan, device="cuda", dtype=BF16)
    big[:130] = normal((130, 72), 95, BF16)
    wide = torch.full((72, 304), math.nan, device="cuda", dtype=BF16)
    wide[:, :137] = normal((72, 137), 96, BF16)
    product_check(zen.product(big[:130], wide[:, :137]), big[:130], wide[:, :137], None, 1.0, 0.0)
    deep = torch.full((130, 200), math.nan, device="cuda", dtype=BF16)
    deep[:, :72] = big[:130]
    tall = torch.full((100, 137), math.nan, device="cuda", dtype=BF16)
    tall[:72] = wide[:, :137]
    for k in (72, 70):
        product_check(zen.product(deep[:, :k], tall[:k]), deep[:, :k], tall[:k], None, 1.0, 0.0)


@pytest.mark.gpu
def test_product_refusals():
    a, b = normal((64, 32), 97, BF16), normal((32, 64), 98, BF16)
    for call, error in [
            (lambda: zen.product(a, a), ValueError), (lambda: zen.product(a, b.half()), TypeError),
            (lambda: zen.product(a.float(), b.float()), TypeError), (lambda: zen.product(a, b[None]), ValueError),
            (lambda: zen.product(a[0], b), ValueError), (lambda: zen.product(a, b[:, :5], symmetric=True), ValueError),
            (lambda: zen.product(a, b, residual=a), ValueError), (lambda: zen.product(a, b, dtype=torch.float64), TypeError),
            (lambda: zen.product(a, b, out=a.new_empty(64, 64), dtype=F32), TypeError),
            (lambda: zen.product(a, b, out=a.new_empty(64, 1).expand(64, 64)), ValueError),
            (lambda: zen.product(a[:32], b[:, :32], out=a[32:]), None),
            (lambda: zen.product(a[:32], b[:, :32], out=a[16:48]), ValueError),
            (lambda: zen.product(a, b.cpu()), ValueError),
            (lambda: zen.product(a, b.clone().requires_grad_()), RuntimeError)]:
        if error is None:
            call()
        else:
            with pytest.raises(error):
                call()


# ----------------------------------------------------------- orthogonalisation

A, B, C = 3.4445, -4.7750, 2.0315


def newton_schulz(u, steps=5, eps=1e-7, half=False, abc=(A, B, C)):
    """In 64 bits; `half`: with the roundings of the fp16 path where the kernels have them."""
    a, b, c = abc
    x = u.double().cpu()
    turn = x.shape[0] > x.shape[1]
    x = x.T if turn else x
    x = x / (x.norm() + eps)
    r = (lambda t: t.half().double()) if half else (lambda t: t)
    eye = torch.eye(x.shape[0], dtype=torch.float64)
    for s in range(steps):
        near = half and s >= steps - 2
        h = r(x)
        g = r(h @ h.T)
        p = r(b * g + c * (g @ g) + ((a - 1) * eye if near else 0))
        x = (1 if near else a) * x + p @ h
    return x.T if turn else x


def newton_schulz_fp32(u, steps=5, eps=1e-7):
    x = u.float().cpu()
    x = x / (x.norm() + eps)
    for _ in range(steps):
        g = x @ x.T
        x = A * x + (B * g + C * (g @ g)) @ x
    return x


def off(got, want):
    """2-norm of the difference over that of the result."""
    return ((got.double().cpu() - want).norm() / want.norm()).item()


def update_like(m, n, seed, kind="gauss"):
    u = normal((m, n), seed)
    if kind == "strong":  # few strong directions, the rest 50 times weaker
        r = 4
        u = u * 0.02 + (normal((m, r), seed + 1) * torch.logspace(0, -2, r, device="cuda")) @ normal((r, n), seed + 2)
    return u * 1e-3


def room_of(u, dtype, **more):
    """Tolerance of a result of `dtype`, 2-norm, relative: rounding the result, and twice what the operands' roundings do (their
    effect depends on where they fall; a second run of the same ones with other inputs differs by some ten per cent).
    fp32 and fp16: four times what fp32 products do (an operand of 22 bits instead of 24 is off four times as far)."""
    exact = newton_schulz(u, **more)
    if dtype != BF16 and not more:
        fp32 = newton_schulz_fp32(u if u.shape[0] <= u.shape[1] else u.T)
        return exact, U[dtype] + 4 * max(off(fp32 if u.shape[0] <= u.shape[1] else fp32.T, exact), 4 * U[F32])
    return exact, U[dtype] + 2 * off(newton_schulz(u, half=True, **more), exact)


SHAPES = [(1, 1), (1, 40), (320, 128), (1024, 256), (40, 1), (1100, 1030), (700, 2100), (3, 2), (64, 64), (65, 63), (128, 128), (48, 500), (500, 48), (200, 333), (300, 257), (130, 1030)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("kind", ["gauss", "strong"])
def test_orthogonalize(m, n, dtype, kind):
    u = update_like(m, n, 100, kind).to(dtype)
    want, room = room_of(u, dtype)
    got = zen.orthogonalize(u)
    assert got.shape == u.shape and got.dtype == dtype
    assert off(got, want) <= room, (off(got, want), room)


@pytest.mark.gpu
def test_orthogonalize_gives_singular_values_about_one():
    s = torch.linalg.svdvals(zen.orthogonalize(update_like(128, 300, 105)).cpu().double())
    assert 0.6 < s.min() and s.max() < 1.25


@pytest.mark.gpu
@pytest.mark.parametrize("stack,m,n", [(2, 64, 96), (7, 100, 40), (35, 33, 65), (3, 256, 128)])
def test_orthogonalize_stacks_and_lists(stack, m, n):
    u = torch.stack([update_like(m, n, 110 + 3 * i, "strong" if i % 2 else "gauss") for i in range(stack)]).to(BF16)
    u[stack // 2] = 0  # an update of nothing among others
    got = zen.orthogonalize(u)
    alone = [zen.orthogonalize(x) for x in u]
    listed = zen.orthogonalize([x.t().contiguous().t() for x in u])
    mixed = zen.orthogonalize([x if i % 2 else x.t().contiguous().t() for i, x in enumerate(u)])
    assert got[stack // 2].eq(0).all()
    for i in range(stack):
        assert torch.equal(got[i], alone[i]) and torch.equal(got[i], listed[i]) and torch.equal(got[i], mixed[i])
        if i != stack // 2:
            want, room = room_of(u[i], BF16)
            assert off(got[i], want) <= room


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_orthogonalize_strides_steps_coefficients_and_place(dtype):
    big = normal((400, 700), 120, dtype, 1e-3)
    for u in (big[3:203, 5:140], big.t()[1:301, ::3], big[::2, 7:90]):
        for steps, abc in ((1, (A, B, C)), (2, (A, B, C)), (3, (1.875, -1.25, 0.375)), (7, (1.875, -1.25, 0.375))):
            want, room = room_of(u, BF16 if dtype == BF16 else F16, steps=steps, abc=abc)
            got = zen.orthogonalize(u, steps=steps, coefficients=abc)
            assert off(got, want) <= room
    want, room = room_of(big, BF16)
    out = torch.full((702, 400), 5.0, device="cuda", dtype=BF16)
    got = zen.orthogonalize(big, out=out[1:-1].t())
    assert off(got, want) <= room and (out[0] == 5).all() and (out[-1] == 5).all()
    own = big.clone()
    plain = zen.orthogonalize(big)
    assert zen.orthogonalize(own, out=own) is own and torch.equal(own, plain)


@pytest.mark.gpu
def test_orthogonalize_sizes_of_values():
    """Only the direction counts, however large or small the values are."""
    u = update_like(96, 80, 130)
    want = zen.orthogonalize(u, eps=0.0)  # eps is 1e-6 of this norm: not to be compared with
    for scale in (2.0 ** -90, 2.0 ** 70, 2.0 ** 120):
        got = zen.orthogonalize(u * scale, eps=0.0)
        assert off(got, want.double().cpu()) <= 1e-6
    assert zen.orthogonalize(u * 0, eps=0.0).eq(0).all()
    assert zen.orthogonalize(u[:0]).shape == (0, 80)
    u[5, 7] = math.nan
    assert zen.orthogonalize(u).isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(64, 64), (100, 260), (260, 100), (129, 127)])
@pytest.mark.parametrize("weight,update", [(BF16, BF16), (F32, F32), (F32, BF16), (F16, F32)])
def test_orthogonal_step(m, n, weight, update):
    u, w = update_like(m, n, 140).to(update), normal((m, n), 141, weight, 0.02)
    lr, decay, scale = 0.02, 0.1, 0.2 * math.sqrt(max(m, n))
    before = w.double().cpu()
    for precision in (None, BF16):
        v = w.clone()
        assert zen.orthogonal_step(v, u, lr, decay, scale, precision=precision) is v
        kind = precision or weight
        o, room = room_of(u, kind)
        want = (1 - lr * decay) * before - lr * scale * o
        # the orthogonal part's share, and the rounding of the weight
        limit = lr * scale * room * o.norm() + U[weight] * want.norm() + 4 * U[F32] * before.norm()
        assert (v.double().cpu() - want).norm() <= limit


@pytest.mark.gpu
def test_orthogonal_refusals():
    u = update_like(64, 48, 150)
    w = u.clone()
    pair = torch.zeros(64, 96, device="cuda")
    for call, error in [
            (lambda: zen.orthogonalize(u[0]), ValueError), (lambda: zen.orthogonalize(u, steps=0), ValueError),
            (lambda: zen.orthogonalize(u, coefficients=(1, 2)), ValueError), (lambda: zen.orthogonalize(u, eps=-1), ValueError),
            (lambda: zen.orthogonalize(u.double()), TypeError), (lambda: zen.orthogonalize([u, u[:5]]), ValueError),
            (lambda: zen.orthogonalize([u, u.half()]), ValueError), (lambda: zen.orthogonalize(u, out=w.t()), ValueError),
            (lambda: zen.orthogonalize(u, dtype=BF16, out=w), TypeError),
            (lambda: zen.orthogonalize(u[:32], out=u[16:48]), ValueError),
            (lambda: zen.orthogonal_step([w, w], [u, u], 0.1), ValueError),
            (lambda: zen.orthogonal_step([w], [u, u], 0.1), ValueError), (lambda: zen.orthogonal_step(u, u, 0.1), ValueError),
            (lambda: zen.orthogonal_step(w, u, 0.1, precision=torch.float64), TypeError),
            (lambda: zen.orthogonal_step(w[:1].expand(64, 48), u, 0.1), ValueError),
            (lambda: zen.orthogonal_step(w.clone().requires_grad_(), u, 0.1), RuntimeError),
            (lambda: zen.orthogonal_step([pair[:, :48], pair[:, 40:88]], [u, u], 0.1), ValueError),
            (lambda: zen.orthogonal_step([pair[:, :48], pair[:, 48:]], [u, u], 0.1), None)]:
        if error is None:
            call()
        else:
            with pytest.raises(error):
                call()
    assert torch.equal(pair[:, :48], pair[:, 48:]) and pair.ne(0).any()
    assert zen.orthogonalize([]) == []


# --------------------------------------------------------------------- together


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls in flight on two streams at a time, from one thread, keep apart."""
    us = [update_like(700, 900, 155 + i).to(BF16) for i in range(2)]
    a, b = normal((400, 1001), 157, F16)[:, 1:], normal((1000, 300), 158, F16)
    want = [zen.orthogonalize(u) for u in us], zen.product(a, b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s, u in zip(streams, us):
            with torch.cuda.stream(s):
                got.append((zen.orthogonalize(u), zen.product(a, b)))
    torch.cuda.synchronize()
    for i, (o, p) in enumerate(got):
        assert torch.equal(o, want[0][i % 2]) and torch.equal(p, want[1])


@pytest.mark.gpu
def test_streams_and_graphs():
    """On a stream of its own, and captured: each graph has its own workspace, replays agree with the eager call."""
    u, w = update_like(150, 200, 160).to(BF16), normal((150, 200), 161, BF16, 0.02)
    a, b = normal((150, 1001), 162, BF16)[:, 1:], normal((1000, 72), 163, BF16)
    n = 30000
    lists = some_lists(n, [500, 700], 164)
    idx, val = [i for i, _ in lists], [v for _, v in lists]
    m = normal(n, 165)

    def work(w, m):
        o = zen.orthogonalize(u)
        zen.orthogonal_step(w, u, 0.02)
        d, status = zen.momentum_update_sparse(m, idx, val)
        return o, zen.product(a, b), d, zen.momentum_update(m, d.float())

    w0, m0 = w.clone(), m.clone()
    first = [t.clone() for t in work(w0, m0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w1, m1 = w.clone(), m.clone()
        other = work(w1, m1)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip((*first, w0, m0), (*other, w1, m1)):
        assert torch.equal(x, y)
    graphs = []
    for _ in range(2):
        wg, mg = w.clone(), m.clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _lib.zeros.fresh(u.device)
            got = work(wg, mg)
        graphs.append((g, wg, mg, got))
    for turn in range(3):
        for g, wg, mg, got in graphs:
            wg.copy_(w)
            mg.copy_(m)
            torch.cuda.synchronize()
            g.replay()
        zen.orthogonalize(update_like(300, 500, 170 + turn))  # eager work in between, on the thread's workspace
        torch.cuda.synchronize()
        for g, wg, mg, got in graphs:
            for x, y in zip((*first, w0, m0), (*got, wg, mg)):
                assert torch.equal(x, y)


@pytest.mark.gpu
def test_merge_to_momentum_to_weights():
    """The merge's own output, its count still on the device, goes into the momentum and on into the weights."""
    rows, cols, ranks = 96, 160, 4
    n = rows * cols
    lba = zen.LoadBalanceAllreduce(zen.LocalGroup(ranks), None, None)
    lists = [(i[i != 0], v[i != 0]) for i, v in some_lists(n, [800] * ranks, 180, shared=50)]
    idx, val, count, status = lba.merge_sparse_flat([i for i, _ in lists], [v for _, v in lists], n)
    m = torch.zeros(rows, cols, device="cuda")
    before = normal((rows, cols), 181, F32, 0.02)
    w = before.clone()
    u, bad = zen.momentum_update_sparse(m, idx, val, counts=count)
    zen.orthogonal_step(w, u, 0.1)
    assert status.item() == 0 and bad.item() == 0
    g, size = dense_of(lists, n)
    momentum_check(torch.zeros(n, device="cuda"), m.view(-1), u.view(-1), g, True, ranks * U[F32] * size)
    o, room = room_of(u, F32)
    want = before.double().cpu() - 0.1 * o
    assert (w.double().cpu() - want).norm() <= 0.1 * room * o.norm() + 4 * U[F32] * want.norm()


@pytest.mark.gpu
def test_muon_behind_the_hook():
    """Gradients leave the hook's bucket, the optimiser's step is the formula's."""
    torch.manual_seed(0)
    shapes = [(64, 96), (96, 64), (64, 96)]
    params = [torch.nn.Parameter(normal(s, 190 + i, F32, 0.02)) for i, s in enumerate(shapes)]
    opt = zen.Muon(params, lr=0.02, weight_decay=0.1, match_rms=0.2)
    hook = zen.SparseCommHook(zen.LoadBalanceAllreduce(zen.LocalGroup(1), None, None), 10, 2, zen.LocalGroup(1))

    class Bucket:
        def __init__(self, t):
            self.t = t

        def buffer(self):
            return self.t

    state = [torch.zeros(s, dtype=torch.float64) for s in shapes]
    for step in range(3):
        flat = normal(sum(a * b for a, b in shapes), 200 + step, F32, 1e-3)
        got = hook(None, Bucket(flat)).value()
        at, before = 0, [p.detach().double().cpu() for p in params]
        for p, s in zip(params, shapes):
            p.grad = got[at:at + p.numel()].view(s)
            at += p.numel()
        versions = [p._version for p in params]
        opt.step()
        for i, (p, s) in enumerate(zip(params, shapes)):
            assert p._version > versions[i]
            g = p.grad.double().cpu()
            state[i] = MU * state[i] + g
            within(opt.state[p]["momentum"].cpu(), state[i], 4 * (step + 1) * U[F32] * (state[i].abs() + g.abs()) + 1e-38)
            u = (g + MU * opt.state[p]["momentum"].double().cpu()).float().to(BF16)
            o, room = room_of(u, BF16)
            scale = 0.2 * math.sqrt(max(s))
            want = (1 - 0.002) * before[i] - 0.02 * scale * o
            # the update's own rounding to bf16 may go the other way where its fp32 value is not the formula's: rarely, one
            # step; it is amplified by at most a^5 along the weakest directions, 2^-8 2^-8 485 of the whole
            limit = 0.02 * scale * (room + 485 * 2.0 ** -16) * o.norm() + 4 * U[F32] * before[i].norm()
            assert (p.detach().double().cpu() - want).norm() <= limit


# ------------------------------------------------- precision of bf16 results


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,kind", [
    (1, 1, "gauss"), (3, 2, "gauss"), (2, 50, "strong"), (8, 500, "gauss"), (16, 400, "gauss"), (48, 48, "gauss"), (48, 3000, "gauss"),
    (3000, 48, "gauss"), (63, 64, "gauss"), (64, 64, "gauss"), (64, 1000, "gauss"), (100, 2000, "gauss"), (3000, 100, "strong"),
    (128, 1023, "gauss"), (192, 6000, "gauss"), (255, 500, "strong"), (384, 6000, "gauss"), (500, 640, "gauss")])
def test_orthogonal_part_for_bf16_is_off_by_less_than_bf16_rounds(m, n, kind):
    """What fewer bits in the products do to a bf16 result is to stay below what the result's own rounding does, whatever the
    shape.  Seen before that rounding: as what an fp32 weight of zeros gets."""
    u = update_like(m, n, 300, kind)
    want = newton_schulz(u, eps=0.0)
    part = torch.zeros(m, n, device="cuda")
    zen.orthogonal_step(part, u, 1.0, scale=-1.0, eps=0.0, precision=BF16)
    # (of fewer than a hundred values the rounding may be any: a quarter of bf16's step is what it is by the mean)
    room = off(want.to(BF16), want) if m * n >= 100 else U[BF16] / 4
    assert off(part, want) <= room


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1.0, 2.0 ** -10, 2.0 ** -20, 2.0 ** -30])  # of gradients with an RMS of 1e-3
@pytest.mark.parametrize("precision", [F32, BF16, F16])
def test_muon_steps_alike_whatever_the_gradients_size(precision, size):
    g, before = update_like(96, 80, 310), normal((96, 80), 311, F32, 0.02)
    p = torch.nn.Parameter(before.clone())
    opt = zen.Muon([p], lr=0.02, eps=0.0, precision=precision)
    p.grad = g * size
    opt.step()
    u = (g.double() + MU * g.double()).float()
    if precision == BF16:
        want = newton_schulz(u.to(BF16), eps=0.0)
        # the products' roundings stay below bf16's own; an update rounded the other way, as in test_muon_behind_the_hook
        room = off(want.to(BF16), want) + 485 * 2.0 ** -16
    else:
        want = newton_schulz(u, eps=0.0)
        plain = newton_schulz_fp32(u.T, eps=0.0).T
        room = 4 * max(off(plain, want), 4 * U[F32])  # as in room_of
    part = 0.02 * math.sqrt(96 / 80)
    limit = part * room * want.norm() + 4 * U[F32] * before.double().norm().item()
    assert (p.detach().double().cpu() - (before.double().cpu() - part * want)).norm() <= limit


@pytest.mark.gpu
def test_lists_of_a_call_that_failed_are_not_taken():
    """The status of the call that made the lists goes along, unseen: whatever it says, nothing is written."""
    n = 6000
    (idx, val), = some_lists(n, [900], 400)
    want = dense_of([(idx, val)], n)
    for bits in (_lib.STAT_RETRY, _lib.STAT_CAPACITY, _lib.STAT_INTERNAL, _lib.STAT_BAD_INDEX, _lib.STAT_SERIAL_OVERFLOW, 0):
        before = normal(n, 401)
        m, out = before.clone(), torch.full((n,), 5.0, device="cuda")
        status = torch.tensor([bits], dtype=torch.int32, device="cuda")
        u, got = zen.momentum_update_sparse(m, idx, val, out=out, status=status)
        assert got is status and u is out and got.item() == bits
        if bits:
            assert torch.equal(m, before) and out.eq(5.0).all()
        else:
            momentum_check(before, m, u, want[0], True, U[F32] * want[1])
    # what this call finds goes into the word
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _, got = zen.momentum_update_sparse(m, torch.tensor([5, 5], dtype=torch.int32, device="cuda"), val[:2], status=status)
    assert got is status and status.item() == _lib.STAT_BAD_INDEX
    for wrong, error in ((status.long(), TypeError), (torch.zeros(2, dtype=torch.int32, device="cuda"), ValueError),
                         (status.cpu(), ValueError), (idx[:1], ValueError)):
        with pytest.raises(error):
            zen.momentum_update_sparse(m, idx, val, status=wrong)


@pytest.mark.gpu
def test_a_merge_that_is_declined_does_not_reach_the_momentum():
    """Entries piled on one key make the merge's fast mode decline, its lists unspecified: its status keeps them out of the momentum
    without a wait in between."""
    n = 1 << 20
    idx = torch.cat([torch.full((100000,), 12345), torch.randint(n, (50000,), generator=torch.Generator().manual_seed(1))]).int().cuda()
    val = normal(idx.numel(), 410)
    lba = zen.LoadBalanceAllreduce(zen.LocalGroup(4), None, None)
    before = normal(n, 411)
    for mode, declined in ((_lib.MODE_FAST, True), (_lib.MODE_GENERAL, False)):
        m = before.clone()
        mi, mv, count, status = lba.merge_sparse_flat(idx, val, n, mode=mode)
        u, status = zen.momentum_update_sparse(m, mi, mv, mu=0.5, nesterov=False, counts=count, status=status)
        if declined:
            assert status.item() & _lib.STAT_RETRY and torch.equal(m, before)
            lba.reset_merge_workspace(m.device)
        else:
            assert status.item() == 0
            wi, wv = lba.merge_sparse(idx, val, n)
            want = before * 0.5
            want[wi] += wv
            assert torch.equal(m, want) and torch.equal(u, want)  # halves are exact, one rounding each


@pytest.mark.gpu
def test_ranks_stay_alike_from_the_exchange_to_the_weights():
    """Four ranks: buckets to their partitions, each partition merged where it belongs, all lists to every rank, momentum and
    weights from them: every rank ends with the update of the whole gradient."""
    rows, cols, ranks = 96, 160, 4
    n = rows * cols
    grads = [torch.zeros(n, device="cuda").index_put_((i.long(),), v) for i, v in some_lists(n, [900] * ranks, 420, shared=60)]
    lba = [zen.LoadBalanceAllreduce(zen.LocalGroup(ranks, r), None, None) for r in range(ranks)]
    sent = [lba[r].tensor_partition.load_balance(g) for r, g in enumerate(grads)]
    merged = [lba[r].merge_rounded([s[0][r].clone() for s in sent], [s[1][r].clone() for s in sent], n, F32) for r in range(ranks)]
    total = torch.stack(grads).double().sum(0)
    size = torch.stack(grads).double().abs().sum(0)
    total[0] = size[0] = 0.0  # the partition's tables have no place for index 0, as the reference's: it is not sent
    before = normal((rows, cols), 421, F32, 0.02)
    results = []
    for r in range(ranks):
        m, w = torch.zeros(rows, cols, device="cuda"), before.clone()
        u, status = zen.momentum_update_sparse(m, [i for i, _ in merged], [v for _, v in merged])
        assert status.item() == 0
        zen.orthogonal_step(w, u, 0.1)
        momentum_check(torch.zeros(n, device="cuda"), m.view(-1), u.view(-1), total, True, ranks * U[F32] * size)
        results.append((m, u, w))
    for r in range(1, ranks):
        assert all(torch.equal(a, b) for a, b in zip(results[0], results[r]))
    o, room = room_of(results[0][1], F32)
    want = before.double().cpu() - 0.1 * o
    assert (results[0][2].double().cpu() - want).norm() <= 0.1 * room * o.norm() + 4 * U[F32] * want.norm()
    # one rank's merge alone is a part of it: the indices that its partition owns
    parts = [set(i.tolist()) for i, _ in merged]
    assert sum(len(p) for p in parts) == len(set().union(*parts)) == int((total != 0).sum())


@pytest.mark.gpu
def test_limits_are_named_before_memory_is_asked_for():
    """Views of one element: nothing of these sizes is there."""
    one = torch.zeros(1, 1, 1, device="cuda")
    half = one.to(BF16)
    side, deep = (1 << 21) + 1, (1 << 21) + 8
    for call, name in [
            (lambda: zen.orthogonalize(one[0].expand(side, 2)), "2^21"), (lambda: zen.orthogonalize(one[0].expand(1, side)), "2^21"),
            (lambda: zen.orthogonal_step(torch.zeros(2, side, device="cuda"), one[0].expand(2, side), 0.1), "2^21"),
            (lambda: zen.product(half[0].expand(1, deep), half[0].expand(deep, 1)), "2^21"),
            (lambda: zen.product(half.expand(4000, 500, deep), half.expand(4000, deep, 1)), "2^21"),  # 8 TB if it were laid out
            (lambda: zen.product(half.expand(65536, 1, 8), half.expand(65536, 8, 1)), "65535")]:
        with pytest.raises(ValueError) as e:
            call()
        assert name in str(e.value)
    assert zen.product(half.expand(65535, 1, 8), half.expand(65535, 8, 1)).eq(0).all()
    assert zen.orthogonalize(one[0].expand(1 << 21, 1)).eq(0).all()
    assert zen.product(half[0].expand(1, 1 << 21), half[0].expand(1 << 21, 1)).eq(0).all()


def test_more_threads_than_a_launch_takes_are_refused(L):
    """Nothing is launched or dereferenced: addresses are made up."""
    one = ctypes.c_void_p(256)
    most = (1 << 32) - 1  # threads
    assert L.zen_momentum(one, 0, one, 0, most // 256 * 2048 + 1, 0.9, 1, one, 0, None) == _lib.EINVAL
    side = 64 * 4097  # 4097 x 4097 tiles of 256 threads, or fewer and larger ones of as many to their elements
    wide = dict(m=side * 8, n=side * 8, k=64, a_rs=64, b_rs=1, b_cs=64, out_rs=side * 8)
    assert L.zen_product(product_args(**wide)) == _lib.EINVAL
    # (k x n, every second element: laid out first)
    assert L.zen_product(product_args(m=64, n=1 << 30, k=1 << 13, b_rs=2, b_cs=1 << 14, out_rs=1 << 30, workspace=256,
                                      workspace_bytes=1 << 62)) == _lib.EINVAL


@pytest.mark.gpu
@pytest.mark.parametrize("abc,steps", [((70.0, 0.0, 0.0), 1), ((70.0, 0.0, 0.0), 2), ((150.0, 0.0, 0.0), 2), ((8.28, -23.6, 17.3), 2),
                                       ((3.0, -4.0, 2.0), 5), ((1.0, 0.0, 0.0), 3), ((2.0, 0.0, 0.0), 6), ((0.0, 100.0, 0.0), 1),
                                       ((-3.4445, 4.7750, -2.0315), 5)])
@pytest.mark.parametrize("m,n", [(64, 96), (40, 30)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_orthogonalize_with_coefficients_that_take_values_far(abc, steps, m, n, dtype):
    u = update_like(m, n, 430).to(dtype)
    want, room = room_of(u, BF16 if dtype == BF16 else F16, steps=steps, abc=abc)
    got = zen.orthogonalize(u, steps=steps, coefficients=abc)
    assert got.isfinite().all() and off(got, want) <= room


@pytest.mark.gpu
@pytest.mark.parametrize("abc,steps", [((8.28, -23.6, 17.3), 5), ((20.0, -100.0, 90.0), 2), ((3.0, -4.0, 2.0), 6), ((4e4, 0.0, 0.0), 1),
                                       ((200.0, 0.0, 0.0), 3), ((math.nan, 0.0, 0.0), 1), ((1.0, math.inf, 0.0), 1),
                                       ((1.0, 0.0, -math.inf), 5), ((math.inf, 0.0, 0.0), 5)])
def test_coefficients_that_would_leave_the_range_are_refused(abc, steps):
    u = update_like(64, 48, 431)
    w = u.clone()
    with pytest.raises(ValueError, match="coefficients"):
        zen.orthogonalize(u, steps=steps, coefficients=abc)
    with pytest.raises(ValueError, match="coefficients"):
        zen.orthogonal_step(w, u, 0.1, steps=steps, coefficients=abc)
    assert torch.equal(w, u)


@pytest.mark.parametrize("m,n", [(4096, 4096), (2048, 2048), (4096, 1024), (1000, 30000), (8192, 4096)])
@pytest.mark.parametrize("precise", [0, 1])
def test_a_stacks_workspace_stays_near_two_gib(L, m, n, precise):
    """Whatever its length: 2 GiB, beside sums of split tiles (512 tiles of 256 x 256 in fp32) and of squares (8 KiB a matrix)."""
    for count in (1, 7, 40, 1000):
        assert L.zen_orthogonal_workspace(m, n, count, precise) <= (2 << 30) + 512 * 256 * 256 * 4 + (1 << 20)
    few = L.zen_orthogonal_workspace(m, n, 40, precise)
    assert L.zen_orthogonal_workspace(m, n, 1000, precise) == few > L.zen_orthogonal_workspace(m, n, 1, precise)
