"""Products and orthogonalisation on every tile that the cost table may choose, with every way an operand is stored, split steps and
whole ones, and every way a result goes out.  What a shape takes is asked of the library: a new cost table that moves a
shape to another tile fails here by name, and the shape is to be chosen anew."""
import ctypes

import pytest
import torch

import zen_repro_amd as zen
from zen_repro_amd import _lib
from test_update import A, B, BF16, C, F16, F32, U, normal, product_check

SIDES = {(256, 1): "256", (192, 1): "192", (128, 1): "128", (128, 2): "128, two to a unit", (64, 2): "64"}


def tile(path):
    """(name, split) of what a *_path call says."""
    assert path > 0
    return SIDES[path & 1023, path >> 10 & 3], (path >> 12 & 255) > 1


# m, n, k, a with k as the stride, b with k as the stride, symmetric, tile, split; edges hang over in all of them
PRODUCTS = [
    (64, 65, 72, False, False, False, "64", False), (63, 63, 72, False, False, True, "64", False), (65, 72, 72, False, True, False, "64", False),
    (72, 65, 72, True, False, False, "64", False), (72, 136, 72, True, True, False, "64", False), (72, 72, 72, True, True, True, "64", False),
    (65, 63, 2056, False, False, False, "64", True), (63, 63, 2056, False, False, True, "64", True), (65, 64, 2056, False, True, False, "64", True),
    (64, 65, 2056, True, False, False, "64", True), (72, 72, 2056, True, True, False, "64", True), (72, 72, 2056, True, True, True, "64", True),
    (1033, 2951, 136, False, False, False, "128", False), (2441, 2441, 136, False, False, True, "128", False),
    (1033, 2952, 136, False, True, False, "128", False), (1032, 2951, 136, True, False, False, "128", False),
    (1032, 2952, 136, True, True, False, "128", False), (2440, 2440, 136, True, True, True, "128", False),
    (777, 1289, 4104, False, False, False, "128", True), (1417, 1417, 4104, False, False, True, "128", True),
    (777, 1288, 4104, False, True, False, "128", True), (776, 1289, 4104, True, False, False, "128", True),
    (776, 1288, 4104, True, True, False, "128", True), (1416, 1416, 4104, True, True, True, "128", True),
    (2697, 2695, 264, False, False, False, "128, two to a unit", False), (3465, 3465, 520, False, False, True, "128, two to a unit", False),
    (2697, 2696, 264, False, True, False, "128, two to a unit", False), (2696, 2695, 264, True, False, False, "128, two to a unit", False),
    (2696, 2696, 264, True, True, False, "128, two to a unit", False), (3464, 3464, 520, True, True, True, "128, two to a unit", False),
    (1673, 4615, 264, False, False, False, "192", False), (4105, 4105, 264, False, False, True, "192", False),
    (1289, 2951, 4104, False, False, False, "192", True),
    (2697, 4361, 520, False, False, False, "256", False), (4361, 4361, 2056, False, False, True, "256", False),
    (2697, 4360, 520, False, True, False, "256", False), (2696, 4361, 520, True, False, False, "256", False),
    (2696, 4360, 520, True, True, False, "256", False), (4104, 4104, 2056, True, True, True, "256", False)]
STACKS = [(3, 777, 2441, 520, "128, two to a unit"), (5, 1289, 2441, 264, "192"), (5, 1000, 2441, 520, "256")]

ORTHOGONAL = [  # rows, columns, matrices; bf16: X X^T, A A, the bracket and X; then the same with 22 bits
    (64, 64, 1, BF16), (64, 1930, 1, BF16), (769, 769, 8, BF16), (1030, 1030, 8, BF16), (1030, 1290, 12, BF16), (769, 5000, 3, BF16),
    (1500, 1500, 8, BF16),
    (64, 64, 1, F32), (64, 769, 1, F32), (520, 769, 12, F32), (1500, 1500, 1, F32), (769, 1030, 12, F32), (1030, 1030, 1, F32),
    (1290, 1290, 5, F32), (1290, 3200, 1, F32), (1030, 3200, 2, F32), (1290, 1290, 12, F32), (3200, 3200, 1, F32), (1930, 2180, 1, F32),
    (520, 3460, 8, F32)]


def product_tile(m, n, k, a, b, symmetric=False, batch=1):
    """(name, split) for operands with these strides (rows, columns, matrices) that are read as they lie, and how they are read."""
    p = _lib.ProductArgs(a=256, a_rs=a[0], a_cs=a[1], a_batch=a[2], b=256, b_rs=b[0], b_cs=b[1], b_batch=b[2], dtype=_lib.BF16,
                         out=256, out_dtype=_lib.BF16, out_rs=n, out_cs=1, m=m, n=n, k=k, batch=batch, alpha=1, symmetric=symmetric)
    path = _lib.lib().zen_product_path(ctypes.byref(p))
    assert not path >> 22, "laid out first"
    return (*tile(path), bool(path >> 20 & 1), bool(path >> 21 & 1))


def orthogonal_tiles(m, n, count, dtype):
    L = _lib.lib()
    return [tile(L.zen_orthogonal_path(m, n, count, int(dtype != BF16), product)) for product in range(3)]


def test_the_shapes_take_every_tile():
    seen = set()
    for m, n, k, a_strided, b_strided, symmetric, name, split in PRODUCTS:
        a, b = (1, m, 0) if a_strided else (k, 1, 0), (n, 1, 0) if b_strided else (1, k, 0)
        assert product_tile(m, n, k, a, b, symmetric) == (name, split, a_strided, b_strided), (m, n, k)
        seen.add((name, a_strided, b_strided, symmetric))
    ways = [(False, False, False), (False, True, False), (True, False, False), (True, True, False), (False, False, True), (True, True, True)]
    sides = set(SIDES.values())
    # 192 is for operands with k contiguous
    assert seen == {(side, *way) for side in sides for way in ways if side != "192" or not (way[0] or way[1])}
    for count, m, n, k, name in STACKS:
        assert product_tile(m, n, k, (k, 1, m * k), (1, k, n * k), batch=count)[0] == name
    steps = [[set(), set(), set()], [set(), set(), set()]]
    for m, n, count, dtype in ORTHOGONAL:
        for product, taken in enumerate(orthogonal_tiles(m, n, count, dtype)):
            steps[dtype != BF16][product].add(taken)
    for products in steps:
        for taken in products:
            assert {name for name, _ in taken} == sides
    assert {name for products in steps for taken in products for name, split in taken if split} == sides


def test_paths_of_bad_arguments_are_refused():
    L = _lib.lib()
    assert L.zen_product_path(None) == _lib.EINVAL
    assert L.zen_product_path(ctypes.byref(_lib.ProductArgs(dtype=7))) == _lib.EINVAL
    for bad in ((0, 5, 1, 0, 0), (5, 5, 0, 0, 0), (5, (1 << 21) + 1, 1, 0, 0), (5, 5, 1, 0, 3), (5, 5, 1, 0, -1)):
        assert L.zen_orthogonal_path(*bad) == _lib.EINVAL


def up8(n):
    return (n + 7) // 8 * 8


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,a_strided,b_strided,symmetric,name,split", PRODUCTS)
def test_product_on_every_tile(m, n, k, a_strided, b_strided, symmetric, name, split):
    dtype = F16 if symmetric else BF16
    a = normal((k, m), 500, dtype).t() if a_strided else normal((m, k), 500, dtype)
    b = a.t() if symmetric else normal((k, n), 501, dtype) if b_strided else normal((n, k), 501, dtype).t()
    assert product_tile(m, n, k, (*a.stride(), 0), (*b.stride(), 0), symmetric) == (name, split, a_strided, b_strided)
    # whole lines, lines that are columns, and one by one; with a residual that lies as the result does, and without
    for number, out_type in enumerate((F16 if symmetric else BF16, F32, BF16)):
        room = torch.full((m + 1, up8(n)), 7.0, device="cuda", dtype=out_type) if number == 0 else \
            torch.full((n + 1, up8(m)), 7.0, device="cuda", dtype=out_type) if number == 1 else \
            torch.full((m + 1, up8(n) + 1), 7.0, device="cuda", dtype=out_type)
        out = room[:n, :m].t() if number == 1 else room[:m, :n]
        c = None
        if number != 2 and not (symmetric and number == 0):
            c = torch.empty_strided(out.shape, out.stride(), device="cuda", dtype=out_type).copy_(normal((m, n), 502))
        zen.product(a, b, residual=c, alpha=0.5, beta=-1.5, symmetric=symmetric, out=out)
        product_check(out, a, b, c, 0.5, -1.5)
        if symmetric and c is None:
            assert torch.equal(out, out.t())
        out.fill_(7.0)
        assert room.eq(7.0).all()


def among_nans(rows, cols, seed, dtype):
    """A matrix with NaN behind it, whole tiles and steps far, in rows and in columns."""
    room = torch.full((rows + 512, up8(cols) + 512), float("nan"), device="cuda", dtype=dtype)
    room[:rows, :cols] = normal((rows, cols), seed, dtype)
    return room[:rows, :cols]


@pytest.mark.gpu
@pytest.mark.parametrize("rest", [8, 40])  # k in the last step; the loads behind its first one begin in the middle of it and behind it
@pytest.mark.parametrize("m,n,k,a_strided,b_strided,symmetric,name,split", [p for p in PRODUCTS if not p[5]])
def test_nothing_behind_an_operand_comes_in(m, n, k, a_strided, b_strided, symmetric, name, split, rest):
    k += rest - k % 64
    a = among_nans(k, m, 530, F16).t() if a_strided else among_nans(m, k, 530, F16)
    b = among_nans(k, n, 531, F16) if b_strided else among_nans(n, k, 531, F16).t()
    tiled = product_tile(m, n, k, (*a.stride(), 0), (*b.stride(), 0))
    assert tiled == (name, split, a_strided, b_strided)
    product_check(zen.product(a, b), a, b, None, 1.0, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("count,m,n,k,name", STACKS)
def test_product_of_stacks_on_large_tiles(count, m, n, k, name):
    a, b = normal((count, m, k), 510, F16), normal((count, n, k), 511, F16).transpose(1, 2)
    c = normal((count, m, n), 512, F16)
    out = zen.product(a, b, residual=c, alpha=0.25, beta=2.0)
    for i in range(count):
        product_check(out[i], a[i], b[i], c[i], 0.25, 2.0)


def newton_schulz_on_the_card(u, dtype=torch.float64):
    """In 64 bits, or what elementary torch operations in 32 make of it; rows <= columns."""
    x = u.to(dtype)
    x = x / (x.norm() + 1e-7)
    for _ in range(5):
        g = x @ x.T.contiguous()
        x = A * x + (B * g + C * (g @ g)) @ x
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,count,dtype", ORTHOGONAL)
def test_orthogonal_on_every_tile(m, n, count, dtype):
    """As fp32 weights of zeros get it, wide and tall updates, in whole lines and one by one."""
    u = normal((count, m, n), 520)
    wants = [newton_schulz_on_the_card(x) for x in u]
    rooms = torch.full((count, m + 1, up8(n) + 1), 7.0, device="cuda")
    odd = rooms[:, :m, :n]
    tall = torch.zeros(count, n, up8(m), device="cuda")[:, :, :m]  # columns of the result's side are lines
    plain = torch.zeros(count, m, up8(n), device="cuda")[:, :, :n]
    for part in (plain, odd, tall):
        part.zero_()
        given = u.transpose(1, 2) if part is tall else u
        zen.orthogonal_step(part, given, 1.0, scale=-1.0, precision=dtype)
        for got, x, want in zip(part, u, wants):
            if dtype == BF16:  # fewer bits do less than rounding to bf16 would
                room = ((want.to(BF16).double() - want).norm() / want.norm()).item()
            else:  # 22 bits: four times what fp32 products do
                room = 4 * max(((newton_schulz_on_the_card(x, F32).double() - want).norm() / want.norm()).item(), 4 * U[F32])
            off = (got.T if part is tall else got).double() - want
            assert off.norm() <= room * want.norm()
            # each is a sum of many roundings: sixteen times their mean is none of them
            assert off.abs().max() <= 16 * room * want.square().mean().sqrt()
    odd.fill_(7.0)
    assert rooms.eq(7.0).all()
