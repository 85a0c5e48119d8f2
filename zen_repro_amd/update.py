"""What a training step does with the gradient that the exchange brought: momentum (from the dense bucket or from the
merged lists themselves), matrix products with a residual, and the orthogonalisation of an update by Newton-Schulz
steps.  `Muon` (muon.py) is the optimiser made of them.

Every call works on the current stream of its tensors' device, waits for nothing and can be captured into a graph
(a captured call has a workspace of its own).  None of them is differentiated: with gradients enabled, tensors that require
them are refused."""
import contextlib
import ctypes

import torch

from . import _lib

_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _code(t, name, dtypes=(torch.float32, torch.bfloat16, torch.float16)):
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {str(t.dtype)[6:]}")
    return _CODES[t.dtype]


def _same_device(first, *others):
    if not first.is_cuda:
        raise TypeError("expected GPU tensors")
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")


def _no_gradients(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("an optimiser's step is not differentiated: call this under torch.no_grad()")


def _written(*tensors):
    """Tells autograd that these were written in place."""
    for t in tensors:
        torch.autograd.graph.increment_version(t)


def _on(device):
    """The device becomes the current one for the launches, if it is not."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _workspace(device, name, nbytes):
    """The calling thread's buffer of that name.  A captured call's belongs to its graph: two graphs may replay side by
    side, and the thread's buffer may be replaced by a larger one."""
    if not nbytes:
        return None
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    return _lib.scratch.get(device, name, nbytes)


def _extent(t):
    """First byte and the byte behind the last one of what a tensor's elements cover."""
    if t.numel() == 0:
        return 0, 0
    first = t.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _overlap(a, b):
    """Whether two tensors may share memory.  Told apart beside plain stretches: two equally strided matrices whose
    rows lie between each other's (column ranges of one larger matrix)."""
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    if not (a0 < b1 and b0 < a1):
        return False
    if a.dim() == b.dim() == 2 and a.stride() == b.stride() and a.dtype == b.dtype and min(a.stride()) == 1:
        line = 1 if a.stride(1) == 1 else 0  # the dimension whose neighbours are neighbours in memory
        step, size = a.stride(1 - line), a.element_size()
        apart = (b0 - a0) // size % step if step else 0
        if (b0 - a0) % size == 0 and a.shape[line] <= apart <= step - b.shape[line]:
            return False
    return True


def _is(a, b):
    """Whether two tensors are the same elements in the same order."""
    return a.data_ptr() == b.data_ptr() and a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride()


def _one_place(t, name):
    """Refuses a tensor to be written some of whose elements are one place in memory."""
    at = sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1)
    reach = 0
    for s, n in at:
        if s <= reach:
            raise ValueError(f"{name}: several elements are one place in memory")
        reach += (n - 1) * s


# ------------------------------------------------------------------- momentum


def _momentum_checks(momentum, mu, dtype, out, default):
    _code(momentum, "momentum", (torch.float32, torch.bfloat16))
    _lib.require_gpu(momentum, "momentum")
    if not 0.0 <= mu < float("inf"):
        raise ValueError(f"mu must be finite and not negative, got {mu}")
    if out is None:
        out = torch.empty_like(momentum, dtype=dtype or default, requires_grad=False)
    elif dtype is not None and out.dtype != dtype:
        raise TypeError(f"out is {out.dtype}, not {dtype}")
    _code(out, "update")
    _lib.require_gpu(out, "out")
    if out.shape != momentum.shape:
        raise ValueError(f"out has the shape {tuple(out.shape)}, the momentum {tuple(momentum.shape)}")
    if _overlap(out, momentum):
        raise ValueError("out overlaps the momentum")
    return out


def momentum_update(momentum, grad, mu=0.95, nesterov=True, dtype=None, out=None):
    """momentum = mu * momentum + grad, in place, and the update it gives: grad + mu * momentum (nesterov) or the new
    momentum.  One pass over both; computed in fp32, each result rounded once.

    momentum  fp32 or bf16, contiguous        grad  fp32, bf16 or fp16, of the same shape
    dtype     the update's type (default: grad's)
    out       where the update goes; may be grad itself"""
    _same_device(momentum, grad, out)
    _no_gradients(momentum, grad, out)
    code = _code(grad, "grad")
    _lib.require_gpu(grad, "grad")
    if grad.shape != momentum.shape:
        raise ValueError(f"grad has the shape {tuple(grad.shape)}, the momentum {tuple(momentum.shape)}")
    out = _momentum_checks(momentum, mu, dtype, out, grad.dtype)
    if _overlap(grad, momentum) or (_overlap(out, grad) and not _is(out, grad)):
        raise ValueError("grad overlaps the momentum or a part of out")
    with _on(momentum.device):
        rc = _lib.lib().zen_momentum(momentum.data_ptr(), _CODES[momentum.dtype], grad.data_ptr(), code, grad.numel(), mu,
                                     int(bool(nesterov)), out.data_ptr(), _CODES[out.dtype],
                                     _lib.stream_of(momentum.device))
    _lib.check(rc, "momentum_update")
    _written(momentum, out)
    return out


def momentum_update_sparse(momentum, indices_tensors, values_tensors, mu=0.95, nesterov=True, counts=None, dtype=None,
                           out=None):
    """momentum_update with the gradient as ascending lists of (index, value), zero elsewhere: what merge_sparse_flat
    returns, or every rank's list of the second exchange, without the dense tensor in between.  Returns (update,
    status int32[1]).

    indices_tensors, values_tensors   a tensor each, or a list of up to 64; int32 or int64 indices into the flat momentum,
              every index once to a list; fp32, bf16 or fp16 values.  An index that several lists hold gets its values
              added in the order of the lists
    counts    how many entries of each list hold: None (all), an int64 tensor on the device (one element per list), or a list of
              such one-element tensors or None
    dtype     the update's type (default: the values')
    An index outside the momentum, or not larger than its list's last one, sets STAT_BAD_INDEX in the status: nothing is
    written then (the update's contents are whatever its memory held)."""
    indices = indices_tensors if isinstance(indices_tensors, (list, tuple)) else [indices_tensors]
    values = values_tensors if isinstance(values_tensors, (list, tuple)) else [values_tensors]
    lists = len(indices)
    if not 1 <= lists <= _lib.MOMENTUM_LISTS_MOST or len(values) != lists:
        raise ValueError(f"1 to {_lib.MOMENTUM_LISTS_MOST} lists, as many of indices as of values: got {lists} and {len(values)}")
    _same_device(momentum, out, *indices, *values)
    _no_gradients(momentum, out, *values)
    code = _code(values[0], "values")
    if indices[0].dtype not in (torch.int32, torch.int64):
        raise TypeError(f"indices must be int32 or int64, got {indices[0].dtype}")
    for i, v in zip(indices, values):
        _lib.require_gpu(i, "indices")
        _lib.require_gpu(v, "values")
        if i.dtype != indices[0].dtype or v.dtype != values[0].dtype:
            raise TypeError("the lists' indices, and their values, have one type")
        if i.numel() != v.numel():
            raise ValueError(f"a list has {i.numel()} indices and {v.numel()} values")
    n = momentum.numel()
    if n >= 1 << 31:
        raise ValueError("momentum_update_sparse: at most 2^31 - 1 elements")
    if n == 0 and any(i.numel() for i in indices):
        raise ValueError("momentum_update_sparse: entries for an empty momentum")
    if counts is None:
        counts = [None] * lists
    elif isinstance(counts, torch.Tensor):
        if counts.numel() != lists:
            raise ValueError(f"{counts.numel()} counts for {lists} lists")
        counts = list(counts.reshape(-1).split(1))
    if len(counts) != lists:
        raise ValueError(f"{len(counts)} counts for {lists} lists")
    for c in counts:
        if c is not None:
            _same_device(momentum, c)
            if c.dtype != torch.int64 or c.numel() != 1:
                raise TypeError("counts are int64, one element to a list")
    out = _momentum_checks(momentum, mu, dtype, out, values[0].dtype)
    for t in (*indices, *values, *(c for c in counts if c is not None)):
        if _overlap(t, momentum) or _overlap(t, out):
            raise ValueError("momentum_update_sparse: a list overlaps the momentum or out")
    L = _lib.lib()
    pointers, sizes = ctypes.c_void_p * lists, ctypes.c_int64 * lists
    dev = momentum.device
    with _on(dev):
        status = _lib.status_word(dev)
        ws = _workspace(dev, "momentum", L.zen_momentum_lists_workspace(n, lists))
        rc = L.zen_momentum_lists(
            momentum.data_ptr(), _CODES[momentum.dtype], pointers(*(i.data_ptr() for i in indices)),
            int(indices[0].dtype == torch.int64), pointers(*(v.data_ptr() for v in values)), code,
            sizes(*(i.numel() for i in indices)), pointers(*(_lib.ptr(c) for c in counts)), lists, n, mu,
            int(bool(nesterov)), out.data_ptr(), _CODES[out.dtype], _lib.ptr(ws), ws.numel() if ws is not None else 0,
            _lib.ptr(status), _lib.stream_of(dev))
    _lib.check(rc, "momentum_update_sparse")
    _written(momentum, out)
    return out, status


# -------------------------------------------------------------------- product


def _strides(t):
    """Strides of rows, columns and matrices of a 2-D or 3-D tensor."""
    return t.stride(-2), t.stride(-1), t.stride(0) if t.dim() == 3 else 0


def product(a, b, residual=None, alpha=1.0, beta=1.0, symmetric=False, dtype=None, out=None):
    """alpha * a @ b + beta * residual, summed in fp32 and rounded once.

    a, b       bf16 or fp16 matrices (m x k and k x n), or stacks of as many; any strides.  Where rows or columns are contiguous
               and begin at multiples of 16 bytes they are read as they lie (a transposed view costs nothing), else
               laid out first
    residual   m x n (or a stack), fp32, bf16 or fp16, any strides
    symmetric  the caller vouches that a @ b is symmetric (a matrix and its own transpose, powers of a symmetric
               matrix): half of it is computed and mirrored
    dtype      the result's type (default: the residual's, else a's): fp32, bf16 or fp16
    out        where the result goes, any strides; may be the residual itself"""
    _same_device(a, b, residual, out)
    _no_gradients(a, b, residual, out)
    code = _code(a, "a", (torch.bfloat16, torch.float16))
    if b.dtype != a.dtype:
        raise TypeError(f"a is {a.dtype}, b {b.dtype}")
    if a.dim() not in (2, 3) or b.dim() != a.dim():
        raise ValueError("a and b are two matrices, or two stacks of matrices")
    stack = a.shape[:-2]
    m, k, n = a.shape[-2], a.shape[-1], b.shape[-1]
    if b.shape[:-2] != stack or b.shape[-2] != k:
        raise ValueError(f"the shapes {tuple(a.shape)} and {tuple(b.shape)} have no product")
    if symmetric and m != n:
        raise ValueError("a symmetric result is square")
    shape = (*stack, m, n)
    for t, name in ((residual, "residual"), (out, "out")):
        if t is not None and t.shape != shape:
            raise ValueError(f"{name} has the shape {tuple(t.shape)}, the product {shape}")
    if residual is not None:
        _code(residual, "residual")
    if out is None:
        out = torch.empty(shape, dtype=dtype or (residual if residual is not None else a).dtype, device=a.device)
    elif dtype is not None and out.dtype != dtype:
        raise TypeError(f"out is {out.dtype}, not {dtype}")
    out_code = _code(out, "the result")
    _one_place(out, "out")
    if _overlap(out, a) or _overlap(out, b) or (residual is not None and _overlap(out, residual) and not _is(out, residual)):
        raise ValueError("out overlaps an input")
    L = _lib.lib()
    p = _lib.ProductArgs(
        a.data_ptr(), *_strides(a), b.data_ptr(), *_strides(b), code, None, 0, 0, 0, 0, out.data_ptr(), out_code,
        *_strides(out), m, n, k, stack[0] if stack else 1, alpha, beta, int(bool(symmetric)))
    if residual is not None:
        p.c, p.c_dtype = residual.data_ptr(), _CODES[residual.dtype]
        p.c_rs, p.c_cs, p.c_batch = _strides(residual)
    with _on(a.device):
        nbytes = L.zen_product_workspace(ctypes.byref(p))
        ws = _workspace(a.device, "product", nbytes)
        p.workspace, p.workspace_bytes, p.stream = _lib.ptr(ws), nbytes, _lib.stream_of(a.device)
        rc = L.zen_product(ctypes.byref(p))
    _lib.check(rc, "product")
    _written(out)
    return out


# ----------------------------------------------------------- orthogonalisation

COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # of the polynomial a x + b x^3 + c x^5, steep at zero and near one from 0.7 to 1.2


def _matrices(t, name):
    """The matrices of a tensor (2-D: one; 3-D: a stack) or a list of 2-D tensors."""
    if isinstance(t, (list, tuple)):
        if not all(x.dim() == 2 for x in t):
            raise ValueError(f"{name}: a list is one of matrices")
        return list(t)
    if t.dim() == 3:
        return list(t.unbind(0))
    if t.dim() != 2:
        raise ValueError(f"{name}: a matrix, a stack of matrices or a list of matrices")
    return [t]


def _orthogonal(what, updates, outs, steps, coefficients, eps, precise, weights, keep, gain):
    """One zen_orthogonal call for matrices of one shape, one pair of types and one pair of strides."""
    first, out = updates[0], outs[0]
    dev = first.device
    count = len(updates)
    pointers = ctypes.c_void_p * count
    L = _lib.lib()
    rows, cols = first.shape
    with _on(dev):
        nbytes = L.zen_orthogonal_workspace(rows, cols, count, int(precise))
        ws = _workspace(dev, "orthogonal", nbytes)
        p = _lib.OrthogonalArgs(
            pointers(*(t.data_ptr() for t in updates)), _CODES[first.dtype], *first.stride(),
            pointers(*(t.data_ptr() for t in outs)), _CODES[out.dtype], *out.stride(), rows, cols, count, steps,
            *coefficients, eps, int(precise), int(weights), keep, gain, _lib.ptr(ws), nbytes, _lib.stream_of(dev))
        rc = L.zen_orthogonal(ctypes.byref(p))
    _lib.check(rc, what)


def _orthogonal_all(what, updates, outs, steps, coefficients, eps, precision, weights=False, keep=0.0, gain=0.0):
    if not updates:
        return
    _same_device(*updates, *outs)
    _no_gradients(*updates, *outs)
    steps = int(steps)
    if steps < 1:
        raise ValueError(f"{what}: at least one step, got {steps}")
    if len(coefficients) != 3:
        raise ValueError(f"{what}: three coefficients")
    if not eps >= 0:
        raise ValueError(f"{what}: eps must not be negative, got {eps}")
    for u, o in zip(updates, outs):
        _code(u, "update")
        _code(o, "weight" if weights else "out")
        if u.shape != updates[0].shape or u.dtype != updates[0].dtype or o.dtype != outs[0].dtype:
            raise ValueError(f"{what}: the matrices of a call have one shape and one type")
        if o.shape != u.shape:
            raise ValueError(f"{what}: the shapes {tuple(u.shape)} and {tuple(o.shape)} differ")
        _one_place(o, what)
    if updates[0].numel() == 0:
        return
    # what is written lies apart from everything else (an update may be its own result)
    spans = [(*_extent(o), True, o) for o in outs]
    spans += [(*_extent(u), False, u) for u, o in zip(updates, outs) if weights or not _is(u, o)]
    spans.sort(key=lambda span: span[0])
    open_ = []
    for start, end, writes, t in spans:
        open_ = [other for other in open_ if other[0] > start]
        if any((writes or wrote) and _overlap(t, other) for _, wrote, other in open_):
            raise ValueError(f"{what}: a result overlaps another matrix")
        open_.append((end, writes, t))
    groups = {}
    for u, o in zip(updates, outs):
        groups.setdefault((u.stride(), o.stride()), []).append((u, o))
    precise = precision == torch.float32
    for group in groups.values():
        _orthogonal(what, *zip(*group), steps, coefficients, float(eps), precise, weights, keep, gain)
    _written(*outs)


def orthogonalize(update, steps=5, coefficients=COEFFICIENTS, eps=1e-7, dtype=None, out=None):
    """The update with its singular values taken to about one: from X = U / (|U| + eps) (Frobenius norm), `steps` times
    X = a X + (b A + c A A) X with A = X X^T, on the side of the smaller dimension.  An update of zeros gives zeros.

    update  a matrix, a stack (3-D) or a list of matrices of one shape; fp32, bf16 or fp16, any strides.  Many small matrices
            are quicker in one call than one by one
    dtype   the result's type (default: the update's).  It decides the precision: for fp32 every product's operands
            have 22 bits (three products of fp16), else fp16 operands and an iterate of 22 bits
    out     where the result goes, of the update's shape (a list for a list); may be the update itself"""
    updates = _matrices(update, "update")
    listed = isinstance(update, (list, tuple))
    if out is None:
        if listed:
            out = [torch.empty(t.shape, dtype=dtype or t.dtype, device=t.device) for t in updates]
        else:
            out = torch.empty(update.shape, dtype=dtype or update.dtype, device=update.device)
    outs = _matrices(out, "out")
    if len(outs) != len(updates) or (not listed and out.shape != update.shape):
        raise ValueError("orthogonalize: out is not of the update's shape")
    if dtype is not None and any(t.dtype != dtype for t in outs):
        raise TypeError(f"out is not {dtype}")
    _orthogonal_all("orthogonalize", updates, outs, steps, coefficients, eps, outs[0].dtype if outs else None)
    return out


def orthogonal_step(weight, update, lr, weight_decay=0.0, scale=1.0, steps=5, coefficients=COEFFICIENTS, eps=1e-7,
                    precision=None):
    """weight = (1 - lr * weight_decay) * weight - lr * scale * orthogonalize(update), in place: the last product writes
    the weight itself.  Returns the weight.

    weight, update  a matrix each, a stack or a list of matrices of one shape
    precision       fp32, bf16 or fp16: how precise the orthogonalised update is (see orthogonalize).  Default: as the
                    weight's type asks for; bf16 for fp32 weights is some two to three times quicker"""
    weights, updates = _matrices(weight, "weight"), _matrices(update, "update")
    if len(weights) != len(updates):
        raise ValueError(f"orthogonal_step: {len(weights)} weights and {len(updates)} updates")
    if precision is None and weights:
        precision = weights[0].dtype
    if weights and precision not in _CODES:
        raise TypeError(f"precision must be float32, bfloat16 or float16, got {precision}")
    _orthogonal_all("orthogonal_step", updates, weights, steps, coefficients, eps, precision, True,
                    1.0 - lr * weight_decay, lr * scale)
    return weight
