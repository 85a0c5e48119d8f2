"""What a training step does with the gradient that the exchange brought: momentum (from the dense bucket or from the
merged lists themselves), matrix products with a residual, and the orthogonalisation of an update by Newton-Schulz
steps.  `Muon` (muon.py) is the optimiser made of them.

Every call works on the current stream of its tensors' device, waits for nothing and can be captured into a graph
(where a status is returned, after _lib.zeros.fresh(device) at the start of the capture).  None of them is
differentiated: with gradients enabled, tensors that require them are refused."""
import torch

from . import _lib


def _workspace(device, nbytes):
    """From torch's allocator, in the order of the current stream: calls on several streams, or captured into several
    graphs, never share one."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _called(t, call, *args):
    """call(*args, stream) with t's device as the current one, for the launches, and its current stream."""
    if not t.is_cuda:
        raise TypeError("expected GPU tensors")
    index = t.device.index
    if index == torch.cuda.current_device():
        return call(*args, _lib.current_handle(index))
    with torch.cuda.device(index):
        return call(*args, _lib.current_handle(index))


# ------------------------------------------------------------------- momentum


def momentum_update(momentum, grad, mu=0.95, nesterov=True, dtype=None, out=None):
    """momentum = mu * momentum + grad, in place, and the update it gives: grad + mu * momentum (nesterov) or the new
    momentum.  One pass over both; computed in fp32, each result rounded once.

    momentum  fp32 or bf16, contiguous        grad  fp32, bf16 or fp16, of the same shape
    dtype     the update's type (default: grad's)
    out       where the update goes; may be grad itself"""
    rc, out = _called(momentum, _lib.host.momentum, _lib.lib().zen_momentum, momentum, grad, mu, nesterov, dtype, out)
    if rc:
        _lib.check(rc, "momentum_update")
    return out


def momentum_update_sparse(momentum, indices_tensors, values_tensors, mu=0.95, nesterov=True, counts=None, dtype=None,
                           out=None, status=None):
    """momentum_update with the gradient as ascending lists of (index, value), zero elsewhere, without the dense tensor in
    between: every rank's list of the second exchange (merge_rounded's result of each, gathered).  A rank's own merge
    (merge_rounded, merge_sparse_flat) is the sum over its partition alone, a part of the gradient only.  Returns
    (update, status int32[1]).

    indices_tensors, values_tensors   a tensor each, or a list of up to 64; int32 or int64 indices into the flat momentum,
              every index once to a list; fp32, bf16 or fp16 values.  An index that several lists hold gets its values
              added in the order of the lists
    counts    how many entries of each list hold: None (all), an int64 tensor on the device (one element per list), or a list of
              such one-element tensors or None
    dtype     the update's type (default: the values')
    status    the status of the call that made the lists (int32[1] on the device, as merge_sparse_flat returns it), where
              nobody has looked at it yet.  If it is not zero, nothing is written; else what this call finds goes into it
    An index outside the momentum, or not larger than its list's last one, sets STAT_BAD_INDEX in the status: nothing is
    written then (the update's contents are whatever its memory held)."""
    indices = indices_tensors if isinstance(indices_tensors, (list, tuple)) else [indices_tensors]
    values = values_tensors if isinstance(values_tensors, (list, tuple)) else [values_tensors]
    counted = counts.reshape(-1) if isinstance(counts, torch.Tensor) else None
    if counted is not None:
        counts = None
    L = _lib.lib()
    ws = None
    if momentum.is_cuda:
        ws = _workspace(momentum.device, L.zen_momentum_lists_workspace(momentum.numel(), len(indices)))
    rc, out, status = _called(momentum, _lib.host.momentum_lists, L.zen_momentum_lists, _lib.zeros.native(), momentum, indices,
                              values, mu, nesterov, counted, counts, dtype, out, status, ws)
    if rc:
        _lib.check(rc, "momentum_update_sparse")
    return out, status


# -------------------------------------------------------------------- product


def product(a, b, residual=None, alpha=1.0, beta=1.0, symmetric=False, dtype=None, out=None):
    """alpha * a @ b + beta * residual, summed in fp32 and rounded once.  torch.addmm is up to a fifth quicker on large
    matrices of one type; this also takes results and residuals of other types, symmetric results and any strides.

    a, b       bf16 or fp16 matrices (m x k and k x n), or stacks of as many; any strides.  Where rows or columns are contiguous
               and begin at multiples of 16 bytes they are read as they lie (a transposed view costs nothing), else
               laid out first.  k is at most 2^21, a stack of 65535 matrices
    residual   m x n (or a stack), fp32, bf16 or fp16, any strides (quickest where it lies as the result does).  It is read
               whatever beta is: NaN in it stays NaN
    symmetric  the caller vouches that a @ b is symmetric (a matrix and its own transpose, powers of a symmetric
               matrix): half of it is computed and mirrored
    dtype      the result's type (default: the residual's, else a's): fp32, bf16 or fp16
    out        where the result goes, any strides; may be the residual itself"""
    L = _lib.lib()
    rc, out = _called(a, _lib.host.product, L.zen_product, L.zen_product_workspace,
                      lambda nbytes: _workspace(a.device, nbytes), a, b, residual, alpha, beta, symmetric, dtype, out)
    if rc:
        _lib.check(rc, "product")
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


def _orthogonal(what, updates, outs, steps, coefficients, eps, precision, weights=False, keep=0.0, gain=0.0):
    if not updates:
        return
    if len(coefficients) != 3:
        raise ValueError(f"{what}: three coefficients")
    L = _lib.lib()
    device = updates[0].device
    rc = _called(updates[0], _lib.host.orthogonal, L.zen_orthogonal, L.zen_orthogonal_workspace,
                 lambda nbytes: _workspace(device, nbytes), what, updates, outs, int(steps), *coefficients,
                 eps, precision != torch.bfloat16, weights, keep, gain)
    if rc:
        _lib.check(rc, what)


def orthogonalize(update, steps=5, coefficients=COEFFICIENTS, eps=1e-7, dtype=None, out=None):
    """The update with its singular values taken to about one: from X = U / (|U| + eps) (Frobenius norm), `steps` times
    X = a X + (b A + c A A) X with A = X X^T, on the side of the smaller dimension.  An update of zeros gives zeros.

    update  a matrix, a stack (3-D) or a list of matrices of one shape; fp32, bf16 or fp16, any strides, rows and columns
            up to 2^21.  Many small matrices are quicker in one call than one by one
    coefficients   a, b, c.  A ValueError, if in so many steps they can take a singular value between 0 and 1 (or its square,
            or b A + c A A) beyond 32752: they would not settle around one
    dtype   the result's type (default: the update's).  It decides the precision: for bf16 the products' operands are
            fp16 where the smaller side is at least 64 (off by less than the result's own rounding then), below
            that, and for fp32 and fp16, they have 22 bits (three products of fp16 each, off by up to twice what products in
            fp32 are); the iterate has 22 bits
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
    _orthogonal("orthogonalize", updates, outs, steps, coefficients, eps, outs[0].dtype if outs else None)
    return out


def orthogonal_step(weight, update, lr, weight_decay=0.0, scale=1.0, steps=5, coefficients=COEFFICIENTS, eps=1e-7,
                    precision=None):
    """weight = (1 - lr * weight_decay) * weight - lr * scale * orthogonalize(update), in place: the last product writes
    the weight itself.  Returns the weight.

    weight, update  a matrix each, a stack or a list of matrices of one shape
    precision       fp32, bf16 or fp16: how precise the orthogonalised update is (see orthogonalize).  Default: as the
                    weight's type asks for; bf16 for fp32 weights is up to two and a half times quicker"""
    weights, updates = _matrices(weight, "weight"), _matrices(update, "update")
    if len(weights) != len(updates):
        raise ValueError(f"orthogonal_step: {len(weights)} weights and {len(updates)} updates")
    if precision is None and weights:
        precision = weights[0].dtype
    if weights and precision not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"precision must be float32, bfloat16 or float16, got {precision}")
    _orthogonal("orthogonal_step", updates, weights, steps, coefficients, eps, precision, True,
                    1.0 - lr * weight_decay, lr * scale)
    return weight
