"""Rows that many entries share, and rows sorted by an integer group and back.

A Gaussian scene with a codebook keeps one table of attribute rows and an integer per
Gaussian; training it needs the rows looked up and their gradients summed over the
Gaussians that share them:

* ``table_lookup(table, index, scale)``: ``scale * table[index]``, differentiable in the table;
* ``table_gradient(grad, index, num_rows, scale)``: that gradient by itself, with the mask
  of the rows it touched, as ``SparseGaussianAdam.step(row_mask=...)`` takes it.

Rows that go by group (depth plane, owning GPU, expert), with one or several groups per row:

* ``group_rows(index, num_groups)``: the entries sorted stably by group (a ``RowGroups``);
* ``rows_to_groups(x, groups)``: each row copied to its places, differentiable;
* ``groups_to_rows(y, groups, weights)``: the weighted sum of a row's places, differentiable
  in ``y`` and ``weights``.

An index or group outside its range (-1, say) leaves the entry out: it looks up zeros, adds
nothing to a gradient or a sum, and whatever its weight or gradient holds is not read.
Rows are float32, bfloat16 or float16, contiguous within a row (a slice of a wider tensor
or a row expanded over a batch is used as it is); sums are float32 in a fixed order, so
results repeat bit for bit, and are rounded once; gradients are not differentiable again, and
forward-mode derivatives (dual tensors) are refused.
Nothing is read back to the host: every call can be captured in a CUDA graph, a backward
pass as torch captures any (no earlier autograd graph of the same leaves may be alive).
Every step runs in libcvhrf (cvhrf_table_lookup, cvhrf_table_gradient, cvhrf_group_rows,
cvhrf_rows_to_groups, cvhrf_groups_to_rows); the reference, whose Gaussians own all their
attributes, has no counterpart.
"""
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, profiling

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INDEX_BYTES = {torch.int32: 4, torch.int64: 8}
_MAX_ENTRIES = 2 ** 30 - 1
_MAX_WIDTH = 2 ** 20
_MAX_SCALE = torch.finfo(torch.float32).max


def _call(name, what, device, args):
    """One libcvhrf call on `device` and its current stream, timed as `what`."""
    f = getattr(_lib._lib or _lib.lib(), name)
    at = device.index
    if profiling._active is not None or at != torch._C._cuda_getDevice():
        with torch.cuda.device(device), profiling.timed(what):
            rc = f(args, torch.cuda.current_stream(device).cuda_stream)
    else:
        rc = f(args, torch._C._cuda_getCurrentRawStream(at))
    if rc:
        _lib.check(rc, name)


# Workspaces are multiples of 8 bytes, allocated as elements of the index's type (new_empty of
# the same type is the cheapest allocation there is).
@functools.lru_cache(maxsize=256)
def _gradient_workspace(n, num_rows, width):
    return _lib.lib().cvhrf_table_gradient_workspace_bytes(n, num_rows, width)


@functools.lru_cache(maxsize=256)
def _group_workspace(n, num_groups):
    return _lib.lib().cvhrf_group_rows_workspace_bytes(n, num_groups)


def _rows(t, name):
    """A 2-D tensor of rows whose elements are adjacent, its type's code, width and the
    elements between its rows."""
    code = _TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dim() != 2 or not 1 <= t.shape[1] <= _MAX_WIDTH:
        raise ValueError(f"{name} must be rows x width with 1 <= width <= {_MAX_WIDTH}, got {tuple(t.shape)}")
    stride, one = t.stride()
    width = t.shape[1]
    if one != 1 and width > 1:
        t, stride = t.contiguous(), width
    return t, code, width, stride


def _index(index, device):
    nbytes = _INDEX_BYTES.get(index.dtype)
    if nbytes is None:
        raise TypeError(f"index must be int32 or int64, got {index.dtype}")
    if index.device != device:
        raise ValueError(f"index must be on {device}, got {index.device}")
    n = index.numel()
    if n > _MAX_ENTRIES:
        raise ValueError(f"index has {n} entries: {_MAX_ENTRIES} at most")
    return index.contiguous(), nbytes, n


def _scale(scale):
    if isinstance(scale, torch.Tensor):
        raise TypeError("scale must be a number, not a tensor")
    scale = float(scale)
    if not -_MAX_SCALE <= scale <= _MAX_SCALE:
        raise ValueError(f"scale must be a finite float32, got {scale}")
    return scale


# A call goes through its autograd function where a tensor needs a gradient, and within a
# forward-mode level (forward_ad._current_level >= 0), where a dual tensor does not show and the
# function refuses it.  (The test is written out in each of them: as a function of its own it
# cost a lookup 0.5 of 9 us.)

# ---- shared rows ----------------------------------------------------------------------
def _lookup(table, index, scale):
    table, code, width, stride = _rows(table, "table")
    device = table.device
    index, nbytes, n = _index(index, device)
    out = table.new_empty((*index.shape, width))
    _call("cvhrf_table_lookup", "table_lookup", device, _lib.LOOKUP_ARGS.pack(
        table.data_ptr(), index.data_ptr(), out.data_ptr(), table.shape[0], stride, n, width, code, nbytes, scale))
    return out


def _gradient(grad, index, num_rows, scale, with_mask):
    if grad.dim() != 2:
        if not grad.shape or grad.shape[-1] < 1:
            raise ValueError(f"grad must have rows of 1 element or more, got {tuple(grad.shape)}")
        grad = grad.reshape(-1, grad.shape[-1])
    grad, code, width, stride = _rows(grad, "grad")
    device = grad.device
    index, nbytes, n = _index(index, device)
    out = grad.new_empty((num_rows, width))
    mask = index.new_empty(num_rows, dtype=torch.uint8) if with_mask else None
    need = _gradient_workspace(n, num_rows, width)
    ws = index.new_empty(need // nbytes) if need else None
    _call("cvhrf_table_gradient", "table_gradient", device, _lib.GRADIENT_ARGS.pack(
        grad.data_ptr(), index.data_ptr(), out.data_ptr(), mask.data_ptr() if with_mask else 0,
        ws.data_ptr() if need else 0, need,
        stride, n, num_rows, width, code, nbytes, scale))
    return out, mask


class TableLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale):
        ctx.save_for_backward(index)
        ctx.num_rows, ctx.scale = table.shape[0], scale
        return _lookup(table, index, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        index, = ctx.saved_tensors
        return _gradient(grad, index, ctx.num_rows, ctx.scale, False)[0], None, None


def table_lookup(table, index, scale=1.0):
    """scale * table[index] for a table of rows (V, D) and an int32 or int64 index of any
    shape: (*index.shape, D) in the table's type, zeros where the index is outside [0, V).
    Differentiable in the table (a dense (V, D) gradient, see ``table_gradient``)."""
    scale = _scale(scale)
    if (table.requires_grad and torch.is_grad_enabled()) or forward_ad._current_level >= 0:
        return TableLookup.apply(table, index, scale)
    return _lookup(table, index, scale)


def table_gradient(grad, index, num_rows, scale=1.0):
    """The gradient of ``table_lookup`` with respect to its table of `num_rows` rows: row v is
    scale times the sum of grad[t] over the entries with index[t] = v.  grad has the
    lookup's shape (*index.shape, D).  Returns (gradient (num_rows, D) in grad's type,
    row_mask (num_rows,) uint8: 1 where an entry names the row), so that
    ``SparseGaussianAdam.step(row_mask=row_mask)`` updates the rows that were used.  Not
    differentiable: grad is taken as detached."""
    if grad.shape[:-1] != index.shape or not grad.shape:
        raise ValueError(f"grad must have the shape {tuple(index.shape)} and a row's width, got {tuple(grad.shape)}")
    if not 0 <= num_rows < 2 ** 31 - 1:
        raise ValueError(f"num_rows must be in [0, 2^31 - 1), got {num_rows}")
    return _gradient(grad.detach(), index, num_rows, _scale(scale), True)


# ---- rows by group --------------------------------------------------------------------
class RowGroups:
    """Entries sorted by group (``group_rows``), all int32 on the device: ``order`` (M,) the
    entry at each place, ``slots`` (the index's shape) the place of each entry or -1,
    ``offsets`` (num_groups + 1,) where each group begins and the last one ends.  They are
    read, not written: the moves take their places on trust."""

    __slots__ = ("order", "slots", "offsets", "num_groups", "num_rows", "choices")

    def __init__(self, order, slots, offsets, num_groups, num_rows, choices):
        self.order, self.slots, self.offsets = order, slots, offsets
        self.num_groups, self.num_rows, self.choices = num_groups, num_rows, choices

    def _used(self):
        return self.offsets.data_ptr() + 4 * self.num_groups


def group_rows(index, num_groups):
    """Sort the entries of `index`, (N,) or (N, k) int32 or int64 groups of N rows, stably by
    group.  Entries outside [0, num_groups) come behind the last group and have slot -1."""
    if not index.is_cuda:
        raise ValueError("index must be a CUDA tensor")
    shape = index.shape
    choices = 1 if len(shape) == 1 else shape[1] if len(shape) == 2 else 0
    if choices < 1:
        raise ValueError(f"index must be (N,) or (N, k) with k >= 1, got {tuple(shape)}")
    if not 1 <= num_groups < 2 ** 31 - 1:
        raise ValueError(f"num_groups must be in [1, 2^31 - 1), got {num_groups}")
    device = index.device
    index, nbytes, n = _index(index, device)
    if nbytes == 4:
        order, slots, offsets = index.new_empty(n), index.new_empty(shape), index.new_empty(num_groups + 1)
    else:
        order, slots, offsets = (index.new_empty(s, dtype=torch.int32) for s in (n, shape, num_groups + 1))
    need = _group_workspace(n, num_groups)
    ws = index.new_empty(need // nbytes) if need else None
    _call("cvhrf_group_rows", "group_rows", device, _lib.GROUP_ARGS.pack(
        index.data_ptr(), order.data_ptr(), slots.data_ptr(), offsets.data_ptr(), ws.data_ptr() if need else 0, need,
        n, num_groups, nbytes))
    return RowGroups(order, slots, offsets, num_groups, shape[0], choices)


def _to_groups(x, groups):
    x, code, width, stride = _rows(x, "x")
    device, n, k = x.device, groups.num_rows, groups.choices
    out = x.new_empty((n * k, width))
    _call("cvhrf_rows_to_groups", "rows_to_groups", device, _lib.MOVES_ARGS.pack(
        x.data_ptr(), out.data_ptr(), groups.order.data_ptr(), groups.slots.data_ptr(), groups._used(), 0, n, stride, k,
        width, code, 0))
    return out


def _to_rows(y, groups, weights):
    y, code, width, stride = _rows(y, "y")
    device, n = y.device, groups.num_rows
    out = y.new_empty((n, width))
    w, w_code = (0, 0) if weights is None else (weights.data_ptr(), _TYPES[weights.dtype])
    _call("cvhrf_groups_to_rows", "groups_to_rows", device, _lib.MOVES_ARGS.pack(
        y.data_ptr(), out.data_ptr(), 0, groups.slots.data_ptr(), 0, w, n, stride, groups.choices, width, code, w_code))
    return out


class RowsToGroups(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, groups):
        ctx.groups = groups
        return _to_groups(x, groups)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return _to_rows(grad, ctx.groups, None), None


class GroupsToRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, groups, weights):
        ctx.groups = groups
        # y is read for the weights' gradient alone: it may change or go where none is asked for
        ctx.save_for_backward(y if ctx.needs_input_grad[2] else None, weights)
        return _to_rows(y, groups, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        y, weights = ctx.saved_tensors
        groups = ctx.groups
        grad, code, width, grad_stride = _rows(grad, "grad")
        need_y, _, need_w = ctx.needs_input_grad
        y_at, stride = 0, 0
        if need_w:
            y, _, _, stride = _rows(y, "y")
            y_at = y.data_ptr()
        device = grad.device
        grad_y = grad.new_empty((groups.num_rows * groups.choices, width)) if need_y else None
        grad_w = torch.empty_like(weights) if need_w else None
        w, w_code = (0, 0) if weights is None else (weights.data_ptr(), _TYPES[weights.dtype])
        _call("cvhrf_groups_to_rows_backward", "groups_to_rows_backward", device, _lib.MOVES_BACKWARD_ARGS.pack(
            grad.data_ptr(), y_at, groups.order.data_ptr(), groups.slots.data_ptr(), groups._used(), w,
            grad_y.data_ptr() if need_y else 0, grad_w.data_ptr() if need_w else 0, groups.num_rows, grad_stride,
            stride, groups.choices, width, code, w_code))
        return grad_y, None, grad_w


def _check_groups(t, groups, rows, name):
    if t.dim() != 2 or t.shape[0] != rows:
        raise ValueError(f"{name} must have {rows} rows, got {tuple(t.shape)}")
    if t.device != groups.slots.device:
        raise ValueError(f"{name} must be on {groups.slots.device}, got {t.device}")


def rows_to_groups(x, groups):
    """Rows x (N, D) at their places: (N * k, D), row p the row of entry groups.order[p]; the
    places behind the last group are zeros.  Differentiable in x (the sum over its places)."""
    _check_groups(x, groups, groups.num_rows, "x")
    if (x.requires_grad and torch.is_grad_enabled()) or forward_ad._current_level >= 0:
        return RowsToGroups.apply(x, groups)
    return _to_groups(x, groups)


def groups_to_rows(y, groups, weights=None):
    """Rows y (N * k, D) at their places back to the N rows: out[n] = sum_j weights[n, j]
    y[groups.slots[n, j]], entries left out counting nothing.  weights have the grouped
    index's shape, float32 or y's type (None: ones).  Differentiable in y and weights; the
    gradient of the places behind the last group is zeros."""
    _check_groups(y, groups, groups.num_rows * groups.choices, "y")
    if weights is not None:
        if weights.shape != groups.slots.shape or weights.device != y.device:
            raise ValueError(f"weights must be {tuple(groups.slots.shape)} on {y.device}, got "
                             f"{tuple(weights.shape)} on {weights.device}")
        if weights.dtype not in (torch.float32, y.dtype):
            raise TypeError(f"weights must be float32 or {y.dtype}, got {weights.dtype}")
        weights = weights.contiguous()
    if (torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad))) or (
            forward_ad._current_level >= 0):
        return GroupsToRows.apply(y, groups, weights)
    return _to_rows(y, groups, weights)
