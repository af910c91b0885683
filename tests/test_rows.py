"""Rows shared by many entries and rows sorted by group (rows.py) against plain 64-bit
definitions, at the sizes, types, strides and left-out entries where they can go wrong.

Tolerances: u = 2^-24 is half a step of float32, eps(t) / 2 of a result of type t.  A sum of
n float32 terms in any order is off by at most (n - 1) u sum|term| (first order in u; n is
used), a product by u, and the rounding to t by eps(t) / 2 of the value (or half the smallest
subnormal).  No constant beyond these is added, except 1 + 2^-10 for the terms of second order.
"""
import ctypes
import os
import re

import pytest
import torch

from complex_valued_holographic_radiance_fields_b200 import _lib
from complex_valued_holographic_radiance_fields_b200 import rows as R

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def close(got, exact, slack):
    """got (any type) against exact (float64), with `slack` (float64) before the last rounding."""
    t = got.dtype
    info = torch.finfo(t)
    tol = (slack + (exact.abs() + slack) * info.eps / 2 + info.smallest_normal * info.eps / 2) * (1 + 2.0 ** -10)
    off = (got.double() - exact).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), float(off[bad].max()), float(tol[bad].min()))


def normal(shape, dtype, seed, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(shape, generator=g, device=dev).to(dtype)


def integers(n, high, seed, low=0, dtype=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(low, high, (n,), generator=g, device="cuda").to(dtype)


def inside_of(index, rows):
    return (index >= 0) & (index < rows)


# ---- shared rows ----------------------------------------------------------------------
def lookup_64(table, index, scale):
    index = index.long()
    out = torch.zeros(*index.shape, table.shape[1], dtype=torch.float64, device=table.device)
    ok = inside_of(index, table.shape[0])
    out[ok] = table[index[ok]].double() * scale
    return out


def gradient_64(grad, index, rows, scale):
    """The exact sums, sum |term| and the number of terms of each row."""
    index, grad = index.reshape(-1).long(), grad.reshape(-1, grad.shape[-1])
    at = torch.nonzero(inside_of(index, rows))[:, 0]
    total = torch.zeros(rows, grad.shape[1], dtype=torch.float64, device=grad.device)
    size, count = torch.zeros_like(total), torch.zeros(rows, dtype=torch.float64, device=grad.device)
    g = grad[at].double() * scale
    total.index_add_(0, index[at], g)
    size.index_add_(0, index[at], g.abs())
    count.index_add_(0, index[at], torch.ones_like(at, dtype=torch.float64))
    return total, size, count


def check_gradient(got, mask, grad, index, rows, scale):
    total, size, count = gradient_64(grad, index, rows, scale)
    close(got, total, (count[:, None] + 1) * U * size)
    assert torch.equal(mask, (count > 0).to(torch.uint8))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 7, 8, 17, 20, 59, 64, 129, 333, 515, 1024, 2047, 2049, 4099, 4104])
@pytest.mark.parametrize("n,rows", [(1, 1), (1, 5000), (7, 3), (2049, 64)])
def test_lookup(cuda, dtype, width, n, rows):
    table = normal((rows, width), dtype, width)
    for itype in (torch.int32, torch.int64):
        index = integers(n, rows + 2, n + rows, -2, itype)   # some outside on either side
        for scale in (1.0, -0.7, 45.25):
            out = R.table_lookup(table, index, scale)
            exact = lookup_64(table, index, scale)
            assert out.dtype == dtype and out.shape == exact.shape
            close(out, exact, 0.0 * exact if scale == 1.0 else U * exact.abs())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 8, 12, 20, 59, 64, 130, 256, 333, 1000, 2049, 2056])
@pytest.mark.parametrize("n,rows", [(1, 1), (1, 3000), (5, 2), (513, 1), (2048, 40), (2049, 40), (300, 20011), (3000, 20011), (9000, 700)])
def test_gradient(cuda, dtype, width, n, rows):
    grad = normal((n, width), dtype, width + n)
    for itype in (torch.int32, torch.int64):
        index = integers(n, rows + 1, n + rows, -1, itype)
        got, mask = R.table_gradient(grad, index, rows, 0.75)
        assert got.dtype == dtype
        check_gradient(got, mask, grad, index, rows, 0.75)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [257, 1023, 4736, 4737, 4744, 9001])
@pytest.mark.parametrize("n,rows", [(1, 1), (1, 200), (7, 33), (2048, 3), (2048, 300), (600, 5000)])
def test_gradient_of_few_wide_rows(cuda, dtype, width, n, rows):
    if rows * width > 6_000_000:
        width = width // 8 * 2 + 1
    few_wide_rows(dtype, width, n, rows)


@gpu
@pytest.mark.parametrize("n,rows,width", [(5, 70001, 957), (5, 70001, 960), (2048, 2 ** 24, 4), (2048, 2 ** 24 + 1, 4)])
def test_gradient_of_few_entries_in_large_tables(cuda, n, rows, width):
    few_wide_rows(torch.bfloat16, width, n, rows)


def few_wide_rows(dtype, width, n, rows):
    grad = normal((n, width), dtype, width + n)
    for kind in ("mixed", "one_row"):
        index = integers(n, rows + 1, n + rows, -1) if kind == "mixed" else torch.full((n,), rows - 1, device="cuda")
        got, mask = R.table_gradient(grad, index, rows, 0.75)
        check_gradient(got, mask, grad, index, rows, 0.75)


def skewed(kind, n, rows):
    if kind == "one_row":
        return torch.full((n,), rows // 2, device="cuda")
    if kind == "first_and_last":
        return torch.where(integers(n, 2, 1) == 1, rows - 1, 0)
    if kind == "none":
        return torch.full((n,), -1, device="cuda")
    if kind == "sorted":
        return integers(n, rows, 2).sort()[0]
    if kind == "reversed":
        return integers(n, rows, 3).sort(descending=True)[0]
    if kind == "half_in_one":
        return torch.where(integers(n, 2, 4) == 1, rows // 3, integers(n, rows, 5))
    u = torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    return (u.pow(4) * rows).long().clamp_(max=rows - 1)   # "popular"


@gpu
@pytest.mark.parametrize("kind", ["one_row", "first_and_last", "none", "sorted", "reversed", "half_in_one", "popular"])
@pytest.mark.parametrize("n,rows,width,dtype", [(100003, 4096, 3, torch.float32), (70001, 257, 59, torch.float32),
                                                (20000, 30000, 264, torch.bfloat16), (40000, 2, 130, torch.float16),
                                                (3001, 1, 8, torch.float32), (300000, 65536, 4, torch.float32),
                                                (1500001, 100, 5, torch.float32), (100003, 511, 32, torch.bfloat16),
                                                (90001, 16384, 1, torch.float16), (90001, 512, 33, torch.float32)])
def test_gradient_of_skewed_rows(cuda, kind, n, rows, width, dtype):
    grad = (normal((n, width), torch.float32, n) * 0.05).to(dtype)
    index = skewed(kind, n, rows)
    got, mask = R.table_gradient(grad, index, rows)
    check_gradient(got, mask, grad, index, rows, 1.0)
    again, mask2 = R.table_gradient(grad, index, rows)
    assert torch.equal(got, again) and torch.equal(mask, mask2)


@gpu
@pytest.mark.parametrize("rows", [255, 256, 257, 511, 512, 513, 65536, 262144, 262145, (1 << 24) + 3])
def test_gradient_at_the_edges_of_the_sort(cuda, rows):
    index = torch.cat([integers(5000, rows, rows), torch.tensor([0, rows - 1, rows - 1, rows, -1], device="cuda")])
    grad = normal((index.numel(), 2), torch.float32, 1)
    got, mask = R.table_gradient(grad, index, rows)
    check_gradient(got, mask, grad, index, rows, 1.0)


@gpu
def test_indices_far_outside(cuda):
    table = normal((100, 6), torch.float32, 0)
    index = torch.tensor([2 ** 62, -2 ** 63, 2 ** 32 + 5, -2 ** 32 + 5, 2 ** 31, 99, 100, 2 ** 63 - 1], device="cuda")
    out = R.table_lookup(table, index)
    assert torch.equal(out[5], table[99])
    assert not out[[0, 1, 2, 3, 4, 6, 7]].any()
    grad = torch.full((8, 6), float("nan"), device="cuda")
    grad[5] = 1.0
    got, mask = R.table_gradient(grad, index, 100)          # what is left out is not read, NaN or not
    assert torch.equal(mask.nonzero()[:, 0], torch.tensor([99], device="cuda"))
    assert torch.equal(got[99], torch.ones(6, device="cuda")) and not got[:99].any()
    groups = R.group_rows(index, 100)
    assert groups.offsets[100] == 1 and groups.slots[5] == 0


@gpu
def test_infinities_stay_in_their_row(cuda):
    grad = torch.ones(64, 5, device="cuda")
    grad[10, 2], grad[11, 2], grad[12, 3] = float("inf"), float("-inf"), float("nan")
    index = torch.arange(64, device="cuda") // 2
    got, _ = R.table_gradient(grad, index, 40)
    exact = torch.zeros(40, 5, device="cuda").index_add_(0, index, grad)
    assert torch.equal(torch.nan_to_num(got, 7, 8, 9), torch.nan_to_num(exact, 7, 8, 9))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows(cuda, dtype):
    big = normal((50, 100), dtype, 0)
    index = integers(70, 50, 1)
    for table in (big[:, 8:40], big[:, 3:36], big[::2], big.t(), big[:, ::3], big[:, 5:6]):
        idx = index % table.shape[0]
        assert torch.equal(R.table_lookup(table, idx), table[idx])
    wide = normal((70, 100), dtype, 2)
    for grad in (wide[:, 8:40], wide[:, 1:34], wide[:, ::2], wide[:1].expand(70, 100), wide[:, :1].expand(70, 20)):
        got, mask = R.table_gradient(grad, index, 50)
        check_gradient(got, mask, grad.contiguous(), index, 50, 1.0)
    # indices of other shapes and orders
    square = index[:64].reshape(8, 8).t()
    assert torch.equal(R.table_lookup(big, square), big[square])
    got, mask = R.table_gradient(wide[:64].reshape(8, 8, 100), square, 50)
    check_gradient(got, mask, wide[:64], square.reshape(-1), 50, 1.0)
    assert torch.equal(R.table_lookup(big, index[3]), big[index[3]])          # one index: one row


@gpu
def test_nothing_to_do(cuda):
    table = normal((5, 12), torch.float32, 0)
    empty = torch.empty(0, dtype=torch.int64, device="cuda")
    assert R.table_lookup(table, empty).shape == (0, 12)
    got, mask = R.table_gradient(torch.empty(0, 12, device="cuda"), empty, 5)
    assert got.shape == (5, 12) and not got.any() and not mask.any()
    none = torch.empty(0, 12, device="cuda")
    assert not R.table_lookup(none, torch.zeros(3, dtype=torch.int64, device="cuda")).any()
    got, mask = R.table_gradient(table, torch.zeros(5, dtype=torch.int64, device="cuda"), 0)
    assert got.shape == (0, 12) and mask.shape == (0,)
    groups = R.group_rows(empty, 3)
    assert groups.order.numel() == 0 and not groups.offsets.any()
    assert R.rows_to_groups(none, groups).shape == (0, 12)
    assert R.groups_to_rows(none, groups).shape == (0, 12)


@gpu
def test_offsets_beyond_32_bits(cuda):
    rows, width = 1100000, 2048                       # 2.25e9 elements
    table = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    last = torch.tensor([rows - 1, 1048576, 1048575, 0, rows - 2], device="cuda")
    table[last] = normal((5, width), torch.bfloat16, 0)
    assert torch.equal(R.table_lookup(table, last), table[last])
    del table
    grad = normal((5, width), torch.bfloat16, 1)
    got, mask = R.table_gradient(grad, last, rows)
    assert torch.equal(got[last], grad)
    assert int(mask.sum()) == 5 and int(torch.count_nonzero(got)) == int(torch.count_nonzero(grad))
    del got
    # a wide batch: the places of the rows go beyond 2^31 elements
    n = 1050000
    index = (torch.arange(n, device="cuda") % 3).to(torch.int32)
    groups = R.group_rows(index, 3)
    x = torch.empty(n, width, dtype=torch.bfloat16, device="cuda")
    x[-3:] = normal((3, width), torch.bfloat16, 2)
    xs = R.rows_to_groups(x, groups)
    assert torch.equal(xs[groups.slots[-3:].long()], x[-3:])
    del x
    assert torch.equal(R.groups_to_rows(xs, groups)[-3:], xs[groups.slots[-3:].long()])


@gpu
@pytest.mark.parametrize("dtype,width,n", [(torch.bfloat16, 2048, 1050000),     # aligned rows
                                           (torch.bfloat16, 2047, 1050000),     # tiles
                                           (torch.bfloat16, 4097, 525000),      # words and spans
                                           (torch.float16, 15, 144000000)])     # flat
def test_every_layout_beyond_32_bits(cuda, dtype, width, n):
    """Inputs, outputs and gradients of more than 2^31 elements, checked at their ends and at the border."""
    border = 2 ** 31 // width
    assert 4 < border < n - 4
    some = torch.tensor([0, 1, border - 1, border, border + 1, n - 2, n - 1], device="cuda")
    x = torch.zeros(n, width, dtype=dtype, device="cuda")
    x[some] = normal((7, width), dtype, 0)
    index = torch.arange(n, dtype=torch.int32, device="cuda")
    assert torch.equal(R.table_lookup(x, some), x[some])
    assert torch.equal(R.table_lookup(x, index)[some], x[some])
    got, mask = R.table_gradient(x, n - 1 - index, n)
    assert torch.equal(got[n - 1 - some], x[some]) and int(mask.sum()) == n
    assert int(torch.count_nonzero(got)) == int(torch.count_nonzero(x))
    del got, mask

    g = R.group_rows(index % 3, 3)
    at = g.slots[some].long()
    assert torch.equal(g.order[at].long(), some)
    leaf = x.requires_grad_(True)
    xs = R.rows_to_groups(leaf, g)
    assert torch.equal(xs[at], x[some]) and torch.equal(xs[some], x[g.order[some].long()])
    dx, = torch.autograd.grad(xs, leaf, xs.detach())
    assert torch.equal(dx[some], x[some])
    del dx
    y, w = xs.detach().requires_grad_(True), torch.rand(n, device="cuda").requires_grad_(True)
    out = R.groups_to_rows(y, g, w)
    exact = w.detach()[some, None].double() * x.detach()[some].double()
    close(out.detach()[some], exact, U * exact.abs())
    dy, dw = torch.autograd.grad(out, (y, w), x.detach())
    close(dy[at], exact, U * exact.abs())
    terms = x.detach()[some].double().square()
    close(dw[some], terms.sum(1), width * U * terms.sum(1))


# ---- rows by group --------------------------------------------------------------------
def places_64(index, groups):
    """(order, slots, offsets) by a stable sort on the host."""
    flat = index.reshape(-1).long().cpu()
    key = torch.where(inside_of(flat, groups), flat, groups)
    order = torch.sort(key, stable=True)[1]
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel())
    slots = torch.where(key < groups, place, -1).reshape(index.shape)
    offsets = torch.zeros(groups + 1, dtype=torch.int64)
    offsets[1:] = torch.bincount(key, minlength=groups + 1)[:groups].cumsum(0)
    return order, slots, offsets


@gpu
@pytest.mark.parametrize("groups", [1, 2, 3, 7, 64, 255, 256, 510, 511, 512, 1000, 70000])
@pytest.mark.parametrize("n,k", [(1, 1), (31, 1), (5, 3), (1024, 1), (1025, 2), (4096, 2), (8193, 1), (20011, 4), (310007, 1)])
def test_groups(cuda, groups, n, k):
    for itype in (torch.int32, torch.int64):
        index = integers(n * k, groups + 1, n + groups, -1, itype).reshape(n, k)
        index = index[:, 0] if k == 1 else index
        got = R.group_rows(index, groups)
        for a, b in zip((got.order, got.slots, got.offsets), places_64(index, groups)):
            assert a.dtype == torch.int32 and torch.equal(a.long().cpu(), b)


@gpu
@pytest.mark.parametrize("groups", [8191, 8192, 8193, 65537, 1000003])
@pytest.mark.parametrize("n", [1, 5000, 8192, 8193])
def test_more_groups_than_entries(cuda, groups, n):
    for itype in (torch.int32, torch.int64):
        index = integers(n, groups + 1, n + groups, -1, itype)
        got = R.group_rows(index, groups)
        for a, b in zip((got.order, got.slots, got.offsets), places_64(index, groups)):
            assert torch.equal(a.long().cpu(), b)


@gpu
def test_groups_of_one_kind(cuda):
    for value in (0, 2, -1, 9):
        index = torch.full((5000,), value, dtype=torch.int32, device="cuda")
        got = R.group_rows(index, 3)
        for a, b in zip((got.order, got.slots, got.offsets), places_64(index, 3)):
            assert torch.equal(a.long().cpu(), b)


@gpu
@pytest.mark.parametrize("dtype,wtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         (torch.float16, None)])
@pytest.mark.parametrize("width", [1, 3, 8, 17, 20, 59, 64, 333, 530, 1024, 2051, 2056])
@pytest.mark.parametrize("n,k,groups", [(1, 1, 1), (3, 8, 8), (301, 2, 7), (1000, 3, 300)])
def test_moves_and_their_gradients(cuda, dtype, wtype, width, n, k, groups):
    moves_and_their_gradients(dtype, wtype, width, n, k, groups)


@gpu
@pytest.mark.parametrize("dtype,wtype", [(torch.float32, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("width", [2, 5, 6, 7, 12, 33, 40, 41, 63, 66, 129])
@pytest.mark.parametrize("n,k,groups", [(1, 128, 200), (70, 129, 200), (1200, 1, 3), (777, 7, 9), (20, 300, 40)])
def test_moves_of_narrow_rows_and_many_choices(cuda, dtype, wtype, width, n, k, groups):
    moves_and_their_gradients(dtype, wtype, width, n, k, groups)


@gpu
@pytest.mark.parametrize("dtype,wtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("width", [260, 1032, 4096, 4097, 8200, 9001])
@pytest.mark.parametrize("n,k,groups", [(1, 1, 1), (1, 8, 16), (2, 3, 5), (64, 4, 32), (700, 2, 9)])
def test_moves_of_few_wide_rows(cuda, dtype, wtype, width, n, k, groups):
    moves_and_their_gradients(dtype, wtype, width, n, k, groups)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [4096, 4097, 8200, 9001, 65544])
@pytest.mark.parametrize("n", [1, 3, 64])
def test_lookup_of_few_wide_rows(cuda, dtype, width, n):
    table, index = normal((50, width), dtype, 1), integers(n, 51, 2, -1)
    inside = index >= 0
    exact = torch.where(inside[:, None], table[index.clamp(min=0)].double() * 0.75, 0.0)
    close(R.table_lookup(table, index, 0.75), exact, 0 * exact)


def moves_and_their_gradients(dtype, wtype, width, n, k, groups):
    index = integers(n * k, groups + 1, n + width, -1).reshape(n, k)
    if n > 1:
        index[n // 2] = -1                                   # a row without any group
    ix = index[:, 0] if k == 1 else index
    g = R.group_rows(ix, groups)
    order, slots, offsets = (t.cuda() for t in places_64(ix, groups))
    used = int(offsets[-1])
    x = normal((n, width), dtype, 1).requires_grad_(True)
    y0 = normal((n * k, width), dtype, 2)
    y0[used:] = float("nan")                                 # what is left out is not read
    y = y0.clone().requires_grad_(True)
    w = None
    if wtype is not None:
        w0 = torch.rand(ix.shape, device="cuda").to(wtype)
        w0[~inside_of(ix, groups)] = float("nan")
        w = w0.clone().requires_grad_(True)
    d_xs, d_out = normal((n * k, width), dtype, 3), normal((n, width), dtype, 4)
    d_xs[used:] = float("nan")

    xs = R.rows_to_groups(x, g)
    assert torch.equal(xs[:used], x.detach()[order[:used] // k]) and not xs[used:].any()
    out = R.groups_to_rows(y, g, w)

    kept = (slots >= 0).reshape(n, k)
    at = slots.reshape(n, k).clamp(min=0)
    weight = torch.ones(n, k, dtype=torch.float64, device="cuda") if w is None else w0.double().reshape(n, k)
    weight = torch.where(kept, weight, 0.0)
    rows = torch.where(kept[:, :, None], y0.double()[at], 0.0)
    terms = weight[:, :, None] * rows
    close(out, terms.sum(1), k * U * terms.abs().sum(1))

    leaves = (x, y) if w is None else (x, y, w)
    got = torch.autograd.grad((xs, out), leaves, (d_xs, d_out))
    terms = torch.where(kept[:, :, None], d_xs.double()[at], 0.0)
    close(got[0], terms.sum(1), k * U * terms.abs().sum(1))
    exact = torch.zeros(n * k, width, dtype=torch.float64, device="cuda")
    exact[at[kept]] = (weight[:, :, None] * d_out.double()[:, None, :])[kept]
    close(got[1], exact, U * exact.abs())
    if w is not None:
        terms = d_out.double()[:, None, :] * rows
        assert got[2].dtype == wtype and got[2].shape == ix.shape
        close(got[2].reshape(n, k), terms.sum(2), width * U * terms.abs().sum(2))


@gpu
def test_gradients_only_of_what_is_asked(cuda):
    g = R.group_rows(integers(40, 5, 0).reshape(20, 2), 4)
    y, w = normal((40, 6), torch.float32, 1), torch.rand(20, 2, device="cuda")
    d = normal((20, 6), torch.float32, 2)
    a, b = y.clone().requires_grad_(), w.clone().requires_grad_()
    dy, dw = torch.autograd.grad(R.groups_to_rows(a, g, b), (a, b), d)
    assert torch.equal(torch.autograd.grad(R.groups_to_rows(a, g, w), a, d)[0], dy)
    assert torch.equal(torch.autograd.grad(R.groups_to_rows(y, g, b), b, d)[0], dw)
    assert not R.groups_to_rows(y, g, w).requires_grad
    with torch.no_grad():
        assert not R.groups_to_rows(a, g, b).requires_grad


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("width", [1, 2, 12, 20, 33, 59, 64, 333, 1032, 2049, 4097, 9001])
def test_rows_are_kept_for_the_weights_gradient_alone(cuda, dtype, width):
    """y may be overwritten or let go after the forward pass unless the weights' gradient reads it."""
    g = R.group_rows(integers(60, 5, 0, -1).reshape(30, 2), 4)
    y0, up = normal((60, width), dtype, 1), normal((30, width), dtype, 2)
    w = torch.rand(30, 2, device="cuda")
    kept = g.slots >= 0
    for weights in (None, w):
        leaf = y0.clone().requires_grad_(True)
        y = leaf * 1
        saved = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t.shape) or t, lambda t: t):
            out = R.groups_to_rows(y, g, weights)
        assert y.shape not in saved
        y.detach().fill_(float("nan"))
        y.mul_(2)                                            # would be refused if the backward pass needed y
        exact = torch.zeros(60, width, dtype=torch.float64, device="cuda")
        terms = (w.double() if weights is not None else torch.ones_like(w).double())[:, :, None] * up.double()[:, None]
        exact[g.slots[kept].long()] = terms[kept]
        close(torch.autograd.grad(out, leaf, up)[0], exact, U * exact.abs())
    y, wl = y0.clone(), w.clone().requires_grad_(True)
    out = R.groups_to_rows(y, g, wl)
    y.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, wl, up)


@gpu
def test_strided_moves(cuda):
    g = R.group_rows(integers(60, 4, 0).reshape(30, 2), 4)
    big, bigy = normal((30, 50), torch.float32, 1), normal((60, 100), torch.float32, 2)
    w = torch.rand(2, 30, device="cuda").t()                 # weights in the other order
    for x in (big[:, 4:24], big[:, 1:22], big[:, ::2], big[:1].expand(30, 50)):
        assert torch.equal(R.rows_to_groups(x, g), R.rows_to_groups(x.contiguous(), g))
    for y in (bigy[:, 4:24], bigy[:, 1:22], bigy[:, ::3]):
        assert torch.equal(R.groups_to_rows(y, g, w), R.groups_to_rows(y.contiguous(), g, w.contiguous()))
        a, b, c, d = y.clone().requires_grad_(), w.clone().requires_grad_(), y.detach().requires_grad_(), w.detach().requires_grad_()
        for upstream in (torch.ones(30, 1, device="cuda").expand(30, y.shape[1]), big[:, 1:1 + y.shape[1]]):
            if upstream.shape[1] != y.shape[1]:
                continue
            one = torch.autograd.grad(R.groups_to_rows(a, g, b), (a, b), upstream.contiguous())
            two = torch.autograd.grad(R.groups_to_rows(c, g, d), (c, d), upstream)
            assert torch.equal(one[0], two[0])
            # a row that can be read 16 bytes at a time adds its columns to the dot product in
            # another order than one that cannot, so the two are not bit-equal: each is within
            # (width) u sum|term| of the exact value
            terms = upstream.double()[:, None, :] * torch.where(
                (g.slots >= 0)[:, :, None], y.double()[g.slots.long().clamp(min=0)], 0.0)
            for dw in (one[1], two[1]):
                close(dw, terms.sum(2), y.shape[1] * U * terms.abs().sum(2))


@gpu
@pytest.mark.parametrize("dtype,width", [(torch.float32, 5), (torch.float32, 40), (torch.float32, 64),
                                         (torch.bfloat16, 3), (torch.bfloat16, 24), (torch.float16, 40),
                                         (torch.float16, 333), (torch.float16, 2051)])
@pytest.mark.parametrize("ahead", [1, 3, 8])
def test_outputs_that_begin_anywhere(cuda, dtype, width, ahead):
    """Through the C entry points, outputs `ahead` elements behind a boundary: the same values,
    and nothing before or behind them is written."""
    L, code = _lib.lib(), {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    st = torch.cuda.current_stream().cuda_stream
    n, k, rows = 300, 2, 37
    guard = 7.0

    def check(call, *expected):
        bufs = [torch.full((e.numel() + ahead + 64,), guard, dtype=dtype, device="cuda") for e in expected]
        assert call(*[b[ahead:].data_ptr() for b in bufs]) == 0
        for b, e in zip(bufs, expected):
            assert torch.equal(b[ahead:ahead + e.numel()].view(e.shape), e)
            assert (b[:ahead] == guard).all() and (b[ahead + e.numel():] == guard).all()

    table, index = normal((rows, width), dtype, 0), integers(n * k, rows + 1, 1, -1)
    p = index.data_ptr()
    check(lambda o: L.cvhrf_table_lookup(_lib.LOOKUP_ARGS.pack(table.data_ptr(), p, o, rows, width, n * k, width, code,
                                                               8, 0.5), st), R.table_lookup(table, index, 0.5))
    grad = torch.randint(-3, 4, (n * k, width), device="cuda").to(dtype)         # exact in any order
    for entries, table_rows in ((n * k, rows), (n * k, 2000)):
        check(lambda o: L.cvhrf_table_gradient(_lib.GRADIENT_ARGS.pack(
            grad.data_ptr(), p, o, 0, 0, 0, width, entries, table_rows, width, code, 8, 0.5), st),
            R.table_gradient(grad, index, table_rows, 0.5)[0])
    many, more = torch.cat([index] * 8), torch.cat([grad] * 8)
    need = L.cvhrf_table_gradient_workspace_bytes(many.numel(), 5000, width)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    check(lambda o: L.cvhrf_table_gradient(_lib.GRADIENT_ARGS.pack(
        more.data_ptr(), many.data_ptr(), o, 0, ws.data_ptr(), need, width, many.numel(), 5000, width, code, 8, 1.0),
        st), R.table_gradient(more, many, 5000)[0])

    g = R.group_rows(index.reshape(n, k), rows)
    x, y, w = normal((n, width), dtype, 2), grad, torch.randint(0, 3, (n, k), device="cuda").float()
    ptrs = (g.order.data_ptr(), g.slots.data_ptr(), g._used())
    check(lambda o: L.cvhrf_rows_to_groups(_lib.MOVES_ARGS.pack(x.data_ptr(), o, *ptrs, 0, n, width, k, width, code, 0),
                                           st), R.rows_to_groups(x, g))
    check(lambda o: L.cvhrf_groups_to_rows(_lib.MOVES_ARGS.pack(y.data_ptr(), o, *ptrs, w.data_ptr(), n, width, k, width,
                                                                code, 0), st), R.groups_to_rows(y, g, w))
    yl, wl = y.clone().requires_grad_(), w.clone().requires_grad_()
    up = torch.randint(-2, 3, (n, width), device="cuda").to(dtype)
    dy, dw = torch.autograd.grad(R.groups_to_rows(yl, g, wl), (yl, wl), up)
    got_w = torch.empty_like(w)
    check(lambda o: L.cvhrf_groups_to_rows_backward(_lib.MOVES_BACKWARD_ARGS.pack(
        up.data_ptr(), y.data_ptr(), *ptrs, w.data_ptr(), o, got_w.data_ptr(), n, width, width, k, width, code, 0), st),
        dy)
    assert torch.equal(got_w, dw)


@gpu
def test_no_second_derivative(cuda):
    g = R.group_rows(integers(12, 4, 0).reshape(6, 2), 4)
    t, x = normal((5, 3), torch.float32, 1).requires_grad_(), normal((6, 3), torch.float32, 2).requires_grad_()
    for out, leaf in ((R.table_lookup(t, integers(7, 5, 3)), t), (R.rows_to_groups(x, g), x)):
        first, = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            first.sum().backward()


@gpu
def test_forward_mode_is_refused(cuda):
    """A dual tensor needs no backward gradient; its tangent must not vanish without an error."""
    from torch.autograd import forward_ad
    g = R.group_rows(integers(12, 4, 0).reshape(6, 2), 4)
    index = integers(7, 5, 3)
    table, x, y, w = (normal(s, torch.float32, 1) for s in ((5, 3), (6, 3), (12, 3), (6, 2)))
    calls = [(lambda t: R.table_lookup(t, index), table), (lambda t: R.rows_to_groups(t, g), x),
             (lambda t: R.groups_to_rows(t, g), y), (lambda t: R.groups_to_rows(t, g, w), y),
             (lambda t: R.groups_to_rows(y, g, t), w)]
    for call, at in calls:
        plain = call(at)
        with forward_ad.dual_level():
            for grads in (torch.enable_grad, torch.no_grad):
                with grads(), pytest.raises(NotImplementedError, match="forward mode"):
                    call(forward_ad.make_dual(at, torch.ones_like(at)))
            inside = call(at)                                # no dual tensor: as outside
            assert torch.equal(inside, plain) and not inside.requires_grad
        leaf = at.clone().requires_grad_(True)
        with forward_ad.dual_level():
            assert torch.equal(call(leaf), plain) and call(leaf).requires_grad


# ---- gradients against differences -------------------------------------------------------
@gpu
def test_gradients_against_differences(cuda):
    """The operators are linear (bilinear in y and weights), so a central difference with any
    step is exact up to rounding: small integers make every sum and product exact."""
    gen = torch.Generator(device="cuda").manual_seed(0)

    def ints(*shape):
        return torch.randint(-4, 5, shape, generator=gen, device="cuda").float()

    index = integers(12, 6, 1, -1)
    groups = R.group_rows(integers(12, 4, 2, -1).reshape(6, 2), 3)
    up, up_rows, up_places = ints(12, 3), ints(6, 3), ints(12, 3)
    cases = [(lambda t: (R.table_lookup(t, index, 2.0) * up).sum(), ints(5, 3)),
             (lambda x: (R.rows_to_groups(x, groups) * up_places).sum(), ints(6, 3))]
    y, w = ints(12, 3), ints(6, 2)
    cases += [(lambda t: (R.groups_to_rows(t, groups, w) * up_rows).sum(), y),
              (lambda t: (R.groups_to_rows(y, groups, t) * up_rows).sum(), w)]
    for f, at in cases:
        leaf = at.clone().requires_grad_(True)
        f(leaf).backward()
        for i in range(at.numel()):
            step = torch.zeros_like(at)
            step.view(-1)[i] = 1.0
            assert leaf.grad.view(-1)[i] == (f(at + step) - f(at - step)) / 2


# ---- as they are used together ---------------------------------------------------------
@gpu
def test_table_trained_with_sparse_adam(cuda):
    """Lookup, its gradient and the row-sparse optimizer: rows no entry names keep their values."""
    from complex_valued_holographic_radiance_fields_b200 import SparseGaussianAdam
    table = normal((50, 3), torch.float32, 0).requires_grad_(True)
    start = table.detach().clone()
    index = integers(400, 30, 1)
    target = normal((400, 3), torch.float32, 2)
    opt = SparseGaussianAdam([{"params": [table], "lr": 1e-2}], lr=1e-2, eps=1e-15)
    out = R.table_lookup(table, index)
    (out - target).square().sum().backward()
    grad, mask = R.table_gradient(2 * (out.detach() - target), index, 50)
    assert torch.equal(grad, table.grad)
    opt.step(row_mask=mask)
    assert torch.equal(table.detach()[30:], start[30:])
    named = torch.unique(index)
    g = table.grad[named]
    m, v = 0.1 * g, 0.001 * g * g
    assert torch.allclose(table.detach()[named], start[named] - 1e-2 * m / (v.sqrt() + 1e-15), rtol=1e-5, atol=1e-6)


@gpu
def test_round_trip_through_groups(cuda):
    n, k = 999, 3
    g = R.group_rows(integers(n * k, 5, 0).reshape(n, k), 5)
    x = torch.randint(-8, 9, (n, 33), device="cuda").float()
    assert torch.equal(R.groups_to_rows(R.rows_to_groups(x, g), g), 3 * x)


SHARED = {"colours": 64, "pre_act_phase": 300, "pre_act_scales": 1}


def shared_trainer(cuda, **kw):
    from complex_valued_holographic_radiance_fields_b200.train_step import HoloTrainer
    return HoloTrainer(N=5000, W=128, H=96, K=3, device=cuda, seed=5, shared_rows=dict(SHARED), **kw)


@gpu
def test_trainer_with_shared_rows(cuda):
    """The tables' gradients are the per-Gaussian ones summed; the step leaves unnamed rows alone."""
    tr = shared_trainer(cuda)
    tr.codes["colours"] = tr.codes["colours"] % 60            # rows 60 to 63 are named by nobody
    own = {k: v.detach().clone().requires_grad_(True) for k, v in tr.scene_params().items()}
    for k, v in own.items():
        assert torch.equal(v, tr.tables[k][tr.codes[k]] if k in SHARED else tr.params[k])
    from complex_valued_holographic_radiance_fields_b200.train_step import HoloTrainer
    plain = HoloTrainer(N=5000, W=128, H=96, K=3, device=cuda, seed=5)
    plain.params = own
    loss, _ = plain.forward()
    loss.backward()
    before = {k: t.detach().clone() for k, t in tr.tables.items()}
    assert torch.equal(tr.step(), loss.detach())
    for k, t in tr.tables.items():
        total, size, count = gradient_64(own[k].grad, tr.codes[k], t.shape[0], 1.0)
        close(t.grad, total, (count[:, None] + 1) * U * size)
    assert torch.equal(tr.tables["colours"][60:], before["colours"][60:])
    moved = (tr.tables["colours"] != before["colours"]).any(1)
    assert moved[:60].any() and all((t.grad is not None) for _, t in tr._leaves())


@gpu
def test_trainer_with_shared_rows_captured(cuda):
    a, b = shared_trainer(cuda), shared_trainer(cuda)
    b.capture(warmup=2)                                       # three steps
    losses = [float(a.step()) for _ in range(6)]
    assert losses[3:] == [float(b.replay()) for _ in range(3)]
    assert not b.graph_overflowed()
    for (k, x), (_, y) in zip(a._leaves(), b._leaves()):
        assert torch.equal(x, y), k


def test_assigned_codes_and_tables_are_copied_into_place():
    """A captured iteration reads the tensors it was captured with: assigning must fill those."""
    from complex_valued_holographic_radiance_fields_b200.train_step import HoloTrainer
    tr = HoloTrainer(shared_rows={"colours": 4, "pre_act_phase": 7}, N=20, W=16, H=16, K=2, device="cpu")
    at, table = tr.codes["colours"], tr.tables["colours"]
    for new in (torch.arange(20, dtype=torch.int32) % 4, torch.arange(20) % 3, at % 2,
                torch.full((40,), 5, dtype=torch.int32)[::2]):
        tr.codes["colours"] = new
        assert tr.codes["colours"] is at and torch.equal(at, new.int())
    tr.codes["colours"] %= 3
    assert tr.codes["colours"] is at and bool((at == 2).all())
    tr.codes["colours"] = torch.tensor([2 ** 32 + 1, -2 ** 40, 2 ** 31, 2 ** 31 - 1] * 5)   # no row in 64 bits either
    assert at.tolist() == [-1, -1, -1, 2 ** 31 - 1] * 5
    tr.tables["colours"] = torch.ones(4, 3)
    assert tr.tables["colours"] is table and table.requires_grad and table.is_leaf and bool((table == 1).all())
    assert any(p is table for _, p in tr._leaves())
    for bad in (torch.zeros(19, dtype=torch.int32), torch.zeros(21, dtype=torch.int32),
                torch.zeros(20, 1, dtype=torch.int32), torch.zeros((), dtype=torch.int32),
                torch.zeros(20, dtype=torch.int32, device="meta")):
        with pytest.raises(ValueError, match="colours must be"):
            tr.codes["colours"] = bad
    for bad in (torch.zeros(20), torch.zeros(20, dtype=torch.int16), torch.zeros(20, dtype=torch.bool), [0] * 20, 3):
        with pytest.raises(TypeError, match="colours must be"):
            tr.codes["colours"] = bad
    for bad in (torch.ones(5, 3), torch.ones(4, 4), torch.ones(12)):
        with pytest.raises(ValueError, match="colours must be"):
            tr.tables["colours"] = bad
    for held in (tr.codes, tr.tables):
        with pytest.raises(KeyError):
            held["pre_act_scales"] = torch.zeros(20, dtype=torch.int32)
    with pytest.raises(AttributeError):
        tr.codes = {"colours": at}
    assert at.tolist() == [-1, -1, -1, 2 ** 31 - 1] * 5 and bool((table == 1).all())


@gpu
def test_codes_assigned_after_capture(cuda):
    """Replays use codes and tables assigned after the capture, as eager steps do."""
    a, b = shared_trainer(cuda), shared_trainer(cuda)
    b.capture(warmup=2)                                       # three steps
    for _ in range(3):
        a.step()
    for seed in (1, 2):
        for tr in (a, b):
            tr.codes["colours"] = integers(5000, 64, seed, 0, torch.int32 if seed == 1 else torch.int64)
            tr.codes["pre_act_phase"] = integers(5000, 300, seed + 5)
            tr.tables["colours"] = tr.tables["colours"].detach() * 0.5
        fill = [torch.full((5000,), 10 ** 9, dtype=torch.int32, device=cuda) for _ in range(50)]   # memory let go
        assert [float(a.step()) for _ in range(2)] == [float(b.replay()) for _ in range(2)]
        del fill
    for (k, x), (_, y) in zip(a._leaves(), b._leaves()):
        assert torch.equal(x, y), k


@gpu
def test_trainer_with_shared_rows_and_adan(cuda):
    tr = shared_trainer(cuda, optimizer="adan")
    before = tr.tables["pre_act_phase"].detach().clone()
    tr.step()
    assert not torch.equal(tr.tables["pre_act_phase"].detach(), before)


def test_trainer_refusals_of_shared_rows():
    from complex_valued_holographic_radiance_fields_b200.distributed import dp_step
    from complex_valued_holographic_radiance_fields_b200.scene import PinholeCamera
    from complex_valued_holographic_radiance_fields_b200.train_step import HoloTrainer, MultiViewTrainer
    small = dict(N=20, W=16, H=16, K=2, device="cpu")
    for bad in ({"means": 4}, {"pre_act_opacities": 4}, {"colour": 4}, {"colours": 0}, {"colours": 21}):
        with pytest.raises(ValueError):
            HoloTrainer(shared_rows=bad, **small)
    with pytest.raises(ValueError, match="one GPU"):
        MultiViewTrainer(cameras=[PinholeCamera(16, 16)], shared_rows={"colours": 4}, **small)
    tr = HoloTrainer(shared_rows={"colours": 4}, **small)
    for call in (tr.densify, lambda: tr.capture(exchange=lambda t, m: m), lambda: dp_step(tr)):
        with pytest.raises(ValueError, match="shared_rows"):
            call()


def test_checkpoint_of_shared_rows_is_refused_in_words(tmp_path):
    from complex_valued_holographic_radiance_fields_b200 import scene as SC
    from complex_valued_holographic_radiance_fields_b200.train_step import HoloTrainer
    tr = HoloTrainer(shared_rows={"colours": 4}, N=20, W=16, H=16, K=2, device="cpu")
    with pytest.raises(KeyError, match="colours.*scene_params"):
        SC.save_gaussians(tr.params, tmp_path / "g.pth")
    assert not (tmp_path / "g.pth").exists()


@gpu
def test_shared_rows_saved_and_assigned_to_another_trainer(cuda, tmp_path):
    from complex_valued_holographic_radiance_fields_b200 import scene as SC
    a, b = shared_trainer(cuda), shared_trainer(cuda)
    for _ in range(2):
        a.step()
    SC.save_gaussians(a.scene_params(), tmp_path / "g.pth")
    whole = SC.load_gaussians(tmp_path / "g.pth", device=cuda)
    torch.save({"tables": dict(a.tables), "codes": dict(a.codes)}, tmp_path / "shared.pth")
    shared = torch.load(tmp_path / "shared.pth", map_location=cuda)
    for k in SHARED:
        b.codes[k], b.tables[k] = shared["codes"][k], shared["tables"][k]
    with torch.no_grad():
        for k, p in b.params.items():
            p.copy_(whole[k])
    for k, v in b.scene_params().items():
        assert torch.equal(v, a.scene_params()[k]) and torch.equal(v, whole[k])
    assert torch.equal(a.forward()[0], b.forward()[0])


def test_no_exchange_takes_shared_rows():
    """Every exchange between GPUs steps the Gaussians' own parameters only: the tables would stay
    behind without an error."""
    from complex_valued_holographic_radiance_fields_b200 import distributed as D
    from complex_valued_holographic_radiance_fields_b200.train_step import HoloTrainer
    tr = HoloTrainer(shared_rows={"colours": 4}, N=20, W=16, H=16, K=2, device="cpu")
    for call in (lambda: D.dp_step(tr), lambda: D.exchange_and_step(tr, torch.arange(3)),
                 lambda: D.graph_exchange()(tr, torch.zeros(20, dtype=torch.uint8))):
        with pytest.raises(ValueError, match="shared_rows"):
            call()


# ---- streams, graphs, devices ------------------------------------------------------------
@gpu
def test_captured_and_replayed(cuda):
    """A whole step in a CUDA graph, replayed on new contents of its inputs, with an eager step between."""
    def make(seed):
        return dict(index=integers(5000, 301, seed, -1), x=normal((2500, 20), torch.float32, seed),
                    table=normal((300, 20), torch.float32, seed + 1), up=normal((5000, 20), torch.float32, seed + 2),
                    w=torch.rand(2500, 2, device="cuda"))

    def step(s):
        t = s["table"].detach().requires_grad_(True)
        out = R.table_lookup(t, s["index"], 0.5)
        dt, = torch.autograd.grad(out, t, s["up"])
        g = R.group_rows(s["index"].reshape(2500, 2), 300)
        x, w = s["x"].detach().requires_grad_(True), s["w"].detach().requires_grad_(True)
        xs = R.rows_to_groups(x, g)
        back = R.groups_to_rows(xs, g, w)
        dx, dw = torch.autograd.grad(back, (x, w), s["up"][:2500])
        return out, dt, g.order, g.slots, g.offsets, xs, back, dx, dw

    static = make(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for seed in (10, 20):
        new = make(seed)
        expected = [t.clone() for t in step(new)]
        for name, t in new.items():
            static[name].copy_(t)
        graph.replay()
        for a, b in zip(outs, expected):
            assert torch.equal(a, b)


@gpu
def test_two_streams_at_once(cuda):
    index = [integers(200000, 5000, s, -1) for s in (1, 2)]
    grad = [normal((200000, 12), torch.float32, s) for s in (3, 4)]
    alone = [R.table_gradient(g, i, 5000)[0].clone() for g, i in zip(grad, index)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(R.table_gradient(grad[k], index[k], 5000)[0])
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(t, alone[k]) for t in got[k])


@gpu
def test_another_device_than_the_current_one(cuda):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    table = normal((10, 4), torch.float32, 0, "cuda:1")
    index = torch.tensor([3, 3, 9], device="cuda:1")
    assert torch.cuda.current_device() == 0
    assert torch.equal(R.table_lookup(table, index), table[index])
    with pytest.raises(ValueError):
        R.table_lookup(table, index.to("cuda:0"))


# ---- refusals -----------------------------------------------------------------------------
def test_refusals_need_no_gpu():
    cpu = torch.zeros(3, 4)
    index = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        R.table_lookup(cpu, index)
    with pytest.raises(ValueError, match="CUDA"):
        R.table_gradient(torch.zeros(2, 4), index, 3)
    with pytest.raises(ValueError, match="CUDA"):
        R.group_rows(index, 3)
    with pytest.raises(TypeError, match="float32"):
        R.table_lookup(cpu.double(), index)
    with pytest.raises(TypeError, match="number"):
        R.table_lookup(cpu, index, torch.ones(()))
    for bad in (float("nan"), float("inf"), -1e39):
        with pytest.raises(ValueError, match="finite"):
            R.table_lookup(cpu, index, bad)
    with pytest.raises(ValueError, match="shape"):
        R.table_gradient(torch.zeros(3, 4), index, 3)
    with pytest.raises(ValueError, match="num_rows"):
        R.table_gradient(torch.zeros(2, 4), index, -1)


def test_c_abi_refusals_need_no_gpu():
    """Bad arguments come back as a status before anything is launched."""
    L = _lib.lib()
    p = 256   # never read: every call is refused
    for f in (L.cvhrf_table_lookup, L.cvhrf_table_gradient, L.cvhrf_group_rows, L.cvhrf_rows_to_groups,
              L.cvhrf_groups_to_rows, L.cvhrf_groups_to_rows_backward):
        assert f(None, None) == 1

    def lookup(table=p, index=p, out=p, rows=4, stride=4, n=2, width=4, dtype=0, nbytes=4):
        return L.cvhrf_table_lookup(_lib.LOOKUP_ARGS.pack(table, index, out, rows, stride, n, width, dtype, nbytes, 1.0),
                                    None)

    for bad in (dict(table=0), dict(rows=-1), dict(rows=2 ** 31), dict(width=0), dict(width=2 ** 20 + 1),
                dict(stride=-1), dict(dtype=3), dict(index=0), dict(nbytes=2), dict(n=-1), dict(out=0)):
        assert lookup(**bad) == 1, bad
    assert lookup(n=2 ** 30) == 4
    assert lookup(n=0) == 0

    need = L.cvhrf_table_gradient_workspace_bytes(10000, 10, 8)
    assert need > 0 and L.cvhrf_table_gradient_workspace_bytes(100000, 10 ** 5, 80) > 100000
    assert L.cvhrf_table_gradient_workspace_bytes(-1, 10, 8) == 0
    assert L.cvhrf_table_gradient_workspace_bytes(100, 10, 8) == 0     # a few entries need none

    def gradient(grad=p, index=p, out=p, ws=p, need=need, stride=8, n=10000, rows=10, width=8, dtype=0, nbytes=8):
        return L.cvhrf_table_gradient(_lib.GRADIENT_ARGS.pack(grad, index, out, 0, ws, need, stride, n, rows, width,
                                                              dtype, nbytes, 1.0), None)

    for bad in (dict(grad=0), dict(stride=-1), dict(dtype=-1), dict(width=0), dict(index=0), dict(nbytes=1),
                dict(n=-1), dict(out=0), dict(rows=-1), dict(ws=264)):
        assert gradient(**bad) == 1, bad
    assert gradient(ws=0) == 2 and gradient(need=need - 1) == 2
    assert gradient(n=2 ** 30) == 4

    need = L.cvhrf_group_rows_workspace_bytes(10000, 5)
    assert need > 0 and L.cvhrf_group_rows_workspace_bytes(100, 5) == 0

    def group(index=p, order=p, slots=p, offsets=p, ws=p, need=need, n=10000, groups=5, nbytes=4):
        return L.cvhrf_group_rows(_lib.GROUP_ARGS.pack(index, order, slots, offsets, ws, need, n, groups, nbytes), None)

    for bad in (dict(index=0), dict(nbytes=3), dict(n=-1), dict(groups=0), dict(order=0), dict(slots=0),
                dict(offsets=0), dict(ws=264)):
        assert group(**bad) == 1, bad
    assert group(ws=0) == 2 and group(need=need - 1) == 2 and group(n=2 ** 30) == 4

    def moves(f, a=p, to=p, order=p, slots=p, used=p, w=0, n=5, stride=4, k=1, width=4, dtype=0, w_dtype=0):
        return f(_lib.MOVES_ARGS.pack(a, to, order, slots, used, w, n, stride, k, width, dtype, w_dtype), None)

    for f in (L.cvhrf_rows_to_groups, L.cvhrf_groups_to_rows):
        for bad in (dict(a=0), dict(to=0), dict(slots=0), dict(n=-1), dict(stride=-1), dict(k=0), dict(width=0),
                    dict(dtype=5)):
            assert moves(f, **bad) == 1, bad
        assert moves(f, n=2 ** 29, k=2) == 4
    assert moves(L.cvhrf_rows_to_groups, used=0) == 1 and moves(L.cvhrf_rows_to_groups, order=0) == 1
    assert moves(L.cvhrf_groups_to_rows, w=p, dtype=1, w_dtype=2) == 1      # weights of another 16-bit type

    def backward(grad=p, y=p, order=p, slots=p, used=p, w=p, dy=p, dw=p, dtype=0, w_dtype=0):
        return L.cvhrf_groups_to_rows_backward(_lib.MOVES_BACKWARD_ARGS.pack(
            grad, y, order, slots, used, w, dy, dw, 5, 4, 4, 1, 4, dtype, w_dtype), None)

    for bad in (dict(grad=0), dict(y=0), dict(order=0), dict(slots=0), dict(used=0), dict(w=0), dict(dtype=2, w_dtype=1)):
        assert backward(**bad) == 1, bad
    assert backward(dy=0, dw=0) == 0                                        # nothing asked for


def test_argument_structs_match_the_header():
    """The packed layouts have the sizes a C compiler gives the structs."""
    sizes = {}
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "cvhrf.h")).read()
    for body, name in re.findall(r"typedef struct \{([^{}]*)\} (cvhrf_\w+_args);", src):
        fields = []
        for line in body.strip().splitlines():
            kind, names = re.match(r"\s*((?:const )?(?:long long|\w+)\s?\*?)\s*(.*);", line).groups()
            c = (ctypes.c_void_p if "*" in kind else
                 {"long long": ctypes.c_longlong, "int": ctypes.c_int, "float": ctypes.c_float,
                  "size_t": ctypes.c_size_t}[kind.strip()])
            fields += [(f.strip(), c) for f in names.split(",")]
        sizes[name] = ctypes.sizeof(type(name, (ctypes.Structure,), {"_fields_": fields}))
    assert sizes == {"cvhrf_lookup_args": _lib.LOOKUP_ARGS.size, "cvhrf_gradient_args": _lib.GRADIENT_ARGS.size,
                     "cvhrf_group_args": _lib.GROUP_ARGS.size, "cvhrf_moves_args": _lib.MOVES_ARGS.size,
                     "cvhrf_moves_backward_args": _lib.MOVES_BACKWARD_ARGS.size}


@gpu
def test_refusals_on_the_gpu(cuda):
    table, index = torch.zeros(3, 4, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    for bad in (index.cpu(), ):
        with pytest.raises(ValueError, match="index must be on"):
            R.table_lookup(table, bad)
    for bad in (index.to(torch.int16), index.float(), index.bool()):
        with pytest.raises(TypeError, match="int32 or int64"):
            R.table_lookup(table, bad)
        with pytest.raises(TypeError, match="int32 or int64"):
            R.group_rows(bad, 3)
    with pytest.raises(ValueError, match="width"):
        R.table_lookup(table[0], index)
    with pytest.raises(ValueError, match="width"):
        R.table_lookup(table[:, :0], index)
    with pytest.raises(ValueError, match="num_groups"):
        R.group_rows(index, 0)
    with pytest.raises(ValueError, match="k >= 1"):
        R.group_rows(index.reshape(1, 1, 2), 3)
    g = R.group_rows(index, 3)
    with pytest.raises(ValueError, match="2 rows"):
        R.rows_to_groups(table, g)
    with pytest.raises(ValueError, match="2 rows"):
        R.groups_to_rows(table, g)
    with pytest.raises(ValueError, match="weights must be"):
        R.groups_to_rows(table[:2], g, torch.ones(2, 1, device="cuda"))
    with pytest.raises(TypeError, match="weights must be"):
        R.groups_to_rows(table[:2], g, torch.ones(2, device="cuda", dtype=torch.float16))



def test_chained_kernels_read_their_inputs_plainly():
    """A kernel launched with launch_after is on the GPU while the one before it still writes, so
    what that one writes must not be declared constant for the kernel's life (const __restrict__:
    read-only loads); the caller's own inputs may be."""
    csrc = os.path.join(os.path.dirname(os.path.abspath(_lib.__file__)), "csrc")
    chained = 0
    for name in sorted(os.listdir(csrc)):
        src = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, name)).read())
        for kernel in set(re.findall(r"\blaunch_after\((\w+_kernel)", src)):
            params, = re.findall(r"__global__[^;{]*?\b" + kernel + r"\(([^{]*?)\)\s*\{", src)
            chained += 1
            constant = set(re.findall(r"\bconst\b[^,]*\*\s*__restrict__\s*(\w+)", params))
            assert constant <= {"grad"}, (name, kernel, constant)
    assert chained >= 7


def test_c_abi_refuses_rows_that_are_too_wide():
    """Columns are counted in int on the GPU: every entry point refuses more than 2^20 on the host."""
    L = _lib.lib()
    p = 256   # never read
    for width in (2 ** 20 + 1, 2 ** 31 - 1):
        for f in (L.cvhrf_rows_to_groups, L.cvhrf_groups_to_rows):
            assert f(_lib.MOVES_ARGS.pack(p, p, p, p, p, 0, 5, width, 1, width, 0, 0), None) == 1
        assert L.cvhrf_groups_to_rows_backward(_lib.MOVES_BACKWARD_ARGS.pack(
            p, p, p, p, p, p, p, p, 5, width, width, 1, width, 0, 0), None) == 1
        assert L.cvhrf_table_lookup(_lib.LOOKUP_ARGS.pack(p, p, p, 4, width, 2, width, 0, 4, 1.0), None) == 1
        assert L.cvhrf_table_gradient(_lib.GRADIENT_ARGS.pack(p, p, p, 0, 0, 0, width, 9, 4, width, 0, 4, 1.0), None) == 1
        assert L.cvhrf_table_gradient_workspace_bytes(9, 4, width) == 0
