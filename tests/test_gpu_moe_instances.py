"""Every kernel instance that the row calls of a mixture-of-experts layer and the 8-bit
checkpoints can select: lanes and waves a token, sums held for 1, 2, 4, 8 or 16 choices,
loads that stay in the caches or do not (tensors past 128 MB), whole and partial units,
each row type and format.  Also bias gradients of segments of very different lengths, one
row named by several slots of a sum, the lowest and largest values of a type.
Compared with the formulas in 64 bits (elementary torch operations on the device), with
moe_ref.py's bounds."""
import math

import numpy as np
import pytest
import torch

import cme213_amd as M
import moe_ref as R
from gpu_util import host, note
from tol import BWD_ATOL, BWD_RTOL, COL_RTOL, FWD_ATOL, FWD_RTOL, assert_exact

pytestmark = pytest.mark.gpu

SIZE = {"f32": 4, "f16": 2, "bf16": 2}
FORMATS = {"int8": M.CKPT8_INT8, "e4m3": M.CKPT8_E4M3}
KS = [1, 2, 3, 4, 6, 8, 9, 16]


def _half(t, ref):
    """moe_ref.half_step of a device tensor, with what the fp32 result's own error adds to it."""
    fi = torch.finfo(R.TYPES[t])
    return (ref.abs() * fi.eps / 2 + float(fi.smallest_normal) * fi.eps / 2) * (1 + 2.0 ** -10)


def _near(name, got, want, bound):
    over = ~((got.double() - want).abs() <= bound)
    if over.any():
        i = tuple(over.nonzero()[0].tolist())
        raise AssertionError(f"{name}: {int(over.sum())} of {over.numel()} off; at {i} got "
                             f"{float(got[i])!r}, want {float(want[i])!r}, bound "
                             f"{float(torch.as_tensor(bound).expand(over.shape)[i]):.3e}")


def _cols(chunks, ragged, t):
    """A width of `chunks` 16-byte pieces, the last one cut where ragged."""
    return chunks * 16 // SIZE[t] - (1 if ragged else 0)


def _check_rows(dev, n, k, c, t):
    r = np.random.default_rng(n * 31 + k * 7 + c)
    ids = r.integers(0, 5, n * k).astype(np.int32)
    ids[r.random(n * k) < 0.1] = -1
    _, order, pos = R.sort(ids, 5)
    rows = max(1, len(order) - 1)  # one row too few: its slot is dropped as well
    gen = torch.Generator(device="cuda").manual_seed(n + k + c)
    dtype = R.TYPES[t]
    P = torch.from_numpy(pos).to(dev)

    def rand(*shape, type=dtype):
        return torch.randn(*shape, device=dev, generator=gen).to(type)
    on = ((P >= 0) & (P < rows)).view(n, k)
    at = torch.where(on, P.view(n, k), 0).long()
    moved = torch.zeros(rows + 1, dtype=torch.bool, device=dev)
    moved[at[on]] = True

    x = rand(n, c)
    xs = torch.full((rows + 1, c), 77.0, dtype=dtype, device=dev)
    M.moe_dispatch_forward(x, P, xs, n, k, rows, c)
    want = torch.full_like(xs, 77.0)
    want[at[on]] = x.repeat_interleave(k, 0).view(n, k, c)[on]
    assert torch.equal(xs, want), "dispatch"

    y, w = rand(rows + 1, c), rand(n, k, type=torch.float32)
    for name, weights in (("dispatch gradient", None), ("combine", w)):
        total = torch.zeros(n, c, dtype=torch.float64, device=dev)
        size = torch.zeros_like(total)
        for j in range(k):
            term = torch.where(on[:, j, None], y[at[:, j]].double(), 0.0)
            term *= 1.0 if weights is None else weights[:, j, None].double()
            total += term
            size += term.abs()
        out = torch.full((n + 1, c), 77.0, dtype=dtype, device=dev)
        if weights is None:
            M.moe_dispatch_backward(y, P, out, n, k, rows, c)
        else:
            M.moe_combine_forward(y, P, weights, out, n, k, rows, c)
        # k products and k sums in fp32, then the row type's rounding
        _near(name, out[:n], total, 2 * k * R.U * size + _half(t, total))
        assert (out[n] == 77).all(), name

    g = rand(n, c)
    rdy = torch.full((rows + 1, c), 77.0, dtype=torch.float64, device=dev)
    rdw = torch.zeros(n, k, dtype=torch.float64, device=dev)
    size = torch.zeros_like(rdw)
    for j in range(k):
        o, a = on[:, j], at[:, j]
        rdy[a[o]] = g[o].double() * w[o, j, None].double()
        prod = g.double() * y[a].double()
        rdw[:, j] = torch.where(o, prod.sum(1), 0.0)
        size[:, j] = torch.where(o, prod.abs().sum(1), 0.0)
    # a lane adds at most c / 64 + 8 products, then the lanes' and waves' sums: as in
    # test_gpu_moe.py
    bound = (c / 64 + 24) * R.U * size
    dy = torch.full((rows + 1, c), 77.0, dtype=dtype, device=dev)
    dw = torch.full((n * k + 1,), 77.0, device=dev)
    M.moe_combine_backward(g, y, P, w, dy, dw, n, k, rows, c)
    _near("dy", dy, rdy, torch.where(moved[:, None], _half(t, rdy) + R.U * rdy.abs(), 0.0))
    _near("dweights", dw[:n * k].view(n, k), rdw, bound)
    assert dw[n * k] == 77
    kept = y.clone()
    dw = torch.full((n * k + 1,), 77.0, device=dev)
    M.moe_combine_backward(g, y, P, w, y, dw, n, k, rows, c)
    assert torch.equal(y[moved], dy[moved]), "dy in place"
    assert torch.equal(y[~moved], kept[~moved]), "y's other rows"
    _near("dweights in place", dw[:n * k].view(n, k), rdw, bound)
    assert dw[n * k] == 77


# Lanes of a token for short rows; one wave; four waves for long rows, or for few tokens; 16
# waves for long rows of few tokens (up to 8 choices); and widths whose moved-back last
# piece falls to another wave than its neighbour (129, 257, 321).
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("k", KS)
@pytest.mark.parametrize("n,chunks,ragged", [
    (37, 13, True), (37, 29, True), (37, 50, True), (515, 70, False), (515, 129, True),
    (37, 120, True), (37, 129, True), (515, 258, True), (515, 257, True), (21, 300, True),
    (21, 300, False), (21, 321, True)])
def test_rows_of_every_shape(dev, n, chunks, ragged, k, t):
    c = _cols(chunks, ragged, t)
    note(f"rows {n} tokens k={k} c={c} {t}")
    _check_rows(dev, n, k, c, t)


@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("k", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("chunks,ragged", [(11, True), (27, True), (60, False), (127, True),
                                           (250, True), (301, True)])
def test_rows_past_the_cache(dev, chunks, ragged, k, t):
    """Rows of more than 128 MB, which are read without being kept in the caches (dropped slots
    left out of the count; combine's gradient reads and writes more than the sums do)."""
    c = _cols(chunks, ragged, t)
    n = math.ceil(160e6 / (c * SIZE[t]) / (1 + k))
    note(f"rows past the cache {n} tokens k={k} c={c} {t}")
    _check_rows(dev, n, k, c, t)


def _gelu64(u):
    z = math.sqrt(2 / math.pi) * (u + 0.044715 * u ** 3)
    s = 1 / (1 + torch.exp(-2 * z))
    return u * s, s + 2 * u * s * (1 - s) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * u * u)


def _check_checkpoint(dev, rows, cols, offsets, t, fmt, act):
    groups, dtype = len(offsets) - 1, R.TYPES[t]
    gen = torch.Generator(device="cuda").manual_seed(rows + cols)

    def blank(type, c=cols):
        return torch.full((rows, c), 77, dtype=type, device=dev)
    x = (torch.randn(rows, cols, device=dev, generator=gen) * 2).to(dtype)
    g = torch.randn(rows, cols, device=dev, generator=gen).to(dtype)
    b = 0.3 * torch.randn(groups, cols, device=dev, generator=gen)
    off = torch.tensor(offsets, dtype=torch.int32, device=dev)
    row = torch.arange(rows, device=dev)
    of = torch.bucketize(row, off[1:].contiguous(), right=True)
    used = (row >= off[0]) & (of < groups)
    of = of.clamp(max=groups - 1)
    nb = -(-cols // 32)

    q, s = blank(torch.uint8), blank(torch.uint8, nb)
    M.float_to_ckpt8(x, q, s, rows, cols, FORMATS[fmt])
    for part in (slice(0, 40), slice(rows // 2, rows // 2 + 40), slice(rows - 40, rows)):
        rq, rs = R.to_ckpt8(host(x[part].double()), fmt)
        assert_exact("scales", host(s[part]), rs)
        assert_exact("codes", host(q[part]), rq)
    kept = blank(torch.float32)
    M.ckpt8_to_float(q, s, kept, rows, cols, FORMATS[fmt])
    e = s.double() - (133 if fmt == "int8" else 135)
    code = q.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).double()
    code *= torch.exp2(e).repeat_interleave(32, 1)[:, :cols]
    assert torch.equal(kept.double(), code), "values"
    back = blank(dtype)
    M.ckpt8_to_float(q, s, back, rows, cols, FORMATS[fmt])
    assert torch.equal(back, code.to(dtype)), "values in the row type"

    out, q2, s2 = blank(dtype), blank(torch.uint8), blank(torch.uint8, nb)
    M.bias_gelu_forward_ckpt8(x, b, off, out, q2, s2, rows, cols, groups, FORMATS[fmt])
    assert torch.equal(q2[used], q[used]) and torch.equal(s2[used], s[used]), "checkpoint"
    assert (q2[~used] == 77).all() and (s2[~used] == 77).all() and (out[~used] == 77).all()
    # the bounds of test_gpu_ckpt8.py: u rounded, the fp32 GELU's tolerance, the row type's
    u = x.double() + b[of].double()
    y = _gelu64(u)[0]
    slack = 1.2 * R.U * u.abs() + FWD_ATOL + FWD_RTOL * y.abs()
    _near("out", out[used], y[used], (slack + _half(t, y) * 1.01)[used])
    del out, y, slack

    gin, a = blank(dtype), blank(dtype) if act else None
    db = torch.ones(groups, cols, device=dev)
    M.gelu_backward_with_bias_backward_ckpt8(q, s, b, off, g, gin, a, db, rows, cols, groups,
                                             FORMATS[fmt])
    u = code + b[of].double()
    y, d = _gelu64(u)
    ref = g.double() * d
    gslack = (1.6 * R.U * u.abs() + BWD_ATOL + BWD_RTOL * d.abs()) * g.double().abs()
    _near("grad_in", gin[used], ref[used], (gslack + _half(t, ref) * 1.01)[used])
    assert (gin[~used] == 77).all()
    if act:
        slack = 1.2 * R.U * u.abs() + FWD_ATOL + FWD_RTOL * y.abs()
        _near("act", a[used], y[used], (slack + _half(t, y) * 1.01)[used])
        assert (a[~used] == 77).all()

    def sums(v):
        r = torch.zeros(groups, cols, dtype=torch.float64, device=dev)
        return r.index_add_(0, of[used], v[used])
    _near("dbias", db, 1 + sums(ref),
          COL_RTOL * (sums(ref * ref).sqrt() + 1) + 2 * sums(gslack * gslack).sqrt())


@pytest.mark.parametrize("act", [False, True])
@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("cols", [1801, 1800, 1024])
def test_checkpoints_past_the_cache(dev, cols, t, fmt, act):
    """Tensors of more than 128 MB in each call (the checkpoint alone moves the least): units
    that are partial, whole or empty, and all whole; a short last segment, rows behind it."""
    rows = math.ceil(140e6 / cols / (SIZE[t] + 1))
    note(f"checkpoint past the cache {rows}x{cols} {t} {fmt} act={act}")
    _check_checkpoint(dev, rows, cols, [0, rows - 90, rows - 40], t, fmt, act)


@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("rows,cols,groups,longest", [(16384, 1600, 128, 37), (8192, 264, 64, 0),
                                                      (5000, 2049, 300, 299)])
def test_bias_gradients_of_uneven_segments(dev, rows, cols, groups, longest, t):
    """One segment holds more than nine tenths of the rows, the others a few rows or none."""
    note(f"uneven segments {rows}x{cols} groups={groups} {t}")
    r = np.random.default_rng(groups)
    length = r.multinomial(rows // 15, np.full(groups, 1 / groups))
    length[longest] += rows - length.sum()
    assert length[longest] > 0.9 * rows
    _check_checkpoint(dev, rows, cols, [0] + np.cumsum(length).tolist(), t, "int8", False)


@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("c", [3, 40, 1030])
def test_sums_take_one_row_twice(dev, c, t):
    """Slots that name the same row, of one token and of several: each adds it."""
    n, k, rows = 5, 3, 4
    note(f"one row twice c={c} {t}")
    r = np.random.default_rng(c)
    pos = np.array([2, 2, 2, 0, 1, 0, 3, 3, -1, 4, 1, 1, 0, 2, 3], np.int32)
    y = torch.from_numpy(r.standard_normal((rows, c))).to(R.TYPES[t])
    w = r.standard_normal((n, k)).astype(np.float32)
    P, Y, W = torch.from_numpy(pos).to(dev), y.to(dev), torch.from_numpy(w).to(dev)
    for name, weights in (("dispatch gradient", None), ("combine", w.astype(np.float64))):
        out = torch.full((n, c), 77.0, dtype=R.TYPES[t], device=dev)
        if weights is None:
            M.moe_dispatch_backward(Y, P, out, n, k, rows, c)
        else:
            M.moe_combine_forward(Y, P, W, out, n, k, rows, c)
        ref, size = R.gather_sum(y.double().numpy(), pos, weights, n, k, rows)
        R.near(name, host(out.double()), ref,
               2 * k * R.U * size + R.half_step(t, ref) * (1 + 2.0 ** -10))


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("t", list(R.TYPES))
def test_lowest_and_largest_values_of_a_type(dev, t, fmt):
    """Elements of the type's lowest value, as masks have them: gelu and its slope are zero
    there (to 1e-30), those of its largest value 1 times them, and nothing is NaN."""
    rows, cols = 6, 64
    note(f"lowest values {t} {fmt}")
    fi = torch.finfo(R.TYPES[t])
    x = torch.zeros(rows, cols, dtype=R.TYPES[t], device=dev)
    x[1:4, 5], x[2, 40:], x[4, 7] = fi.min, fi.min, fi.max
    low, high = x == fi.min, x == fi.max
    b = torch.linspace(-1, 1, cols, device=dev)[None].contiguous()
    q = torch.empty(rows, cols, dtype=torch.uint8, device=dev)
    s = torch.empty(rows, 2, dtype=torch.uint8, device=dev)
    out, gin, act = (torch.full_like(x, 77.0) for _ in range(3))
    M.bias_gelu_forward_ckpt8(x, b, None, out, q, s, rows, cols, 1, FORMATS[fmt])
    db = torch.zeros(1, cols, device=dev)
    M.gelu_backward_with_bias_backward_ckpt8(q, s, b, None, torch.ones_like(x), gin, act, db, rows,
                                             cols, 1, FORMATS[fmt])
    for name, v in (("out", out), ("grad_in", gin), ("act", act)):
        assert (v[low].abs() <= 1e-30).all(), name
        assert not v.isnan().any(), name
    assert (gin[high] == 1).all() and (out[high] == fi.max).all()
    # the largest value's code is 127 of 128 (int8) or 448 of 512 (e4m3) of the next power
    part = 127 / 128 if fmt == "int8" else 448 / 512
    power = 2.0 ** (16 if t == "f16" else 128)
    assert (act[high].double() == part * power).all()
    # all other elements are zero: their column's slope is gelu'(b), once for each
    zeros = (~(low | high)).sum(0).double()
    d = _gelu64(b[0].double())[1]
    _near("dbias", db[0], zeros * d + high.sum(0),
          rows * (BWD_ATOL + BWD_RTOL * d.abs()) + 8 * R.U * rows)
