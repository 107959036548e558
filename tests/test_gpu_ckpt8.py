"""GPU parity of the 8-bit checkpoints against plain 64-bit implementations
(moe_ref.py): codes and scales exactly, for every rounding border, subnormal, huge,
infinite and NaN blocks; bias + GELU with a checkpoint and its backward pass, over
segments that are empty, short, long or absent, odd widths, one row and one column,
buffers off any alignment, rows outside the segments left as they were."""
import numpy as np
import pytest
import torch

import cme213_amd as M
import moe_ref as R
from gpu_util import dev_t, host, note
from tol import BWD_ATOL, BWD_RTOL, COL_RTOL, FWD_ATOL, FWD_RTOL, assert_exact

pytestmark = pytest.mark.gpu

FORMATS = {"int8": M.CKPT8_INT8, "e4m3": M.CKPT8_E4M3}


def _off(t):
    b = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda:0")
    v = b[1:].view(t.shape)
    v.copy_(t)
    return v


def _dev(t):
    return t.contiguous().to("cuda:0")


def _h64(t):
    return host(t.double())


def _check_roundtrip(x, t, fmt, off=False):
    """x: a torch CPU tensor [rows, cols] of type t."""
    rows, cols = x.shape
    put = _off if off else _dev
    q = put(torch.full((rows, cols), 77, dtype=torch.uint8))
    s = put(torch.full((rows, -(-cols // 32)), 77, dtype=torch.uint8))
    M.float_to_ckpt8(put(x), q, s, rows, cols, FORMATS[fmt])
    rq, rs = R.to_ckpt8(x.double().numpy(), fmt)
    assert_exact("scales", host(s), rs)
    assert_exact("codes", host(q), rq)
    back = put(torch.full((rows, cols), 77.0, dtype=R.TYPES[t]))
    M.ckpt8_to_float(q, s, back, rows, cols, FORMATS[fmt])
    want = torch.from_numpy(R.from_ckpt8(rq, rs, fmt)).to(R.TYPES[t]).double().numpy()
    R.near("values", _h64(back), want, 0)
    return want


@pytest.mark.parametrize("off", [False, True])
@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (2, 8), (5, 31), (4, 32), (7, 33),
                                       (130, 512), (9, 515), (6, 1600), (3, 2049)])
def test_checkpoint(dev, rows, cols, t, fmt, off):
    note(f"checkpoint {rows}x{cols} {t} {fmt} off={off}")
    r = np.random.default_rng(rows + cols)
    x = r.standard_normal((rows, cols)) * np.exp2(r.integers(-12, 10, (rows, 1)))
    x[r.random((rows, cols)) < 0.1] = 0
    _check_roundtrip(torch.from_numpy(x).to(R.TYPES[t]), t, fmt, off)


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_checkpoint_borders(dev, fmt):
    """Every code, every border between two of them and its neighbours on both sides, in
    blocks whose largest value fixes the scale; then the same far up and far down."""
    note(f"checkpoint borders {fmt}")
    vals = R.E4M3[:127] if fmt == "e4m3" else np.arange(0, 128.0)
    mid = (vals[:-1] + vals[1:]) / 2
    v = np.concatenate([vals, mid, np.nextafter(mid.astype(np.float32), np.float32(0)),
                        np.nextafter(mid.astype(np.float32), np.float32(1e9))]).astype(np.float64)
    top = 256.0 if fmt == "e4m3" else 64.0  # a block of [top, 2 top) has the codes' own scale
    v = v[v < 2 * top]
    v = np.concatenate([v, -v])
    v = np.concatenate([v, np.zeros(-len(v) % 31)]).reshape(-1, 31)
    x = np.concatenate([np.full((len(v), 1), top), v], 1)
    for shift in (0, -20, 100, -125, -140):
        _check_roundtrip(torch.from_numpy(np.ldexp(x, shift).astype(np.float32)), "f32", fmt)


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("t", list(R.TYPES))
def test_checkpoint_special_blocks(dev, t, fmt):
    note(f"checkpoint special {t} {fmt}")
    fi = torch.finfo(R.TYPES[t])
    rows = []
    for big in (0.0, -0.0, fi.max, fi.min, float(fi.smallest_normal),
                float(fi.smallest_normal) * fi.eps, np.nan, np.inf, -np.inf, 1.999, 127.75, 448.0,
                511.9):
        row = np.random.default_rng(5).uniform(-1, 1, 96) * (abs(big) if np.isfinite(big) else 1)
        row[40] = big
        rows.append(row)
    x = torch.from_numpy(np.array(rows)).to(R.TYPES[t])
    want = _check_roundtrip(x, t, fmt)
    bad = np.isnan(want)
    assert bad[6:9, 32:64].all() and bad.sum() == 3 * 32  # the block, and no other


# ----- bias + GELU -----------------------------------------------------------------------

# rows, cols, groups, how the rows are shared out
CASES = [(1, 1, 1, None), (1, 40, 1, None), (5, 33, 1, None), (200, 512, 1, None),
         (129, 515, 1, None), (70, 1600, 1, None), (1, 64, 3, "even"), (257, 100, 4, "even"),
         (300, 96, 7, "empty"), (64, 2049, 5, "short"), (1000, 24, 1000, "even"),
         (500, 130, 2, "late"), (90, 48, 3, "none"), (2000, 1030, 9, "short"), (40, 8, 1, "part")]


def _offsets(rows, groups, how, r):
    if how is None:
        return None
    cut = np.sort(r.integers(0, rows + 1, groups - 1))
    if how == "empty":  # equal neighbours, the first and the last group empty
        cut[0], cut[-1] = 0, rows
        cut[2:4] = cut[2]
    first, last = 0, rows
    if how == "short":
        last = rows - rows // 5
    if how == "late":
        first = rows // 4
    if how == "part":
        first, last = rows // 3, rows // 2
    o = np.concatenate([[first], np.clip(np.sort(cut), first, last), [last]]).astype(np.int32)
    return np.zeros(groups + 1, np.int32) if how == "none" else o


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("rows,cols,groups,how", CASES)
def test_bias_gelu_checkpoint(dev, rows, cols, groups, how, t, fmt):
    note(f"gelu checkpoint {rows}x{cols} groups={groups} {how} {t} {fmt}")
    r = np.random.default_rng(rows + cols + groups)
    x = torch.from_numpy(r.standard_normal((rows, cols)) * 2).to(R.TYPES[t])
    g = torch.from_numpy(r.standard_normal((rows, cols))).to(R.TYPES[t])
    b = (0.3 * r.standard_normal((groups, cols))).astype(np.float32)
    offs = _offsets(rows, groups, how, r)
    of = R.groups_of(offs, rows, groups)
    used = of >= 0
    put = _off if cols % 2 else _dev
    X, B = put(x), dev_t(b)
    O = None if offs is None else dev_t(offs)

    def blank(dtype=R.TYPES[t], c=cols):
        return put(torch.full((rows, c), 77, dtype=dtype))
    out, q, s = blank(), blank(torch.uint8), blank(torch.uint8, -(-cols // 32))
    M.bias_gelu_forward_ckpt8(X, B, O, out, q, s, rows, cols, groups, FORMATS[fmt])
    x64, b64 = x.double().numpy(), b.astype(np.float64)[np.maximum(of, 0)]
    rq, rs = R.to_ckpt8(x64, fmt)
    assert_exact("scales", host(s), np.where(used[:, None], rs, 77))
    assert_exact("codes", host(q), np.where(used[:, None], rq, 77))
    y = R.gelu(x64 + b64)[0]
    # u = x + b is rounded (the GELU's slope is at most 1.13), then the fp32 GELU's own
    # tolerance, then the row type's rounding
    slack = 1.2 * R.U * np.abs(x64 + b64) + FWD_ATOL + FWD_RTOL * np.abs(y)
    R.near("out", _h64(out), np.where(used[:, None], y, 77),
           np.where(used[:, None], slack + R.half_step(t, y) * 1.01, 0))
    inplace = put(x)
    q2, s2 = blank(torch.uint8), blank(torch.uint8, -(-cols // 32))
    M.bias_gelu_forward_ckpt8(inplace, B, O, inplace, q2, s2, rows, cols, groups, FORMATS[fmt])
    assert_exact("out in place", _h64(inplace)[used], _h64(out)[used])
    assert_exact("codes in place", host(q2), host(q))

    db0 = r.standard_normal((groups, cols)).astype(np.float32)
    gin, act, db = blank(), blank(), dev_t(db0)
    M.gelu_backward_with_bias_backward_ckpt8(q, s, B, O, put(g), gin, act, db, rows, cols, groups,
                                             FORMATS[fmt])
    u = R.from_ckpt8(rq, rs, fmt) + b64
    y, d = R.gelu(u)
    g64 = g.double().numpy()
    ref = g64 * d
    # gelu' has slope at most 1.6; the rounding of u enters through it
    gslack = (1.6 * R.U * np.abs(u) + BWD_ATOL + BWD_RTOL * np.abs(d)) * np.abs(g64)
    R.near("grad_in", _h64(gin), np.where(used[:, None], ref, 77),
           np.where(used[:, None], gslack + R.half_step(t, ref) * 1.01, 0))
    slack = 1.2 * R.U * np.abs(u) + FWD_ATOL + FWD_RTOL * np.abs(y)
    R.near("act", _h64(act), np.where(used[:, None], y, 77),
           np.where(used[:, None], slack + R.half_step(t, y) * 1.01, 0))
    want, size, floor = db0.astype(np.float64), np.zeros((groups, cols)), np.zeros((groups, cols))
    for i in range(groups):
        want[i] += ref[of == i].sum(0)
        size[i] = np.sqrt((ref[of == i] ** 2).sum(0)) + np.abs(db0[i])
        floor[i] = np.sqrt((gslack[of == i] ** 2).sum(0)) * 2
    R.near("dbias", host(db), want, COL_RTOL * size + floor)
    assert_exact("dbias of empty groups", host(db)[[i for i in range(groups) if not (of == i).any()]],
                 db0[[i for i in range(groups) if not (of == i).any()]])
    # without act, grad_in in place of grad_out, dbias again: the same bits
    again, db2 = put(g), dev_t(db0)
    M.gelu_backward_with_bias_backward_ckpt8(q, s, B, O, again, again, None, db2, rows, cols,
                                             groups, FORMATS[fmt])
    assert_exact("grad_in in place", _h64(again)[used], _h64(gin)[used])
    assert_exact("dbias again", host(db2), host(db))


# Rows that end inside a cache line: several tiles and bands, the last tile wide and of whole
# units, wide with a partial one, narrow; a number of bands that is no multiple of eight; rows
# of one unit and a part.
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("rows,cols,groups,how", [(613, 1000, 3, "short"), (337, 2008, 2, "even"),
                                                  (901, 1799, 5, "late"), (45, 5160, 1, None),
                                                  (33, 9, 2, "even"), (20, 15, 1, None)])
def test_rows_that_end_inside_a_line(dev, rows, cols, groups, how, t):
    test_bias_gelu_checkpoint(dev, rows, cols, groups, how, t, "int8")
    test_checkpoint(dev, rows, cols, t, "e4m3", False)


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_bias_gelu_checkpoint_non_finite(dev, fmt):
    """Infinite and NaN inputs: out as gelu defines it; the block they are in reads as NaN in
    the backward pass, and only that one."""
    rows, cols = 6, 96
    x = np.random.default_rng(1).standard_normal((rows, cols)).astype(np.float32)
    x[1, 40], x[2, 40], x[3, 40], x[4, 0] = np.inf, -np.inf, np.nan, 3e38
    X, B = dev_t(x), torch.zeros(1, cols, device=dev)
    out, gin = torch.empty_like(X), torch.empty_like(X)
    q = torch.empty(rows, cols, dtype=torch.uint8, device=dev)
    s = torch.empty(rows, 3, dtype=torch.uint8, device=dev)
    M.bias_gelu_forward_ckpt8(X, B, None, out, q, s, rows, cols, 1, FORMATS[fmt])
    y = R.gelu(x.astype(np.float64))[0]
    R.near("out", host(out), y, 1e-6 + 1e-5 * np.abs(np.where(np.isfinite(y), y, 0)))
    db = torch.zeros(1, cols, device=dev)
    M.gelu_backward_with_bias_backward_ckpt8(q, s, B, None, torch.ones_like(X), gin, None, db,
                                             rows, cols, 1, FORMATS[fmt])
    nan = np.zeros((rows, cols), bool)
    nan[1:4, 32:64] = True
    assert (np.isnan(host(gin)) == nan).all()
    assert (np.isnan(host(db)[0]) == nan.any(0)).all()


def test_bias_gelu_gradient_against_differences(dev):
    """Where the checkpoint holds the input exactly, the gradient is that of the forward call:
    central differences with step 2^-6 are off by h^2/6 max|gelu'''| (about 8e-5) and by the
    rounding of the outputs, 2^-24 * 8 / h = 3e-5."""
    rows, cols, h = 16, 64, 2.0 ** -6
    x = (np.random.default_rng(2).integers(-127, 128, (rows, cols)) / 32).astype(np.float32)
    x[:, ::32] = 3.5  # the blocks' scale: a step of 1/32
    B = torch.zeros(1, cols, device=dev)
    q = torch.empty(rows, cols, dtype=torch.uint8, device=dev)
    s = torch.empty(rows, 2, dtype=torch.uint8, device=dev)

    def forward(a):
        out = torch.empty(rows, cols, device=dev)
        M.bias_gelu_forward_ckpt8(dev_t(a.astype(np.float32)), B, None, out, q, s, rows, cols)
        return host(out).astype(np.float64)
    num = (forward(x + h) - forward(x - h)) / (2 * h)
    forward(x)
    gin, db = torch.empty(rows, cols, device=dev), torch.zeros(1, cols, device=dev)
    M.gelu_backward_with_bias_backward_ckpt8(q, s, B, None, torch.ones(rows, cols, device=dev),
                                             gin, None, db, rows, cols)
    R.near("gradient", host(gin), num, 2e-4)


def test_long_column_sums(dev):
    """Many rows into one dbias row: the sums keep their precision."""
    rows, cols = 70000, 72
    note(f"long column sums {rows}x{cols}")
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, cols, device=dev, generator=gen).bfloat16()
    g = torch.randn(rows, cols, device=dev, generator=gen).bfloat16()
    q = torch.empty(rows, cols, dtype=torch.uint8, device=dev)
    s = torch.empty(rows, 3, dtype=torch.uint8, device=dev)
    M.float_to_ckpt8(x, q, s, rows, cols)
    B, gin = torch.zeros(1, cols, device=dev), torch.empty_like(x)
    db = torch.zeros(1, cols, device=dev)
    M.gelu_backward_with_bias_backward_ckpt8(q, s, B, None, g, gin, None, db, rows, cols)
    ref = _h64(g) * R.gelu(R.from_ckpt8(host(q), host(s), "int8"))[1]
    size = np.sqrt((ref ** 2).sum(0))
    R.near("dbias", host(db)[0], ref.sum(0), 1e-5 * size)
