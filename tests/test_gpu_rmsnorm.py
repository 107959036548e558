"""GPU parity of the RMS norm calls against plain 64-bit implementations (step_ref.py, where
the bounds are derived): every way a row is held (parts of a wave to a workgroup, or walked),
odd widths, buffers off any alignment, rows of zeros, tiny, huge, infinite and NaN values,
outputs in 8 bits, in place, from a graph, on another stream, past 2^31 elements."""
import numpy as np
import pytest
import torch

import cme213_amd as M
import moe_ref as R
import step_ref as S
from gpu_util import dev_t, host, note
from tol import assert_exact

pytestmark = pytest.mark.gpu

EPS = 1e-5
# rows up to 1024 take more waves each than more rows do; widths on both sides of each step
SHAPES = [(1, 1), (5, 3), (3, 7), (1, 8), (4, 4), (2, 64), (9, 100), (5, 127), (16, 129), (33, 256),
          (7, 257), (3, 300), (17, 512), (2, 516), (17, 768), (1030, 769), (1025, 1026), (1027, 1300),
          (1026, 1600), (1025, 2047), (1026, 2101), (1025, 3002), (1026, 4093), (4, 1600), (3, 2050), (2, 3999), (5, 4096), (3, 5003), (2, 6145),
          (2, 8192), (1, 8200), (3, 12289), (2, 16384), (1, 16387), (1, 40001)]
FORMATS = {"int8": (M.ROW8_INT8, 127.0, torch.int8), "e4m3": (M.ROW8_E4M3, 448.0, torch.float8_e4m3fn)}


def _h64(t):
    return host(t.double())


def _off(t):
    """The same tensor on the GPU, one element off the allocation's alignment."""
    b = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda:0")
    v = b[1:].view(t.shape)
    v.copy_(t)
    return v


def _rows(r, n, c, t, scale=1.0):
    return torch.from_numpy(r.standard_normal((n, c)) * scale).to(R.TYPES[t])


def _inputs(n, c, t, seed, hard=True):
    r = np.random.default_rng(seed)
    a, b = _rows(r, n, c, t), _rows(r, n, c, t, 0.5)
    if hard and n > 1:  # the other rows: zeros, tiny, large but in fp32's range when squared
        for i, f in enumerate((0.0, 2.0 ** -12, 2.0 ** 10)[:n - 1]):
            a[i], b[i] = a[i] * f, b[i] * f
    gamma = (1 + 0.1 * r.standard_normal(c)).astype(np.float32)
    return a, b, gamma


def _check_rows(t, got, want, rel):
    R.near("out", _h64(got), want, rel[:, None] * np.abs(want) * (1 + 2.0 ** -7) +
           R.half_step(t, want) * (1 + 2.0 ** -9))


@pytest.mark.parametrize("resid", [False, True])
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,c", SHAPES)
def test_forward(dev, n, c, t, resid):
    note(f"rmsnorm forward {n}x{c} {t} residual={resid}")
    a, b, gamma = _inputs(n, c, t, n * 7 + c)
    A, B, G = _off(a), _off(b), dev_t(gamma)
    out, total = _off(torch.full_like(a, 77)), _off(torch.full_like(a, 77))
    inv = torch.full((n + 1,), 77.0, device=dev)
    if resid:
        M.residual_rmsnorm_forward(A, B, G, total, out, inv, n, c, EPS)
    else:
        M.rmsnorm_forward(A, G, out, inv, n, c, EPS)
    h, r, y, rel_r, rel_y = S.rms(a.double().numpy(), b.double().numpy() if resid else None,
                                  gamma.astype(np.float64), EPS)
    R.near("inv_rms", host(inv)[:n], r, rel_r * r)
    assert host(inv)[n] == 77
    _check_rows(t, out, y, np.full(n, rel_y))
    if resid:  # one fp32 addition, rounded to the type
        R.near("sum", _h64(total), h, S.U * np.abs(h) + R.half_step(t, h) * (1 + 2.0 ** -9))
    # inv_rms not wanted: the same rows
    again = torch.empty_like(out)
    if resid:
        M.residual_rmsnorm_forward(A, B, G, total, again, None, n, c, EPS)
    else:
        M.rmsnorm_forward(A, G, again, None, n, c, EPS)
    assert torch.equal(again, out)


@pytest.mark.parametrize("block", [0, 128])
@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,c", SHAPES)
def test_forward_in_8_bits(dev, n, c, t, fmt, block):
    note(f"rmsnorm row8 {n}x{c} {t} {fmt} block={block}")
    resid = (n + c) % 2 == 0
    code, largest, dtype = FORMATS[fmt]
    a, b, gamma = _inputs(n, c, t, n * 11 + c)
    A, B, G = _off(a), _off(b), dev_t(gamma)
    q = torch.full((n * c + 1,), 77, dtype=torch.uint8, device=dev)
    scales = torch.full((M.row8_scales(n, c, block) + 1,), 77.0, device=dev)
    total, out = torch.full_like(A, 77), torch.full_like(A, 77)
    inv = torch.empty(n, device=dev)

    def call(out, inv):
        if resid:
            M.residual_rmsnorm_forward_row8(A, B, G, total, q, scales, out, inv, n, c, EPS, block,
                                            code)
        else:
            M.rmsnorm_forward_row8(A, G, q, scales, out, inv, n, c, EPS, block, code)
    call(None, None)
    h, r, y, rel_r, rel_y = S.rms(a.double().numpy(), b.double().numpy() if resid else None,
                                  gamma.astype(np.float64), EPS)
    want, v = S.scales_of(y, block, largest)
    # the largest value's error, the division's
    R.near("scales", host(scales)[:-1].reshape(want.shape), want, (rel_y + 2 * S.U) * want)
    codes = host(q)[:-1].reshape(n, c)
    R.near("codes", S.code_values(codes, fmt), v, S.code_bound(v, fmt))
    assert host(q)[-1] == 77 and host(scales)[-1] == 77
    if resid:
        R.near("sum", _h64(total), h, S.U * np.abs(h) + R.half_step(t, h) * (1 + 2.0 ** -9))
    # with the rows too: those of the call that gives nothing else, and the same codes
    q0, s0 = q.clone(), scales.clone()
    call(out, inv)
    assert torch.equal(q, q0) and torch.equal(scales, s0)
    plain, inv1 = torch.empty_like(out), torch.empty_like(inv)
    if resid:
        M.residual_rmsnorm_forward(A, B, G, total, plain, inv1, n, c, EPS)
    else:
        M.rmsnorm_forward(A, G, plain, inv1, n, c, EPS)
    assert torch.equal(out, plain) and torch.equal(inv, inv1)
    # torch reads the codes as what they stand for
    back = q[:-1].view(dtype).float().cpu().numpy().reshape(n, c)
    assert np.array_equal(back, S.code_values(codes, fmt).astype(np.float32))


@pytest.mark.parametrize("block", [0, 128])
@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("c", [5, 40, 777, 2304, 20000])
def test_rows_that_hold_no_numbers(dev, c, t, fmt, block):
    """NaN and infinities stay in their row, or in the block whose values they touch: all of a
    row's values are NaN where its mean square is, and 0 (but the infinite ones) where it is
    infinite.  Rows of zeros have scale 2^-100 / Q and codes 0."""
    note(f"rmsnorm non-finite {c} {t} {fmt} block={block}")
    code, largest, _ = FORMATS[fmt]
    x = torch.ones(6, c, dtype=R.TYPES[t])
    x[1, 3], x[2, c - 1], x[3, 0], x[4] = np.nan, np.inf, -np.inf, 0.0
    x[5] = float(torch.finfo(R.TYPES[t]).smallest_normal)
    q = torch.full((6, c), 77, dtype=torch.uint8, device=dev)
    scales = torch.empty(6, M.row8_scales(1, c, block), device=dev)
    out, inv = torch.empty(6, c, dtype=x.dtype, device=dev), torch.empty(6, device=dev)
    M.rmsnorm_forward_row8(x.to(dev), torch.ones(c, device=dev), q, scales, out, inv, 6, c, EPS,
                           block, code)
    y, s, codes = _h64(out), host(scales), S.code_values(host(q), fmt)
    assert np.isnan(y[1]).all() and np.isnan(s[1]).all()
    for i, at in ((2, c - 1), (3, 0)):
        assert np.isnan(y[i, at]) and (np.delete(y[i], at) == 0).all()
        bad = np.zeros(s.shape[1], bool)
        bad[at // 128 if block else 0] = True
        assert np.isnan(s[i][bad]).all()
        assert (s[i][~bad] == np.float32(2.0 ** -100) / np.float32(largest)).all()
    assert (codes[1:5] == 0).all() and (s[4] == np.float32(2.0 ** -100) / np.float32(largest)).all()
    assert (codes[0] == largest).all() and np.isfinite(y[[0, 4, 5]]).all()
    assert host(inv)[2] == 0 and host(inv)[3] == 0 and np.isnan(host(inv)[1])
    assert np.isfinite(s[5]).all()
    # eps = 0: a row of zeros has no root to divide by
    M.rmsnorm_forward_row8(x.to(dev), torch.ones(c, device=dev), q, scales, out, inv, 6, c, 0.0,
                           block, code)
    assert np.isnan(_h64(out)[4]).all() and np.isnan(host(scales)[4]).all()
    assert (S.code_values(host(q), fmt)[4] == 0).all()


@pytest.mark.parametrize("resid", [False, True])
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,c", SHAPES + [(5000, 64), (3000, 200), (700, 6100)])
def test_backward(dev, n, c, t, resid):
    note(f"rmsnorm backward {n}x{c} {t} residual={resid}")
    rng = np.random.default_rng(n * 13 + c)
    x, _, gamma = _inputs(n, c, t, n * 13 + c, hard=False)
    dy, old = _rows(rng, n, c, t), _rows(rng, n, c, t)
    r = S.rms(x.double().numpy(), None, 1.0, EPS)[1].astype(np.float32)
    dg0 = rng.standard_normal(c).astype(np.float32)
    DX, DG = _off(old), dev_t(dg0)
    f = M.rmsnorm_backward_residual if resid else M.rmsnorm_backward
    f(_off(dy), _off(x), dev_t(r), dev_t(gamma), DX, DG, n, c)
    dx, bound, dg, dg_bound = S.rms_back(dy.double().numpy(), x.double().numpy(),
                                         r.astype(np.float64), gamma.astype(np.float64),
                                         old.double().numpy() if resid else None)
    R.near("dx", _h64(DX), dx, bound + R.half_step(t, dx) * (1 + 2.0 ** -9))
    R.near("dgamma", host(DG), dg0 + dg, dg_bound + 2 * S.U * np.abs(dg0 + dg))


MANY = [(8192, 8), (8200, 60), (9000, 116), (8193, 130), (8192, 200), (8300, 252), (8197, 256),
        (8192, 339), (8199, 386), (8211, 450), (8192, 512), (8205, 576), (8192, 646), (8207, 771),
        (8192, 782), (8199, 1000), (8193, 1030), (8192, 1330)]


@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,c", MANY)
def test_many_rows(dev, n, c, t):
    """Many rows that share waves, in every number of steps: some rows against 64 bits, forward
    with the residual as rows and in both kinds of 8 bits, backward; gamma's gradient whole."""
    note(f"rmsnorm many rows {n}x{c} {t}")
    r = np.random.default_rng(c)
    gen = torch.Generator(device="cuda").manual_seed(c)
    a, b, dy = (torch.randn(n, c, device=dev, generator=gen).to(R.TYPES[t]) for _ in range(3))
    gamma = (1 + 0.1 * r.standard_normal(c)).astype(np.float32)
    A, B, DY, G = _off(a), _off(b), _off(dy), dev_t(gamma)
    some = np.unique(np.concatenate([np.arange(20), r.integers(0, n, 60), np.arange(n - 20, n)]))
    at = torch.from_numpy(some).to(dev)
    g64 = gamma.astype(np.float64)
    h, inv, y, rel_r, rel_y = S.rms(_h64(a[at]), _h64(b[at]), g64, EPS)
    out, total, gi = torch.full_like(a, 77), torch.full_like(a, 77), torch.full((n,), 77.0, device=dev)
    M.residual_rmsnorm_forward(A, B, G, total, out, gi, n, c, EPS)
    _check_rows(t, out[at], y, np.full(len(some), rel_y))
    R.near("sum", _h64(total[at]), h, S.U * np.abs(h) + R.half_step(t, h) * (1 + 2.0 ** -9))
    R.near("inv_rms", _h64(gi[at]), inv, rel_r * inv)
    q = torch.full((n, c), 77, dtype=torch.uint8, device=dev)
    for block, fmt in ((0, "int8"), (128, "e4m3"), (128, "int8")):
        code, largest, _ = FORMATS[fmt]
        scales = torch.full((n, M.row8_scales(1, c, block)), 77.0, device=dev)
        M.residual_rmsnorm_forward_row8(A, B, G, total, q, scales, None, None, n, c, EPS, block, code)
        want, v = S.scales_of(y, block, largest)
        R.near("scales", _h64(scales[at]), want, (rel_y + 2 * S.U) * want)
        R.near("codes", S.code_values(host(q[at]), fmt), v, S.code_bound(v, fmt))
    x, rr = total, gi
    dg = torch.zeros(c, device=dev)
    for resid in (False, True):
        dx = b.clone()
        f = M.rmsnorm_backward_residual if resid else M.rmsnorm_backward
        f(DY, x, rr, G, dx, dg.zero_(), n, c)
        want, bound, _, _ = S.rms_back(_h64(dy[at]), _h64(x[at]), _h64(rr[at]), g64,
                                       _h64(b[at]) if resid else None)
        R.near("dx", _h64(dx[at]), want, bound + R.half_step(t, want) * (1 + 2.0 ** -9))
        terms = dy.double() * x.double() * rr.double()[:, None]
        # as in step_ref.rms_back
        R.near("dgamma", host(dg), host(terms.sum(0)),
               host(terms.abs().sum(0)) * (n // 256 + 103) * S.U)


@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,c", [(140_001, 60), (40_003, 600), (17_001, 2101), (8_300, 4200),
                                 (290_001, 251)])
def test_more_rows_than_workgroups(dev, n, c, t):
    """Rows in 8 bits, without the residual: a workgroup takes several, one after another.  Rows
    with it, among them rows that are streamed and end inside cache lines."""
    note(f"rmsnorm more rows than workgroups {n}x{c} {t}")
    r = np.random.default_rng(c)
    gen = torch.Generator(device="cuda").manual_seed(c)
    a = torch.randn(n, c, device=dev, generator=gen).to(R.TYPES[t])
    gamma = (1 + 0.1 * r.standard_normal(c)).astype(np.float32)
    A, G = _off(a), dev_t(gamma)
    some = np.unique(np.concatenate([np.arange(20), r.integers(0, n, 80), np.arange(n - 20, n)]))
    at = torch.from_numpy(some).to(dev)
    _, inv, y, rel_r, rel_y = S.rms(_h64(a[at]), None, gamma.astype(np.float64), EPS)
    q = torch.full((n + 1, c), 77, dtype=torch.uint8, device=dev)
    for block, fmt in ((0, "int8"), (128, "e4m3")):
        code, largest, _ = FORMATS[fmt]
        scales = torch.full((n + 1, M.row8_scales(1, c, block)), 77.0, device=dev)
        gi = torch.full((n + 1,), 77.0, device=dev)
        M.rmsnorm_forward_row8(A, G, q, scales, None, gi, n, c, EPS, block, code)
        want, v = S.scales_of(y, block, largest)
        R.near("inv_rms", _h64(gi[at]), inv, rel_r * inv)
        R.near("scales", _h64(scales[at]), want, (rel_y + 2 * S.U) * want)
        R.near("codes", S.code_values(host(q[at]), fmt), v, S.code_bound(v, fmt))
        # in place of the input's rows, and none left out
        assert (scales[:n] < 77).all() and (scales[n:] == 77).all() and (q[n] == 77).all()
        q0, s0, X = q.clone(), scales.clone(), A.clone()
        M.rmsnorm_forward_row8(X, G, q.fill_(77), scales.fill_(77), X, None, n, c, EPS, block, code)
        assert torch.equal(q, q0) and torch.equal(scales, s0)
    # a + a, exactly twice as large
    out, total = torch.full_like(a, 77), torch.full_like(a, 77)
    M.residual_rmsnorm_forward(A, A, G, total, out, gi, n, c, EPS)
    h, inv, y, rel_r, rel_y = S.rms(_h64(a[at]), _h64(a[at]), gamma.astype(np.float64), EPS)
    R.near("inv_rms", _h64(gi[at]), inv, rel_r * inv)
    _check_rows(t, out[at], y, np.full(len(some), rel_y))
    assert torch.equal(total, a + a)


@pytest.mark.parametrize("n,c", [(300, 140_003), (40, 2_097_155)])
def test_very_long_rows(dev, n, c):
    """Rows of so many columns that a workgroup for each would take too many partial rows: each
    takes several rows, one after another."""
    note(f"rmsnorm very long rows {n}x{c}")
    gen = torch.Generator(device="cuda").manual_seed(c)
    a, b = (torch.randn(n, c, device=dev, generator=gen).bfloat16() for _ in range(2))
    gamma = (1 + 0.1 * np.random.default_rng(c).standard_normal(c)).astype(np.float32)
    G, g64 = dev_t(gamma), gamma.astype(np.float64)
    out, total, inv = torch.empty_like(a), torch.empty_like(a), torch.empty(n, device=dev)
    q, s = torch.empty(n, c, dtype=torch.uint8, device=dev), torch.empty(n, M.row8_scales(1, c, 128), device=dev)
    M.residual_rmsnorm_forward_row8(a, b, G, total, q, s, out, inv, n, c, EPS, 128)
    some = [0, 1, n - 17, n - 1]
    _, r, y, rel_r, rel_y = S.rms(_h64(a[some]), _h64(b[some]), g64, EPS)
    R.near("inv_rms", _h64(inv[some]), r, rel_r * r)
    _check_rows("bf16", out[some], y, np.full(len(some), rel_y))
    want, v = S.scales_of(y, 128, 448.0)
    R.near("scales", _h64(s[some]), want, (rel_y + 2 * S.U) * want)
    R.near("codes", S.code_values(host(q[some]), "e4m3"), v, S.code_bound(v, "e4m3"))
    terms = torch.zeros(2, c, dtype=torch.float64, device=dev)
    for i in range(n):
        t = out[i].double() * total[i].double() * inv[i].double()
        terms += torch.stack([t, t.abs()])
    for resid in (False, True):
        dx, dg = b.clone(), torch.zeros(c, device=dev)
        f = M.rmsnorm_backward_residual if resid else M.rmsnorm_backward
        f(out, total, inv, G, dx, dg, n, c)
        want, bound, _, _ = S.rms_back(_h64(out[some]), _h64(total[some]), _h64(inv[some]), g64,
                                       _h64(b[some]) if resid else None)
        R.near("dx", _h64(dx[some]), want, bound + R.half_step("bf16", want) * (1 + 2.0 ** -9))
        # a term's two products and fewer than 400 additions: 300 rows at most, 100 partial rows
        # to a slice, the old value
        R.near("dgamma", host(dg), host(terms[0]), host(terms[1]) * 403 * S.U)


def test_gradient_against_differences(dev):
    """The gradient of sum(c * out) by the backward call and by differences of the forward call.
    Step 2^-6: the difference's own error is about h^2 / 6 = 4e-5 of the third derivative (of
    order 1 here), and the outputs' rounding 3 * 2^-24 / 2^-6 = 1e-5 for each of the row's terms
    that change, in root mean square over 24 columns 6e-5."""
    n, c, step = 3, 24, 2.0 ** -6
    rng = np.random.default_rng(5)
    x, gamma = rng.standard_normal((n, c)), 1 + 0.1 * rng.standard_normal(c)
    w = rng.standard_normal((n, c))

    def value(x, gamma):
        out = torch.empty(n, c, device=dev)
        M.rmsnorm_forward(dev_t(x.astype(np.float32)), dev_t(gamma.astype(np.float32)), out, None, n,
                          c, EPS)
        return (host(out).astype(np.float64) * w).sum(1)
    x32, g32 = x.astype(np.float32).astype(np.float64), gamma.astype(np.float32).astype(np.float64)
    out, inv = torch.empty(n, c, device=dev), torch.empty(n, device=dev)
    X, G = dev_t(x32.astype(np.float32)), dev_t(g32.astype(np.float32))
    M.rmsnorm_forward(X, G, out, inv, n, c, EPS)
    dx, dg = torch.empty(n, c, device=dev), torch.zeros(c, device=dev)
    M.rmsnorm_backward(dev_t(w.astype(np.float32)), X, inv, G, dx, dg, n, c)
    w = w.astype(np.float32).astype(np.float64)
    for j in range(c):
        e = np.zeros(c)
        e[j] = step
        num = (value(x32 + e, g32) - value(x32 - e, g32)) / (2 * step)
        assert np.allclose(host(dx)[:, j], num, rtol=0, atol=5e-4), j
        num = (value(x32, g32 + e) - value(x32, g32 - e)).sum() / (2 * step)
        assert abs(host(dg)[j] - num) <= 5e-4, j


@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,c", [(9, 60), (40, 129), (1030, 769), (6, 5003), (3, 20001), (5, 3)])
def test_in_place(dev, n, c, t):
    """out in x, residual_out in a or b, the codes' rows in x, grad_x in grad_out: the same bits
    as in buffers of their own."""
    note(f"rmsnorm in place {n}x{c} {t}")
    a, b, gamma = _inputs(n, c, t, c)
    A, B, G = a.to(dev), b.to(dev), dev_t(gamma)
    out, total, inv = torch.empty_like(A), torch.empty_like(A), torch.empty(n, device=dev)
    M.rmsnorm_forward(A, G, out, inv, n, c, EPS)
    X = A.clone()
    M.rmsnorm_forward(X, G, X, inv, n, c, EPS)
    assert torch.equal(X, out)
    q, q1 = torch.empty(2, n, c, dtype=torch.uint8, device=dev)
    s = torch.empty(M.row8_scales(n, c, 128), device=dev)
    M.rmsnorm_forward_row8(A, G, q, s, None, None, n, c, EPS, 128)
    X = A.clone()
    M.rmsnorm_forward_row8(X, G, q1, s, X, None, n, c, EPS, 128)
    assert torch.equal(X, out) and torch.equal(q, q1)
    M.residual_rmsnorm_forward(A, B, G, total, out, inv, n, c, EPS)
    for first in (True, False):
        X, Y, out1 = A.clone(), B.clone(), torch.empty_like(A)
        M.residual_rmsnorm_forward(X, Y, G, X if first else Y, out1, None, n, c, EPS)
        assert torch.equal(X if first else Y, total) and torch.equal(out1, out)
        X, Y = A.clone(), B.clone()
        for block in (0, 128):
            X, Y = A.clone(), B.clone()
            M.residual_rmsnorm_forward_row8(X, Y, G, X if first else Y, q1, s, out1, None, n, c,
                                            EPS, block)
            assert torch.equal(X if first else Y, total) and torch.equal(out1, out)
    M.rmsnorm_forward(A, G, out, inv, n, c, EPS)
    dx, dg, dg1 = torch.empty_like(A), torch.zeros(c, device=dev), torch.zeros(c, device=dev)
    M.rmsnorm_backward(B, A, inv, G, dx, dg, n, c)
    Y = B.clone()
    M.rmsnorm_backward(Y, A, inv, G, Y, dg1, n, c)
    assert torch.equal(Y, dx) and torch.equal(dg, dg1)


@pytest.mark.parametrize("c", [64, 1600, 3001])
def test_rows_behind_the_last_are_left(dev, c):
    n = 1029
    a, b, gamma = _inputs(n, c, "bf16", c)
    A, B, G = a.to(dev), b.to(dev), dev_t(gamma)
    m = n - 3
    out, total, dx = (torch.full_like(A, 77) for _ in range(3))
    q = torch.full((n, c), 77, dtype=torch.uint8, device=dev)
    s, inv = torch.full((n, 1), 77.0, device=dev), torch.full((n,), 77.0, device=dev)
    dg = torch.zeros(c, device=dev)
    M.residual_rmsnorm_forward_row8(A, B, G, total, q, s, out, inv, m, c)
    M.rmsnorm_backward(B, total, inv, G, dx, dg, m, c)
    for x in (out, total, q, s, inv, dx):
        assert (x[m:].float() == 77).all()


def test_same_bits_again_and_from_a_graph(dev):
    """Eager calls, calls on another stream and replays of a captured forward and backward give
    the same bits, with eager work of another shape between the replays."""
    n, c = 3000, 1600
    a, b, gamma = _inputs(n, c, "bf16", 3, hard=False)
    A, B, G = a.to(dev), b.to(dev), dev_t(gamma)
    total, out, dx = (torch.empty_like(A) for _ in range(3))
    q = torch.empty(n, c, dtype=torch.uint8, device=dev)
    s, inv, dg = torch.empty(n, 13, device=dev), torch.empty(n, device=dev), torch.empty(c, device=dev)
    names = (total, out, q, s, inv, dx, dg)

    def step():
        dg.fill_(0.0)
        dx.fill_(0.5)
        M.residual_rmsnorm_forward_row8(A, B, G, total, q, s, out, inv, n, c, EPS, 128)
        M.rmsnorm_backward_residual(out, total, inv, G, dx, dg, n, c)
    step()
    torch.cuda.synchronize()
    ref = [x.clone() for x in names]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(names, ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    small = torch.ones(5, 100, device=dev)
    sdg, sinv = torch.zeros(100, device=dev), torch.ones(5, device=dev)
    for rep in range(4):
        for x in names:
            x.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(names, ref)), rep
        M.rmsnorm_backward(small, small, sinv, torch.ones(100, device=dev),
                           torch.empty_like(small), sdg, 5, 100)
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(names, ref)), rep


def test_past_2_31_elements(dev):
    """Element numbers past 2^31: the first and last rows have the bits that a call on these
    rows alone gives (both hold a row the same way)."""
    n, c = 1_100_011, 2000
    note(f"rmsnorm {n}x{c}")
    gen = torch.Generator(device="cuda").manual_seed(1)
    a = torch.randn(n, c, device=dev, generator=gen, dtype=torch.bfloat16)
    g = 1 + 0.1 * torch.randn(c, device=dev, generator=gen)
    out, total = torch.empty_like(a), torch.empty_like(a)
    q = torch.empty(n, c, dtype=torch.uint8, device=dev)
    s, inv = torch.empty(n, 16, device=dev), torch.empty(n, device=dev)
    M.residual_rmsnorm_forward_row8(a, a, g, total, q, s, out, inv, n, c, EPS, 128)
    dx, dg = torch.empty_like(a), torch.zeros(c, device=dev)
    M.rmsnorm_backward(out, total, inv, g, dx, dg, n, c)
    m = 1100
    for part in (slice(0, m), slice(n - m, n)):
        o, t, d = (torch.empty(m, c, dtype=torch.bfloat16, device=dev) for _ in range(3))
        q1, s1, i1 = torch.empty(m, c, dtype=torch.uint8, device=dev), s[:m].clone(), inv[:m].clone()
        x = a[part].contiguous()
        M.residual_rmsnorm_forward_row8(x, x, g, t, q1, s1, o, i1, m, c, EPS, 128)
        M.rmsnorm_backward(o, t, i1, g, d, torch.zeros(c, device=dev), m, c)
        for got, want in ((out, o), (total, t), (q, q1), (s, s1), (inv, i1), (dx, d)):
            assert torch.equal(got[part], want)
    want = torch.zeros(c, dtype=torch.float64, device=dev)
    size = torch.zeros(c, dtype=torch.float64, device=dev)
    for i in range(0, n, 100_000):
        p = slice(i, i + 100_000)
        terms = out[p].double() * total[p].double() * inv[p].double()[:, None]
        want += terms.sum(0)
        size += terms.abs().sum(0)
    R.near("dgamma", host(dg), host(want), host(size) * (n / 256 / 2 + 100) * S.U)


@pytest.mark.parametrize("block", [0, 128])
@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("n,c", [(3, 5), (4, 40), (1030, 300), (1030, 1600), (5, 5000), (2, 14000)])
def test_codes_of_small_products(dev, n, c, fmt, block):
    """Without eps tiny rows are normalised like any others.  h gamma below 2^-110, whose factor
    to a code passes fp32's range, but above its smallest normal numbers, 2^-126: rows whose
    largest y is ordinary, one whose values are all small but in one block, and one below 2^-100."""
    note(f"rmsnorm codes of small products {n}x{c} {fmt} block={block}")
    code, largest, _ = FORMATS[fmt]
    r = np.random.default_rng(c)
    x = np.sign(r.standard_normal((n, c))) * r.uniform(0.5, 1.0, (n, c))
    x[1] *= 2.0 ** 3
    one = np.ones(c)
    one[c // 2] = 2.0 ** 26
    q = torch.full((n, c), 77, dtype=torch.uint8, device=dev)
    scales = torch.full((n, M.row8_scales(1, c, block)), 77.0, device=dev)
    for size, g in ((2.0 ** -30, one * 2.0 ** -86), (2.0 ** -30, np.full(c, 2.0 ** -92)),
                    (2.0 ** -23, np.full(c, 0.7 * 2.0 ** -101))):
        h32, g32 = (x * size).astype(np.float32), g.astype(np.float32)
        M.rmsnorm_forward_row8(dev_t(h32), dev_t(g32), q, scales, None, None, n, c, 0.0, block, code)
        h, _, y, _, rel_y = S.rms(h32.astype(np.float64), None, g32.astype(np.float64), 0.0)
        assert np.abs(h * g32).min() > 2.0 ** -126
        want, v = S.scales_of(y, block, largest)
        R.near("scales", host(scales), want, (rel_y + 2 * S.U) * want)
        R.near("codes", S.code_values(host(q), fmt), v, S.code_bound(v, fmt))
