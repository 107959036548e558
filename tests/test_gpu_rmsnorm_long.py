"""GPU parity of the RMS norm on rows of equal values and millions of columns, where a sum of
fp32 numbers one after another rounds to the same side every time, and on millions of rows of a
few columns.  Bounds do not grow with the number of columns."""
import numpy as np
import pytest
import torch

import cme213_amd as M
import moe_ref as R
import step_ref as S
from gpu_util import host, note

pytestmark = pytest.mark.gpu

EPS = 1e-5
# a thread's sum, rounded once to fp32, then 6 additions over lanes and 3 over waves
CHAIN = 10


def _h64(t):
    return host(t.double())


@pytest.mark.parametrize("value", [1.001, 0.7])
@pytest.mark.parametrize("t,c", [("f32", 20_003), ("bf16", 2 ** 21 + 3), ("f32", 2 ** 21), ("f32", 2 ** 24)])
def test_long_rows_of_equal_values(dev, t, c, value):
    note(f"rmsnorm long rows {c} {t} {value}")
    n = 2
    x = torch.full((n, c), value, dtype=R.TYPES[t], device=dev)
    x[1] = x[1] * 0.25
    G = torch.ones(c, device=dev)
    out, inv = torch.empty_like(x), torch.empty(n, device=dev)
    M.rmsnorm_forward(x, G, out, inv, n, c, EPS)
    v = _h64(x[:, 0])
    r = 1 / np.sqrt(v * v + EPS)
    # the sum's chain, the division by cols, eps's rounding and addition, halved by the root; the
    # root and the division
    rel = ((CHAIN + 3) / 2 + 2) * S.U
    R.near("inv_rms", _h64(inv), r, rel * r)
    for part in (slice(0, 300), slice(c - 300, c)):
        y = np.repeat((v * r)[:, None], 300, 1)
        R.near("out", _h64(out[:, part]), y, (rel + 2 * S.U) * np.abs(y) * (1 + 2.0 ** -7) +
               R.half_step(t, y) * (1 + 2.0 ** -9))
    # with the residual, and in 8 bits: the same statistics of exactly twice the values
    total, q = torch.empty_like(x), torch.empty(n, c, dtype=torch.uint8, device=dev)
    for block in (0, 128):
        s = torch.empty(n, M.row8_scales(1, c, block), device=dev)
        M.residual_rmsnorm_forward_row8(x, x, G, total, q, s, out, inv, n, c, EPS, block)
        r2 = 1 / np.sqrt(4 * v * v + EPS)
        R.near("inv_rms", _h64(inv), r2, rel * r2)
        want = np.repeat((2 * v * r2 / 448)[:, None], s.shape[1], 1)
        R.near("scales", _h64(s), want, (rel + 5 * S.U) * want)
        assert bool((q.view(torch.float8_e4m3fn).float() == 448).all())


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("value", [1.001, 0.7])
@pytest.mark.parametrize("t,c", [("f32", 20_003), ("bf16", 2 ** 21 + 3), ("f32", 2 ** 21)])
def test_gradient_of_long_rows_of_equal_values(dev, t, c, value, add):
    """The mean of g n is what is left of g to within a few roundings: dx nearly vanishes, and an
    error of the mean is all that it shows."""
    note(f"rmsnorm gradient of long rows {c} {t} {value} add={add}")
    n = 2
    x = torch.full((n, c), value, dtype=R.TYPES[t], device=dev)
    dy = torch.full((n, c), 1.37, dtype=R.TYPES[t], device=dev)
    G = torch.full((c,), 0.9, device=dev)
    inv = (1 / torch.sqrt(x[:, 0].double() ** 2 + EPS)).float()
    dx = torch.full_like(x, 0.0)
    dg = torch.zeros(c, device=dev)
    f = M.rmsnorm_backward_residual if add else M.rmsnorm_backward
    f(dy, x, inv, G, dx, dg, n, c)
    r, d, g0 = _h64(inv)[0], _h64(dy)[0, 0], _h64(G)[0]
    norm, g = _h64(x)[0, 0] * r, d * g0
    m = g * norm
    want = r * (g - norm * m)
    # m: three roundings a term, the chain, the division; dx as step_ref.rms_back counts it
    em = (CHAIN + 4) * S.U * m
    bound = r * (5 * S.U * (g + norm * m) + norm * em) + S.U * abs(want)
    for part in (slice(0, 300), slice(c - 300, c)):
        w = np.full((n, 300), want)
        R.near("dx", _h64(dx[:, part]), w, bound + R.half_step(t, w) * (1 + 2.0 ** -9))
        w = np.full(300, 2 * d * norm)
        R.near("dgamma", _h64(dg[part]), w, 6 * S.U * w)


@pytest.mark.parametrize("t,n,c", [("f32", 2 ** 24, 3), ("bf16", 2 ** 23 + 77, 5), ("f16", 2 ** 22, 1)])
def test_many_rows_of_a_few_columns(dev, t, n, c):
    """Gamma's gradient over millions of equal rows."""
    note(f"rmsnorm many rows of a few columns {n}x{c} {t}")
    x = torch.full((n, c), 0.7, dtype=R.TYPES[t], device=dev)
    dy = torch.full((n, c), 1.001, dtype=R.TYPES[t], device=dev)
    r = (1 / torch.sqrt(x[0, 0].double() ** 2 + EPS)).float()
    inv = torch.full((n,), float(r), device=dev)
    dx, dg = torch.empty_like(x), torch.full((c,), 5.0, device=dev)
    M.rmsnorm_backward(dy, x, inv, torch.ones(c, device=dev), dx, dg, n, c)
    want = n * _h64(dy)[0] * _h64(x)[0] * _h64(r)
    # n = x r and its product once each, a workgroup's sum once, its 256 partial rows in 16 slices of 16, the old value
    R.near("dgamma", _h64(dg), want + 5, (3 + 32) * S.U * want + S.U * (want + 5))
