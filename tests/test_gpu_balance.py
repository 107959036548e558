"""GPU parity of the router's balance loss against a plain 64-bit implementation (step_ref.py,
where the bounds are derived): counts exact, padded tokens, masked experts, rows with nothing to
choose, infinite and NaN logits, no valid token, ids out of range, one workgroup and many."""
import numpy as np
import pytest
import torch

import cme213_amd as M
import moe_ref as R
import step_ref as S
from gpu_util import dev_t, host, note
from tol import assert_exact

pytestmark = pytest.mark.gpu

COEF = 0.01
SHAPES = [(1, 1, 1), (1, 8, 2), (16, 8, 2), (17, 16, 16), (5, 33, 4), (64, 64, 6), (300, 20, 3),
          (257, 8, 2), (256, 128, 8), (9, 160, 8), (700, 256, 1), (33, 257, 16), (450, 300, 5),
          (270, 512, 8), (3, 1000, 3), (600, 1024, 16), (20001, 64, 6), (5001, 1024, 2)]


def _h64(t):
    return host(t.double())


def _inputs(n, e, k, t, seed):
    """Logits, a fifth of them masked, some rows wholly; ids of slots, some of them dropped;
    valid tokens."""
    r = np.random.default_rng(seed)
    l = r.standard_normal((n, e)) * 1.5 + r.standard_normal(e) * 0.7
    l[r.random((n, e)) < 0.2] = -np.inf
    if n > 3:
        l[1] = -np.inf
        l[2] = float(torch.finfo(R.TYPES[t]).min)
    ids = r.integers(0, e, (n, k)).astype(np.int32)
    ids[r.random((n, k)) < 0.1] = -1
    if n > 4:
        ids[3, 0], ids[4, 0] = e, 2 ** 31 - 1
        ids[3, -1] = -2 ** 31
    valid = (r.random(n) < 0.8).astype(np.uint8) * r.integers(1, 256, n).astype(np.uint8)
    return torch.from_numpy(l).to(R.TYPES[t]), ids, valid


@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,e,k", SHAPES)
def test_forward_backward(dev, n, e, k, t, padded):
    note(f"balance {n}x{e} k={k} {t} padded={padded}")
    l, ids, valid = _inputs(n, e, k, t, n * 10 + e)
    valid = valid if padded else None
    counts = torch.full((e + 2,), 77, dtype=torch.int32, device=dev)
    probs, loss = torch.full((e + 1,), 77.0, device=dev), torch.full((2,), 77.0, device=dev)
    L, V = l.to(dev), None if valid is None else dev_t(valid)
    M.moe_balance_forward(L, dev_t(ids), V, counts, probs, loss, n, e, k, COEF)
    l64 = l.double().numpy()
    c, p, p_bound, want, bound = S.balance(l64, ids, valid, k, COEF)
    assert_exact("counts", host(counts)[:-1], c)
    R.near("probs", host(probs)[:-1], p, p_bound + 2.0 ** -140)
    R.near("loss", host(loss)[:1], [want], [bound + 2.0 ** -140])
    assert host(counts)[-1] == 77 and host(probs)[-1] == 77 and host(loss)[1] == 77
    # the gradient, with the loss's own and what is there
    r = np.random.default_rng(e)
    dloss = 1024.0
    g, g_bound = S.balance_back(l64, valid, c, dloss, k, COEF)
    old = torch.from_numpy(r.standard_normal((n, e)) * 1e-3).to(R.TYPES[t])
    D = old.to(dev)
    M.moe_balance_backward(L, V, counts[:-1].contiguous(), torch.full((1,), dloss, device=dev), D,
                           n, e, k, COEF, True)
    both = old.double().numpy() + g
    R.near("dlogits +=", _h64(D), both,
           g_bound + S.U * np.abs(both) + R.half_step(t, both) * (1 + 2.0 ** -9))
    if valid is not None:
        assert torch.equal(D.cpu()[valid == 0], old[valid == 0])
    D = torch.full((n, e), 77.0, dtype=R.TYPES[t], device=dev)
    M.moe_balance_backward(L, V, counts[:-1].contiguous(), None, D, n, e, k, COEF * dloss, False)
    R.near("dlogits", _h64(D), g, g_bound + 2 * S.U * np.abs(g) + R.half_step(t, g) * (1 + 2.0 ** -9))


@pytest.mark.parametrize("n", [5, 1000])
def test_no_valid_token(dev, n):
    e, k = 12, 2
    counts = torch.full((e + 1,), 77, dtype=torch.int32, device=dev)
    probs, loss = torch.full((e,), 77.0, device=dev), torch.full((1,), 77.0, device=dev)
    l = torch.full((n, e), float("nan"), device=dev)
    ids = torch.zeros(n, k, dtype=torch.int32, device=dev)
    none = torch.zeros(n, dtype=torch.bool, device=dev)
    M.moe_balance_forward(l, ids, none, counts, probs, loss, n, e, k, COEF)
    assert not host(counts).any() and not host(probs).any() and host(loss)[0] == 0
    d = torch.full((n, e), 77.0, device=dev)
    M.moe_balance_backward(l, none, counts, None, d, n, e, k, COEF, False)
    assert not host(d).any()
    d.fill_(3.0)
    M.moe_balance_backward(l, none, counts, None, d, n, e, k, COEF, True)
    assert (host(d) == 3).all()
    # no tokens at all
    counts.fill_(77), probs.fill_(77), loss.fill_(77)
    M.moe_balance_forward(l, ids, None, counts, probs, loss, 0, e, k, COEF)
    assert not host(counts).any() and not host(probs).any() and host(loss)[0] == 0


@pytest.mark.parametrize("n", [6, 2000])
def test_nan_and_infinity(dev, n):
    """A NaN or +inf logit makes the loss and its own row's gradient NaN, no other row's; in a
    token that is not valid it does nothing."""
    e, k = 24, 2
    l = np.random.default_rng(1).standard_normal((n, e)).astype(np.float32)
    ids = np.random.default_rng(2).integers(0, e, (n, k)).astype(np.int32)
    counts = torch.empty(e + 1, dtype=torch.int32, device=dev)
    probs, loss = torch.empty(e, device=dev), torch.empty(1, device=dev)
    for bad in (np.nan, np.inf):
        x = l.copy()
        x[3, 5] = bad
        valid = np.ones(n, np.uint8)
        M.moe_balance_forward(dev_t(x), dev_t(ids), dev_t(valid), counts, probs, loss, n, e, k, COEF)
        assert np.isnan(host(loss)[0]) and np.isnan(host(probs)).all()
        d = torch.zeros(n, e, device=dev)
        M.moe_balance_backward(dev_t(x), None, counts, None, d, n, e, k, COEF, False)
        assert np.isnan(host(d)[3]).all() and np.isfinite(np.delete(host(d), 3, 0)).all()
        valid[3] = 0
        M.moe_balance_forward(dev_t(x), dev_t(ids), dev_t(valid), counts, probs, loss, n, e, k, COEF)
        assert np.isfinite(host(loss)[0]) and host(counts)[-1] == n - 1
        M.moe_balance_backward(dev_t(x), dev_t(valid), counts, None, d, n, e, k, COEF, False)
        assert np.isfinite(host(d)).all() and not host(d)[3].any()


def test_gradient_against_differences(dev):
    """The loss is a smooth function of the logits while the counts stand: the backward call
    against differences of the forward call's mean probabilities, whose sum with the counts in 64
    bits is the loss.  Step 2^-6: the difference's own error h^2 / 6 times the third derivative
    (at most the scale times the largest count) and the rounding of probs (40 U, over 2 h) times
    the counts: less than 1e-3 of the scale times the largest count."""
    n, e, k, coef, step = 5, 12, 2, 1.0, 2.0 ** -6
    r = np.random.default_rng(0)
    l = r.standard_normal((n, e)).astype(np.float32)
    ids = r.integers(0, e // 2, (n, k)).astype(np.int32)
    counts = torch.empty(e + 1, dtype=torch.int32, device=dev)
    probs, loss = torch.empty(e, device=dev), torch.empty(1, device=dev)

    def value(x):
        M.moe_balance_forward(dev_t(x.astype(np.float32)), dev_t(ids), None, counts, probs, loss, n, e,
                              k, coef)
        c = host(counts)[:e].astype(np.float64)
        v = coef * e / (k * n) * (c * host(probs).astype(np.float64)).sum()
        assert abs(v - host(loss)[0]) <= 4 * S.U * abs(v)
        return v
    value(l)
    d = torch.empty(n, e, device=dev)
    M.moe_balance_backward(dev_t(l), None, counts, None, d, n, e, k, coef, False)
    tol = 1e-3 * coef * e / (k * n) / n * host(counts)[:e].max()
    for t in range(n):
        for j in range(e):
            s = np.zeros((n, e), np.float32)
            s[t, j] = step
            num = (value(l + s) - value(l - s)) / (2 * step)
            assert abs(host(d)[t, j] - num) <= tol, (t, j)


def test_counts_of_several_processes(dev):
    """Two halves of a batch, their counts and probabilities summed as an all-reduce would: the
    whole batch's loss and gradient."""
    n, e, k = 600, 16, 2
    l, ids, _ = _inputs(n, e, k, "f32", 4)
    parts = []
    for p in (slice(0, 250), slice(250, n)):
        c, q, s = torch.empty(e + 1, dtype=torch.int32, device=dev), torch.empty(e, device=dev), torch.empty(1, device=dev)
        m = p.stop - p.start
        M.moe_balance_forward(l[p].to(dev), dev_t(ids[p]), None, c, q, s, m, e, k, COEF)
        parts.append((c, host(q).astype(np.float64) * m))
    counts = parts[0][0] + parts[1][0]
    c, p, p_bound, want, bound = S.balance(l.double().numpy(), ids, None, k, COEF)
    assert_exact("counts", host(counts), c)
    probs = (parts[0][1] + parts[1][1]) / n
    R.near("probs", probs, p, p_bound + 2 * S.U * p)
    g, g_bound = S.balance_back(l.double().numpy(), None, c, 1.0, k, COEF)
    for part in (slice(0, 250), slice(250, n)):
        m = part.stop - part.start
        d = torch.empty(m, e, device=dev)
        M.moe_balance_backward(l[part].to(dev), None, counts, None, d, m, e, k, COEF, False)
        R.near("dlogits", _h64(d), g[part], g_bound[part] + R.half_step("f32", g[part]))


def test_large_counts(dev):
    """Counts near 2^31 (summed over processes): what is left of them after their mean enters."""
    n, e, k = 40, 8, 2
    r = np.random.default_rng(3)
    l = r.standard_normal((n, e)).astype(np.float32)
    c = np.append(2 ** 31 - 1 - r.integers(0, 10 ** 6, e), 2 ** 31 - 1).astype(np.int32)
    d = torch.empty(n, e, device=dev)
    M.moe_balance_backward(dev_t(l), None, dev_t(c), torch.full((1,), 2.0 ** 20, device=dev), d, n, e,
                           k, 1.0, False)
    g, bound = S.balance_back(l.astype(np.float64), None, c.astype(np.int64), 2.0 ** 20, k, 1.0)
    # the mean is a sum of 8 numbers in fp32: what is left may be 4 * 2^7 larger
    R.near("dlogits", _h64(d), g, 3 * bound + R.half_step("f32", g))


def test_same_bits_again_and_from_a_graph(dev):
    n, e, k = 9000, 160, 8
    l, ids, valid = _inputs(n, e, k, "bf16", 9)
    L, I, V = l.to(dev), dev_t(ids), dev_t(valid)
    counts, probs = torch.empty(e + 1, dtype=torch.int32, device=dev), torch.empty(e, device=dev)
    loss, d = torch.empty(1, device=dev), torch.empty(n, e, dtype=torch.bfloat16, device=dev)
    names = (counts, probs, loss, d)

    def step():
        d.fill_(0.0)
        M.moe_balance_forward(L, I, V, counts, probs, loss, n, e, k, COEF)
        M.moe_balance_backward(L, V, counts, loss, d, n, e, k, COEF)
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
    for rep in range(4):
        for x in names:
            x.fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(names, ref)), rep
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(names, ref)), rep


def test_past_2_31_elements(dev):
    n, e, k = 2_200_003, 1000, 1
    note(f"balance {n}x{e}")
    gen = torch.Generator(device="cuda").manual_seed(1)
    l = torch.randn(n, e, device=dev, generator=gen, dtype=torch.bfloat16)
    ids = torch.randint(0, e, (n, k), device=dev, generator=gen, dtype=torch.int32)
    counts, probs = torch.empty(e + 1, dtype=torch.int32, device=dev), torch.empty(e, device=dev)
    loss, d = torch.empty(1, device=dev), torch.empty_like(l)
    M.moe_balance_forward(l, ids, None, counts, probs, loss, n, e, k, COEF)
    assert torch.equal(counts[:e].long(), torch.bincount(ids.view(-1), minlength=e))
    assert int(counts[e]) == n
    want = torch.zeros(e, dtype=torch.float64, device=dev)
    for i in range(0, n, 100_000):
        want += torch.softmax(l[i:i + 100_000].double(), 1).sum(0)
    # each p is off by at most about (4 * 12 + 32) U; n / 2048 rows of a lane, 280 partial rows
    R.near("probs", host(probs), host(want / n), host(want / n) * (80 + n / 2048 + 280) * S.U)
    M.moe_balance_backward(l, None, counts, torch.full((1,), 1e6, device=dev), d, n, e, k, COEF, False)
    for part in (slice(0, 50), slice(n - 50, n)):
        g, bound = S.balance_back(_h64(l[part]), None, host(counts), 1e6, k, COEF)
        R.near("dlogits", _h64(d[part]), g, bound + R.half_step("bf16", g) * (1 + 2.0 ** -9))


def _unlikely(n, e, k, low, seed):
    """Logits near 0, near `low` for the first half of the experts, which all ids are of."""
    r = np.random.default_rng(seed)
    l = r.standard_normal((n, e))
    l[:, :(e + 1) // 2] += low
    return l.astype(np.float32), r.integers(0, (e + 1) // 2, (n, k)).astype(np.int32)


@pytest.mark.parametrize("low", [-8, -14, -20, -30, -45, -75])
@pytest.mark.parametrize("n,e,k", [(200, 64, 2), (300, 64, 2), (9000, 8, 1), (2000, 1000, 4)])
def test_loss_of_unlikely_experts(dev, n, e, k, low):
    """Ids that a bias or a group chose, whose experts have hardly any probability: the loss is
    good to fp32 however small it is, by one workgroup and by many."""
    note(f"balance {n}x{e} k={k}, chosen experts' logits {low}")
    l, ids = _unlikely(n, e, k, low, n + e)
    counts, probs = torch.empty(e + 1, dtype=torch.int32, device=dev), torch.empty(e, device=dev)
    loss = torch.full((1,), 77.0, device=dev)
    M.moe_balance_forward(dev_t(l), dev_t(ids), None, counts, probs, loss, n, e, k, COEF)
    c, p, p_bound, want, bound = S.balance(l.astype(np.float64), ids, None, k, COEF)
    assert_exact("counts", host(counts), c)
    R.near("probs", host(probs), p, p_bound + 2.0 ** -140)
    R.near("loss", host(loss), [want], [bound])
    # and of the probabilities that the call wrote, to a rounding of the loss and of its last sum
    own = COEF * e / (k * n) * (c[:e] * host(probs).astype(np.float64)).sum()
    R.near("loss", host(loss), [own], [4 * S.U * own])
    before = host(loss).copy()
    M.moe_balance_forward(dev_t(l), dev_t(ids), None, counts, probs, loss, n, e, k, COEF)
    assert host(loss)[0] == before[0]


def test_loss_of_unlikely_experts_from_a_graph(dev):
    """Replays with other calls on the workspace between them, likely and unlikely in turn."""
    n, e, k = 3000, 96, 2
    counts, probs = torch.empty(e + 1, dtype=torch.int32, device=dev), torch.empty(e, device=dev)
    losses = torch.empty(2, device=dev)
    inputs = [tuple(dev_t(x) for x in _unlikely(n, e, k, low, 1)) for low in (-25, 0)]

    def step(which):
        l, ids = inputs[which]
        M.moe_balance_forward(l, ids, None, counts, probs, losses[which:which + 1], n, e, k, COEF)
    step(0), step(1)
    torch.cuda.synchronize()
    want = losses.clone()
    assert 0 < want[0] < 1e-9 < 1e-4 < want[1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(0), step(1), step(0)
    for rep in range(4):
        losses.fill_(77)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(losses, want), rep
        step(1)
        torch.cuda.synchronize()
        assert torch.equal(losses, want), rep
