"""GPU parity of the mixture-of-experts entry points against plain 64-bit
implementations (moe_ref.py, where the bounds are derived): the router's choice
and its gradient (ties, masked, infinite and NaN logits, rows with nothing to
choose), the stable sort (exact), rows to their experts and back with their
gradients (dropped slots, odd widths, rows of less than 16 bytes, buffers off any
alignment, rows that no slot has left as they were)."""
import numpy as np
import pytest
import torch

import cme213_amd as M
import moe_ref as R
from gpu_util import dev_t, host, note
from tol import assert_exact

pytestmark = pytest.mark.gpu

GATE_SHAPES = [(1, 1, 1), (1, 8, 2), (3, 2, 2), (17, 16, 16), (5, 33, 4), (64, 64, 6),
               (130, 128, 8), (9, 160, 8), (33, 256, 1), (7, 257, 16), (4, 512, 8), (3, 1000, 3),
               (2, 1024, 16)]
ROW_SHAPES = [(1, 1, 1), (1, 2, 7), (2, 3, 8), (16, 2, 768), (5, 16, 9), (33, 4, 100),
              (257, 2, 769), (64, 8, 1030), (3, 1, 5000), (300, 5, 2050), (70, 9, 33)]


def _logits(n, e, t, seed):
    """Logits on a grid of 1/4, so that many are equal, a fifth of them masked;
    the first rows are the hard ones."""
    r = np.random.default_rng(seed)
    l = np.round(r.standard_normal((n, e)) * 8) / 4
    l[r.random((n, e)) < 0.2] = -np.inf
    hard = [lambda x: x.fill(-np.inf), lambda x: x.fill(0.0), lambda x: x.__setitem__(0, np.nan),
            lambda x: x.__setitem__(e - 1, np.inf),
            lambda x: x.fill(float(torch.finfo(R.TYPES[t]).min)),
            lambda x: (x.fill(-np.inf), x.__setitem__(e // 2, -3.5)),
            lambda x: x.__setitem__(slice(None), np.where(np.arange(e) % 2, -0.0, 0.0))]
    for i, f in enumerate(hard[:max(0, n - 1)]):
        f(l[i])
    return torch.from_numpy(l).to(R.TYPES[t])


def _dev(t):
    return t.contiguous().to("cuda:0")


def _h64(t):
    return host(t.double())


def _rows(r, n, c, t):
    return torch.from_numpy(r.standard_normal((n, c))).to(R.TYPES[t])


def _off(t):
    """The same tensor, one element off the allocation's alignment."""
    b = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda:0")
    v = b[1:].view(t.shape)
    v.copy_(t)
    return v


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,e,k", GATE_SHAPES)
def test_gate_forward(dev, n, e, k, t, renorm):
    note(f"gate forward {n}x{e} k={k} {t} renorm={renorm}")
    l = _logits(n, e, t, n * 1000 + e)
    ids = torch.full((n, k), 77, dtype=torch.int32, device=dev)
    w = torch.full((n, k), 77.0, device=dev)
    M.moe_gate_forward(_dev(l), ids, w, n, e, k, renorm)
    ri, rw, rel = R.gate(l.double().numpy(), k, renorm)
    assert_exact("ids", host(ids), ri)
    R.near("weights", host(w), rw, rel * rw + 2.0 ** -120)


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,e,k", [(4096, 512, 8), (4099, 257, 16)])
def test_gate_of_many_tokens(dev, n, e, k, t, renorm):
    """Between 256 and 512 experts, where many tokens share a wave."""
    test_gate_forward(dev, n, e, k, t, renorm)


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,e,k", GATE_SHAPES)
def test_gate_backward(dev, n, e, k, t, renorm):
    note(f"gate backward {n}x{e} k={k} {t} renorm={renorm}")
    l = _logits(n, e, t, n * 1000 + e + 1)
    ids, w, _ = R.gate(l.double().numpy(), k, renorm)
    w32 = w.astype(np.float32)
    dw = np.random.default_rng(e).standard_normal((n, k)).astype(np.float32)
    dl = torch.full((n, e), 77.0, dtype=R.TYPES[t], device=dev)
    M.moe_gate_backward(None if renorm else _dev(l), dev_t(ids), dev_t(w32), dev_t(dw), dl, n, e,
                        k, renorm)
    ref, bound = R.gate_back(l.double().numpy(), ids, w32.astype(np.float64),
                             dw.astype(np.float64), renorm)
    R.near("dlogits", _h64(dl), ref, bound + R.half_step(t, ref) * (1 + 2.0 ** -10))


def test_gate_gradient_against_differences(dev):
    """The gradient of sum(c * weights), by the backward call and by differences of the
    forward call's weights (step 2^-8: the difference's own error is about h^2 / 6 = 3e-6 and
    the rounding of the weights 2 * 2^-24 / h = 3e-5)."""
    n, e, k = 6, 12, 3
    r = np.random.default_rng(3)
    base = r.permuted(np.tile(np.arange(e), (n, 1)), axis=1) * 0.3  # far from ties
    c = r.standard_normal((n, k)).astype(np.float32)
    for renorm in (True, False):
        def weights(l):
            ids = torch.empty(n, k, dtype=torch.int32, device=dev)
            w = torch.empty(n, k, device=dev)
            M.moe_gate_forward(dev_t(l.astype(np.float32)), ids, w, n, e, k, renorm)
            return ids, w
        ids, w = weights(base)
        dl = torch.empty(n, e, device=dev)
        M.moe_gate_backward(dev_t(base.astype(np.float32)), ids, w, dev_t(c), dl, n, e, k, renorm)
        h = 2.0 ** -8
        num = np.zeros((n, e))
        for j in range(e):
            d = np.zeros((n, e))
            d[:, j] = h
            up, down = host(weights(base + d)[1]), host(weights(base - d)[1])
            num[:, j] = ((up.astype(np.float64) - down) * c).sum(1) / (2 * h)
        R.near(f"renorm={renorm}", host(dl), num, 1e-4 * np.abs(c).sum(1, keepdims=True))


def test_gate_backward_same_expert_twice(dev):
    """Slots that name one expert add up."""
    n, e, k = 5, 20, 4
    r = np.random.default_rng(4)
    l = r.standard_normal((n, e)).astype(np.float32)
    ids = np.tile(np.array([7, 3, 7, -1], np.int32), (n, 1))
    w, dw = r.random((n, k)).astype(np.float32), r.standard_normal((n, k)).astype(np.float32)
    for renorm in (True, False):
        dl = torch.empty(n, e, device=dev)
        M.moe_gate_backward(dev_t(l), dev_t(ids), dev_t(w), dev_t(dw), dl, n, e, k, renorm)
        ref, bound = R.gate_back(l.astype(np.float64), ids, w.astype(np.float64),
                                 dw.astype(np.float64), renorm)
        R.near("dlogits", host(dl), ref, bound + R.half_step("f32", ref))


@pytest.mark.parametrize("experts", [1, 2, 7, 64, 256, 1000, 1024])
@pytest.mark.parametrize("slots", [0, 1, 63, 65, 1000, 4096, 4097, 12289, 300000])
def test_sort(dev, slots, experts):
    note(f"sort {slots} slots, {experts} experts")
    r = np.random.default_rng(slots + experts)
    ids = r.integers(0, experts, slots).astype(np.int32)
    if slots > 10:  # uneven, and some dropped in every way
        ids[r.random(slots) < 0.3] = experts // 2
        ids[r.random(slots) < 0.05] = -1
        ids[3], ids[4], ids[5], ids[6] = experts, 2 ** 31 - 1, -2 ** 31, -7
    off = torch.full((experts + 1,), 77, dtype=torch.int32, device=dev)
    order = torch.full((slots + 1,), 77, dtype=torch.int32, device=dev)
    pos = torch.full((slots + 1,), 77, dtype=torch.int32, device=dev)
    M.moe_sort(dev_t(ids), off, order, pos, slots, experts)
    ro, rorder, rpos = R.sort(ids, experts)
    assert_exact("offsets", host(off), ro)
    assert_exact("position", host(pos)[:slots], rpos)
    assert_exact("order", host(order)[:len(rorder)], rorder)
    assert (host(order)[len(rorder):] == 77).all() and host(pos)[slots] == 77
    again = torch.full((experts + 1,), 78, dtype=torch.int32, device=dev)
    M.moe_sort(dev_t(ids), again, None, pos, slots, experts)
    assert_exact("offsets without order", host(again), ro)


def test_sort_chunks_larger_than_the_least(dev):
    slots, experts = 3_000_001, 130
    note(f"sort {slots} slots")
    ids = np.random.default_rng(9).integers(-1, experts, slots).astype(np.int32)
    off = torch.empty(experts + 1, dtype=torch.int32, device=dev)
    order, pos = (torch.empty(slots, dtype=torch.int32, device=dev) for _ in range(2))
    M.moe_sort(dev_t(ids), off, order, pos, slots, experts)
    ro, rorder, rpos = R.sort(ids, experts)
    assert_exact("offsets", host(off), ro)
    assert_exact("position", host(pos), rpos)
    assert_exact("order", host(order)[:len(rorder)], rorder)


def _positions(r, n, k, drop=0.15):
    """Positions of a sort with dropped slots, and the rows it uses."""
    ids = r.integers(0, 5, n * k).astype(np.int32)
    ids[r.random(n * k) < drop] = -1
    _, order, pos = R.sort(ids, 5)
    return pos, len(order)


@pytest.mark.parametrize("off", [False, True])
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,k,c", ROW_SHAPES)
def test_dispatch(dev, n, k, c, t, off):
    note(f"dispatch {n} tokens k={k} c={c} {t} off={off}")
    r = np.random.default_rng(n * k + c)
    pos, used = _positions(r, n, k)
    rows = max(1, used - 1)  # one row too few: its slot is dropped as well
    put = _off if off else _dev
    x = _rows(r, n, c, t)
    out = put(torch.full((rows + 1, c), 77.0, dtype=R.TYPES[t]))
    P = dev_t(pos)
    M.moe_dispatch_forward(put(x), P, out, n, k, rows, c)
    ref = np.full((rows + 1, c), 77.0)
    for s in range(n * k):
        if R.there(pos[s:s + 1], rows)[0]:
            ref[pos[s]] = x[s // k].double().numpy()
    assert_exact("out", _h64(out), ref)

    g = _rows(r, rows + 1, c, t)
    dx = put(torch.full((n + 1, c), 77.0, dtype=R.TYPES[t]))
    M.moe_dispatch_backward(put(g), P, dx, n, k, rows, c)
    ref, size = R.gather_sum(g.double().numpy(), pos, None, n, k, rows)
    R.near("dx", _h64(dx)[:n], ref, k * R.U * size + R.half_step(t, ref) * (1 + 2.0 ** -10))
    assert (_h64(dx)[n] == 77).all()


@pytest.mark.parametrize("off", [False, True])
@pytest.mark.parametrize("t", list(R.TYPES))
@pytest.mark.parametrize("n,k,c", ROW_SHAPES)
def test_combine(dev, n, k, c, t, off):
    note(f"combine {n} tokens k={k} c={c} {t} off={off}")
    r = np.random.default_rng(n * k + c + 1)
    pos, used = _positions(r, n, k)
    rows = max(1, used - 1)
    put = _off if off else _dev
    y, w = _rows(r, rows + 1, c, t), r.standard_normal((n, k)).astype(np.float32)
    out = put(torch.full((n + 1, c), 77.0, dtype=R.TYPES[t]))
    P, W, Y = dev_t(pos), dev_t(w), put(y)
    M.moe_combine_forward(Y, P, W, out, n, k, rows, c)
    y64, w64 = y.double().numpy(), w.astype(np.float64)
    ref, size = R.gather_sum(y64, pos, w64, n, k, rows)
    R.near("out", _h64(out)[:n], ref, 2 * k * R.U * size + R.half_step(t, ref) * (1 + 2.0 ** -10))
    assert (_h64(out)[n] == 77).all()

    g = _rows(r, n, c, t)
    dy = put(torch.full((rows + 1, c), 77.0, dtype=R.TYPES[t]))
    dw = torch.full((n * k + 1,), 77.0, device=dev)
    M.moe_combine_backward(put(g), Y, P, W, dy, dw, n, k, rows, c)
    g64, rdy, rdw = g.double().numpy(), np.full((rows + 1, c), 77.0), np.zeros((n, k))
    size = np.zeros((n, k))
    for s in range(n * k):
        if R.there(pos[s:s + 1], rows)[0]:
            i, j = s // k, s % k
            rdy[pos[s]] = g64[i] * w64[i, j]
            rdw[i, j] = (g64[i] * y64[pos[s]]).sum()
            size[i, j] = np.abs(g64[i] * y64[pos[s]]).sum()
    R.near("dy", _h64(dy), rdy, R.half_step(t, rdy) * (1 + 2.0 ** -10) + R.U * np.abs(rdy))
    # a lane adds at most c / 64 + 8 products, then six sums over the lanes and
    # a few over waves; each product is rounded
    R.near("dweights", host(dw)[:n * k].reshape(n, k), rdw, (c / 64 + 24) * R.U * size)
    assert host(dw)[n * k] == 77
    # dy in place of y gives the same rows; the products may be added in another order
    # (fewer waves a row), so they are held to the same bound
    dw2 = torch.empty(n * k, device=dev)
    M.moe_combine_backward(put(g), Y, P, W, Y, dw2, n, k, rows, c)
    moved = np.zeros(rows + 1, bool)
    moved[pos[R.there(pos, rows)]] = True
    assert_exact("dy in place", _h64(Y)[moved], _h64(dy)[moved])
    assert_exact("y's other rows", _h64(Y)[~moved], y64[~moved])
    R.near("dweights in place", host(dw2).reshape(n, k), rdw, (c / 64 + 24) * R.U * size)


@pytest.mark.parametrize("n,k,c,t", [(8192, 2, 520, "f32"), (4100, 1, 300, "f32"),
                                     (9000, 2, 1030, "bf16"), (8193, 8, 261, "f16")])
def test_rows_many_tokens(dev, n, k, c, t):
    """Enough tokens that a lane takes several chunks of a row: out against the gather it is,
    and its gradient against the sum over the slots."""
    note(f"rows {n} tokens k={k} c={c} {t}")
    r = np.random.default_rng(n)
    pos, used = _positions(r, n, k, 0.02)
    P, there = dev_t(pos), torch.from_numpy(pos >= 0)
    at = torch.from_numpy(np.maximum(pos, 0)).long()
    x = _rows(r, n, c, t)
    out = torch.zeros(n * k, c, dtype=R.TYPES[t], device=dev)
    M.moe_dispatch_forward(_dev(x), P, out, n, k, n * k, c)
    ref = torch.zeros(n * k, c, dtype=R.TYPES[t])
    ref[at[there]] = x.repeat_interleave(k, 0)[there]
    assert_exact("out", host(out.float()), ref.float().numpy())
    w = torch.from_numpy(r.standard_normal((n, k)).astype(np.float32))
    back = torch.empty(n, c, dtype=R.TYPES[t], device=dev)
    M.moe_combine_forward(out, P, _dev(w), back, n, k, n * k, c)
    wl = torch.where(there.view(n, k), w, 0).double()
    want = (x.double() * wl.sum(1, keepdim=True)).numpy()
    size = (x.double().abs() * wl.abs().sum(1, keepdim=True)).numpy()
    R.near("sum", _h64(back), want, 2 * k * R.U * size + R.half_step(t, want) * (1 + 2.0 ** -10))


@pytest.mark.parametrize("n,k,c,t", [(9001, 2, 2050, "f32"), (4100, 1, 1100, "f32"),
                                     (1500, 2, 700, "f32"), (37, 3, 1500, "f16"),
                                     (1, 2, 20000, "bf16")])
def test_rows_in_segments(dev, n, k, c, t):
    """Rows that several workgroups share, of a number of tokens that fills no last round."""
    test_rows_many_tokens(dev, n, k, c, t)


def test_rows_without_any(dev):
    """No rows at all: dispatch writes nothing, the sums are zero, their gradients too."""
    n, k, c = 7, 2, 40
    pos = torch.zeros(n * k, dtype=torch.int32, device=dev)
    one = torch.zeros(1, c, device=dev)
    w, out = torch.ones(n, k, device=dev), torch.full((n, c), 77.0, device=dev)
    M.moe_dispatch_forward(torch.ones(n, c, device=dev), pos, one, n, k, 0, c)
    assert not host(one).any()
    M.moe_combine_forward(one, pos, w, out, n, k, 0, c)
    assert not host(out).any()
    dw = torch.full((n, k), 77.0, device=dev)
    M.moe_combine_backward(out, one, pos, w, one, dw, n, k, 0, c)
    assert not host(dw).any() and not host(one).any()


def test_rows_non_finite(dev):
    """A NaN or infinity goes where its row goes, times its weight, and nowhere else."""
    n, k, c = 4, 2, 24
    x = np.ones((n, c), np.float32)
    x[1, 3], x[2, 5] = np.nan, np.inf
    pos = np.array([0, 1, 2, -1, 3, 4, -1, 9], np.int32)
    out = torch.zeros(5, c, device=dev)
    M.moe_dispatch_forward(dev_t(x), dev_t(pos), out, n, k, 5, c)
    w = np.array([[1, 2], [3, np.nan], [0.5, 0.25], [np.inf, np.nan]], np.float32)
    back = torch.empty(n, c, device=dev)
    M.moe_combine_forward(out, dev_t(pos), dev_t(w), back, n, k, 5, c)
    ref = x * np.array([3, 3, 0.75, 0], np.float32)[:, None]
    ref[3] = 0  # both of its slots were dropped, their weights with them
    R.near("out", host(back), ref, 0)
