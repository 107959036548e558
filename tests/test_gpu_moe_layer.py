"""A whole mixture-of-experts feed-forward layer, forward and backward, as a program
runs it: router, sort, dispatch, a product per expert, bias + GELU with an 8-bit
checkpoint, a product per expert, combine, and the way back.  The products are the
caller's (torch, one per expert).  Checked against the layer written out in 64 bits on
the host, whose backward pass reads the checkpoint's values too; replayed from a graph;
and on another stream than the default one."""
import numpy as np
import pytest
import torch

import cme213_amd as M
import moe_ref as R
from gpu_util import host, note
from tol import assert_exact

pytestmark = pytest.mark.gpu


class Layer:
    """Buffers and calls of one layer; the products take host-side row ranges."""

    def __init__(self, n, c, f, e, k, t, fmt, seed):
        self.n, self.c, self.f, self.e, self.k, self.fmt = n, c, f, e, k, fmt
        self.dtype, self.rows = R.TYPES[t], n * k
        r = np.random.default_rng(seed)

        def d(a, dtype=torch.float32):
            return torch.from_numpy(a.astype(np.float32)).to(dtype).to("cuda:0")
        self.x, self.dout = d(r.standard_normal((n, c)), self.dtype), d(r.standard_normal((n, c)),
                                                                       self.dtype)
        self.logits = d(r.standard_normal((n, e)) * 1.5)
        self.w1 = d(r.standard_normal((e, c, f)) / np.sqrt(c), self.dtype)
        self.w2 = d(r.standard_normal((e, f, c)) / np.sqrt(f), self.dtype)
        self.b1 = d(r.standard_normal((e, f)) * 0.2)

        def z(*shape, dtype=self.dtype):
            return torch.zeros(shape, dtype=dtype, device="cuda:0")
        i32, f32, u8 = torch.int32, torch.float32, torch.uint8
        self.ids, self.weights = z(n, k, dtype=i32), z(n, k, dtype=f32)
        self.offsets, self.order = z(e + 1, dtype=i32), z(self.rows, dtype=i32)
        self.position = z(self.rows, dtype=i32)
        self.xs, self.h, self.a = z(self.rows, c), z(self.rows, f), z(self.rows, f)
        self.q, self.s = z(self.rows, f, dtype=u8), z(self.rows, -(-f // 32), dtype=u8)
        self.y, self.out = z(self.rows, c), z(n, c)
        self.dy, self.dweights = z(self.rows, c), z(n, k, dtype=f32)
        self.da, self.dh, self.act = z(self.rows, f), z(self.rows, f), z(self.rows, f)
        self.dxs, self.dx, self.dlogits = z(self.rows, c), z(n, c), z(n, e, dtype=f32)
        self.db1 = z(e, f, dtype=f32)
        self.dw1, self.dw2 = torch.zeros_like(self.w1), torch.zeros_like(self.w2)

    def route(self):
        M.moe_gate_forward(self.logits, self.ids, self.weights, self.n, self.e, self.k)
        M.moe_sort(self.ids, self.offsets, self.order, self.position, self.rows, self.e)
        M.moe_dispatch_forward(self.x, self.position, self.xs, self.n, self.k, self.rows, self.c)

    def products(self, src, w, dst, ends):
        for i in range(self.e):
            a, b = ends[i], ends[i + 1]
            if b > a:
                torch.mm(src[a:b], w[i], out=dst[a:b])

    def forward(self, ends):
        self.products(self.xs, self.w1, self.h, ends)
        M.bias_gelu_forward_ckpt8(self.h, self.b1, self.offsets, self.a, self.q, self.s,
                                  self.rows, self.f, self.e, self.fmt)
        self.products(self.a, self.w2, self.y, ends)
        M.moe_combine_forward(self.y, self.position, self.weights, self.out, self.n, self.k,
                              self.rows, self.c)

    def backward(self, ends):
        self.db1.fill_(0.0)
        M.moe_combine_backward(self.dout, self.y, self.position, self.weights, self.dy,
                               self.dweights, self.n, self.k, self.rows, self.c)
        self.products(self.dy, self.w2.transpose(1, 2).contiguous(), self.da, ends)
        M.gelu_backward_with_bias_backward_ckpt8(self.q, self.s, self.b1, self.offsets, self.da,
                                                 self.dh, self.act, self.db1, self.rows, self.f,
                                                 self.e, self.fmt)
        for i in range(self.e):
            a, b = ends[i], ends[i + 1]
            torch.mm(self.act[a:b].t().contiguous(), self.dy[a:b], out=self.dw2[i])
            torch.mm(self.xs[a:b].t().contiguous(), self.dh[a:b], out=self.dw1[i])
        self.products(self.dh, self.w1.transpose(1, 2).contiguous(), self.dxs, ends)
        M.moe_dispatch_backward(self.dxs, self.position, self.dx, self.n, self.k, self.rows, self.c)
        M.moe_gate_backward(self.logits, self.ids, self.weights, self.dweights, self.dlogits,
                            self.n, self.e, self.k)

    def run(self):
        self.route()
        ends = self.offsets.tolist()
        self.forward(ends)
        self.backward(ends)
        return ends


OUTPUTS = ("out", "dx", "dlogits", "db1", "dw1", "dw2")


def _reference(L):
    """The layer written out in 64 bits, slot by expert; the checkpoint's values stand for the
    hidden rows wherever the backward pass uses them."""
    def h(t):
        return t.double().cpu().numpy()
    x, dout, logits = h(L.x), h(L.dout), h(L.logits)
    w1, w2, b1 = h(L.w1), h(L.w2), h(L.b1)
    ids, w, _ = R.gate(logits, L.k, True)
    r = {"out": np.zeros((L.n, L.c)), "dx": np.zeros((L.n, L.c)), "db1": np.zeros_like(b1),
         "dw1": np.zeros_like(w1), "dw2": np.zeros_like(w2)}
    dw = np.zeros_like(w)
    fmt = {M.CKPT8_INT8: "int8", M.CKPT8_E4M3: "e4m3"}[L.fmt]
    kept = R.from_ckpt8(host(L.q), host(L.s), fmt)  # of the rows as the layer computed them
    position = host(L.position).reshape(L.n, L.k)
    for e in range(L.e):
        t, j = np.nonzero(ids == e)
        if not len(t):
            continue
        wt = w[t, j][:, None]
        y = R.gelu(x[t] @ w1[e] + b1[e])[0] @ w2[e]
        np.add.at(r["out"], t, wt * y)
        a, slope = R.gelu(kept[position[t, j]] + b1[e])
        dy = wt * dout[t]
        dw[t, j] = (dout[t] * y).sum(1)
        dh = (dy @ w2[e].T) * slope
        r["dw2"][e], r["dw1"][e], r["db1"][e] = a.T @ dy, x[t].T @ dh, dh.sum(0)
        np.add.at(r["dx"], t, dh @ w1[e].T)
    r["dlogits"] = R.gate_back(logits, ids, w, dw, True)[0]
    return r, ids


@pytest.mark.parametrize("t,fmt", [("f32", M.CKPT8_INT8), ("f32", M.CKPT8_E4M3),
                                   ("bf16", M.CKPT8_INT8), ("f16", M.CKPT8_E4M3)])
@pytest.mark.parametrize("n,c,f,e,k", [(96, 48, 80, 5, 2), (1, 64, 128, 8, 2), (130, 72, 200, 16, 4)])
def test_layer(dev, n, c, f, e, k, t, fmt):
    note(f"moe layer {n}x{c}x{f} e={e} k={k} {t} {fmt}")
    L = Layer(n, c, f, e, k, t, fmt, n + c)
    L.run()
    ref, ids = _reference(L)
    assert_exact("ids", host(L.ids), ids)
    # Relative 2-norm of each output.  Every stored intermediate (xs exact; h, a, y,
    # da, dh, dy rounded to the row type: at most six of them on any path) is off by half a
    # step of its type, and products of sums of 200 fp32 terms by less than 200 U; the two
    # products' own roundings are among the six.  Independent errors would add as
    # sqrt(6), taken here as 6, and the output's own rounding once.
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[t]
    for name in OUTPUTS:
        got = getattr(L, name).double().cpu().numpy()
        rel = np.linalg.norm(got - ref[name]) / max(np.linalg.norm(ref[name]), 1e-300)
        assert rel <= 7 * half + 200 * R.U, (name, rel)


def test_layer_replayed_from_a_graph(dev):
    """The captured layer, replayed, gives the eager layer's bits in every output, with eager
    runs between the replays (more than 4096 slots: the sort uses the workspace)."""
    L = Layer(2100, 64, 96, 6, 2, "bf16", M.CKPT8_INT8, 7)
    M.workspace_reserve(32 << 20)
    ends = L.run()
    names = ["ids", "weights", "offsets", "order", "position", "xs", "a", "q", "s", "out", "dy",
             "dweights", "dh", "act", "dx", "dlogits", "db1"]
    own = [n for n in names if n not in ("q", "s", "order")]

    def calls():  # the framework's calls alone: the products' buffers stay as they are
        L.route()
        M.bias_gelu_forward_ckpt8(L.h, L.b1, L.offsets, L.a, L.q, L.s, L.rows, L.f, L.e, L.fmt)
        M.moe_combine_forward(L.y, L.position, L.weights, L.out, L.n, L.k, L.rows, L.c)
        L.db1.fill_(0.0)
        M.moe_combine_backward(L.dout, L.y, L.position, L.weights, L.dy, L.dweights, L.n, L.k,
                               L.rows, L.c)
        M.gelu_backward_with_bias_backward_ckpt8(L.q, L.s, L.b1, L.offsets, L.da, L.dh, L.act,
                                                 L.db1, L.rows, L.f, L.e, L.fmt)
        M.moe_dispatch_backward(L.dxs, L.position, L.dx, L.n, L.k, L.rows, L.c)
        M.moe_gate_backward(L.logits, L.ids, L.weights, L.dweights, L.dlogits, L.n, L.e, L.k)

    calls()
    torch.cuda.synchronize()
    ref = {n: host(getattr(L, n).float()) for n in names}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for n in names:  # and on another stream
        assert_exact(f"side stream {n}", host(getattr(L, n).float()), ref[n])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    torch.cuda.synchronize()
    for rep in range(3):
        for n in own:
            getattr(L, n).fill_(7)
        L.q.fill_(7), L.s.fill_(7), L.order.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for n in names:
            assert_exact(f"replay {rep} {n}", host(getattr(L, n).float()), ref[n])
        L.run()  # eager work between replays
        torch.cuda.synchronize()
        calls()
        torch.cuda.synchronize()
        for n in names:
            assert_exact(f"eager after replay {rep} {n}", host(getattr(L, n).float()), ref[n])
    assert ends[-1] == L.rows


def test_workspace_is_not_grown_under_capture(dev):
    """A capture that would need a larger workspace is refused before anything is launched,
    and the capture goes on."""
    slots, e = 300000, 1000
    ids = torch.zeros(slots, dtype=torch.int32, device=dev)
    off = torch.zeros(e + 1, dtype=torch.int32, device=dev)
    pos = torch.zeros(slots, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    M.workspace_release()
    assert M.workspace_bytes() == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(M.MIError) as err:
            M.moe_sort(ids, off, None, pos, slots, e)
        assert err.value.code == M.MI_ERR_CAPTURE_ALLOC
        off.fill_(3)
    graph.replay()
    torch.cuda.synchronize()
    assert (host(off) == 3).all() and M.workspace_bytes() == 0
    M.moe_sort(ids, off, None, pos, slots, e)
    assert M.workspace_bytes() >= M.lib.mi_moe_sort_workspace(slots, e)
    want = np.full(e + 1, slots)
    want[0] = 0
    assert_exact("offsets", host(off), want.astype(np.int32))


def test_calls_refuse_what_they_cannot_take(dev):
    """Tensors of the wrong type, size, layout or device are refused by the wrappers."""
    x = torch.zeros(4, 8, device=dev)
    pos, w = torch.zeros(8, dtype=torch.int32, device=dev), torch.zeros(4, 2, device=dev)
    out = torch.zeros(8, 8, device=dev)
    with pytest.raises(ValueError, match="dtype"):
        M.moe_dispatch_forward(x, pos, out.half(), 4, 2, 8, 8)
    with pytest.raises(ValueError, match="dtype"):
        M.moe_dispatch_forward(x, pos.long(), out, 4, 2, 8, 8)
    with pytest.raises(ValueError, match="at least 64"):
        M.moe_dispatch_forward(x, pos, out[:7], 4, 2, 8, 8)
    with pytest.raises(ValueError, match="contiguous"):
        M.moe_combine_forward(out.t(), pos, w, x, 4, 2, 8, 8)
    q, s = torch.zeros(4, 8, dtype=torch.uint8, device=dev), torch.zeros(4, 1, dtype=torch.uint8,
                                                                        device=dev)
    with pytest.raises(ValueError, match="dtype"):
        M.float_to_ckpt8(x, q.view(torch.int8), s, 4, 8, M.CKPT8_E4M3)
    with pytest.raises(ValueError, match="at least 4"):
        M.float_to_ckpt8(x, q, s[:3], 4, 8)
    M.float_to_ckpt8(x, q.view(torch.int8), s, 4, 8)
    M.float_to_ckpt8(x, q.view(torch.float8_e4m3fn), s, 4, 8, M.CKPT8_E4M3)
    current = M._current_device
    try:
        M._current_device = lambda: 1  # as if another device were the current one
        with pytest.raises(ValueError, match="the current device is cuda:1"):
            M.float_to_ckpt8(x, q, s, 4, 8)
    finally:
        M._current_device = current
    big = torch.zeros(2001, dtype=torch.int32, device=dev)
    with pytest.raises(M.MIError, match="experts"):
        M.moe_sort(pos, big, None, pos, 4, 2000)


def test_rows_past_2_31_elements(dev):
    """Element numbers past 2^31 and byte offsets past 2^32: the first and last tokens of a
    dispatch, a combine and their gradients against the rows they are made of."""
    n, k, c = 1_100_003, 2, 1000
    note(f"rows {n}x{c} k={k}")
    rows = n * k
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n, c, device=dev, generator=gen, dtype=torch.bfloat16)
    pos = torch.randperm(rows, device=dev, generator=gen).to(torch.int32)
    w = torch.rand(n, k, device=dev, generator=gen)
    xs = torch.empty(rows, c, device=dev, dtype=torch.bfloat16)
    M.moe_dispatch_forward(x, pos, xs, n, k, rows, c)
    at = pos.view(n, k).long()
    for part in (slice(0, 70), slice(n // 2, n // 2 + 70), slice(n - 70, n)):
        for j in range(k):
            assert torch.equal(xs[at[part, j]], x[part])
    back = torch.empty_like(x)
    M.moe_combine_forward(xs, pos, w, back, n, k, rows, c)
    dy, dw = torch.empty_like(xs), torch.empty(n, k, device=dev)
    M.moe_combine_backward(x, xs, pos, w, dy, dw, n, k, rows, c)
    for part in (slice(0, 70), slice(n - 70, n)):
        x64, w64 = x[part].double(), w[part].double()
        want = x64 * w64.sum(1, keepdim=True)
        R.near("out", host(back[part].double()), host(want),
               host(want.abs()) * (2.0 ** -8 + 8 * R.U))
        sq = (x64 * x64).sum(1, keepdim=True)
        R.near("dweights", host(dw[part]), host(sq.expand(-1, k)), host(sq) * (c / 64 + 24) * R.U)
        for j in range(k):
            want = x64 * w64[:, j:j + 1]
            R.near("dy", host(dy[at[part, j]].double()), host(want), host(want.abs()) * 2.0 ** -7.99)


def test_checkpoint_past_2_31_elements(dev):
    rows, cols = 2_100_001, 1040
    note(f"checkpoint {rows}x{cols}")
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(rows, cols, device=dev, generator=gen, dtype=torch.bfloat16)
    q = torch.empty(rows, cols, dtype=torch.uint8, device=dev)
    s = torch.empty(rows, -(-cols // 32), dtype=torch.uint8, device=dev)
    out, b = torch.empty_like(x), torch.zeros(2, cols, device=dev)
    off = torch.tensor([0, rows - 50, rows], dtype=torch.int32, device=dev)
    M.bias_gelu_forward_ckpt8(x, b, off, out, q, s, rows, cols, 2)
    gin, db = torch.empty_like(x), torch.zeros(2, cols, device=dev)
    M.gelu_backward_with_bias_backward_ckpt8(q, s, b, off, x, gin, None, db, rows, cols, 2)
    back = torch.empty_like(x)
    M.ckpt8_to_float(q, s, back, rows, cols)
    for part in (slice(0, 60), slice(rows - 60, rows)):
        x64 = host(x[part].double())
        rq, rs = R.to_ckpt8(x64, "int8")
        assert_exact("codes", host(q[part]), rq)
        assert_exact("scales", host(s[part]), rs)
        kept = R.from_ckpt8(rq, rs, "int8")
        assert_exact("values", host(back[part].double()),
                     host(torch.from_numpy(kept).to(torch.bfloat16).double()))
        y = R.gelu(x64)[0]
        R.near("out", host(out[part].double()), y, np.abs(y) * (2.0 ** -8 + 1e-5) + 1e-6)
        g = x64 * R.gelu(kept)[1]
        R.near("grad_in", host(gin[part].double()), g,
               np.abs(g) * 2.0 ** -8 + np.abs(x64) * 1e-4 + 1e-38)
        if part.start:
            last = g[-50:]
            R.near("dbias", host(db[1]), last.sum(0), 1e-4 * np.sqrt((last ** 2).sum(0)) + 1e-5)


@pytest.mark.parametrize("n,c", [(17_000_003, 8), (4_300_001, 264)])
def test_more_tokens_than_the_grid_has_room_for(dev, n, c):
    """Tokens past the workgroups of one launch are taken in strides: the router (17 million
    rows) and one choice's rows there and back, by an index that reverses them."""
    note(f"{n} tokens of {c}")
    gen = torch.Generator(device="cuda").manual_seed(4)
    if c == 8:
        l = torch.randn(n, 2, device=dev, generator=gen, dtype=torch.float16)
        ids = torch.empty(n, 1, dtype=torch.int32, device=dev)
        w = torch.empty(n, 1, device=dev)
        M.moe_gate_forward(l, ids, w, n, 2, 1, False)
        lf = l.float()
        assert torch.equal(ids[:, 0], (lf[:, 1] > lf[:, 0]).int())
        p = torch.softmax(lf, 1)
        assert (w[:, 0] - p.amax(1)).abs().max() <= 16 * R.U
        dl, dw = torch.empty_like(l), torch.ones(n, 1, device=dev)
        M.moe_gate_backward(l, ids, w, dw, dl, n, 2, 1, False)
        # p (1 - p) up to its own rounding and fp16's
        want = (p[:, 0] * p[:, 1]) * torch.where(ids[:, 0] == 0, 1.0, -1.0)
        assert (dl[:, 0].float() - want).abs().max() <= 0.25 * 2.0 ** -11 + 32 * R.U
    x = torch.randn(n, c, device=dev, generator=gen, dtype=torch.bfloat16)
    pos = torch.arange(n - 1, -1, -1, dtype=torch.int32, device=dev)
    out, one = torch.empty_like(x), torch.ones(n, 1, device=dev)
    M.moe_dispatch_forward(x, pos, out, n, 1, n, c)
    assert torch.equal(out, x.flip(0))
    back = torch.empty_like(x)
    M.moe_dispatch_backward(out, pos, back, n, 1, n, c)
    assert torch.equal(back, x)
    M.moe_combine_forward(out, pos, one, back.zero_(), n, 1, n, c)
    assert torch.equal(back, x)
    dw = torch.empty(n, 1, device=dev)
    M.moe_combine_backward(x, out, pos, one, out, dw, n, 1, n, c)
    assert torch.equal(out, x.flip(0))
    want = torch.empty(n, device=dev)
    for i in range(0, n, 1 << 20):
        want[i:i + (1 << 20)] = x[i:i + (1 << 20)].double().square().sum(1)
    assert ((dw[:, 0] - want).abs() <= (c / 64 + 24) * R.U * want).all()


def test_narrow_rows_of_many_tokens(dev):
    """Rows of less than 16 bytes, one thread a token, past one launch's first million."""
    n, k, c = 3_000_001, 2, 3
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(n, c, device=dev, generator=gen)
    pos = torch.randperm(n * k, device=dev, generator=gen).to(torch.int32)
    out = torch.empty(n * k, c, device=dev)
    M.moe_dispatch_forward(x, pos, out, n, k, n * k, c)
    assert torch.equal(out[pos.view(n, k)[:, 1].long()], x)
    w = torch.full((n, k), 0.5, device=dev)
    back = torch.empty_like(x)
    M.moe_combine_forward(out, pos, w, back, n, k, n * k, c)
    assert torch.equal(back, x)
