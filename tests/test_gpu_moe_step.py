"""A training step of a block with a mixture of experts, as a program runs it: the residual's
addition and RMS norm, the router with its balance loss, the layer forward and backward, the norm's
gradient into the residual stream's, the gradients of all weights clipped by their global norm into
the optimizer's flat buffer, and Adam.  The products are the caller's (torch).  Each part is checked
against 64 bits of what it was given; the framework's calls are replayed from a graph."""
import numpy as np
import pytest
import torch

import cme213_amd as M
import moe_ref as R
import step_ref as S
from gpu_util import dev_t, host, note
from test_gpu_moe_layer import OUTPUTS, Layer, _reference

pytestmark = pytest.mark.gpu

EPS, COEF, MAX_NORM = 1e-5, 0.02, 1.0


def _h64(t):
    return host(t.double())


class Block:
    """x = a + b; n = rms(x); out = x + experts(n), with the router's logits n @ wr."""

    def __init__(self, n, c, f, e, k, t, seed):
        self.L = L = Layer(n, c, f, e, k, t, M.CKPT8_INT8, seed)
        r = np.random.default_rng(seed + 1)

        def d(a, dtype=torch.float32):
            return torch.from_numpy(a.astype(np.float32)).to(dtype).to("cuda:0")
        self.a, self.b = d(r.standard_normal((n, c)), L.dtype), d(r.standard_normal((n, c)), L.dtype)
        self.gamma, self.wr = d(1 + 0.1 * r.standard_normal(c)), d(r.standard_normal((c, e)) / np.sqrt(c))
        self.valid = d(r.random(n) < 0.9, torch.uint8)
        z = torch.zeros
        kw = {"device": "cuda:0"}
        self.x, self.dstream = z(n, c, dtype=L.dtype, **kw), z(n, c, dtype=L.dtype, **kw)
        self.inv = z(n, **kw)
        self.counts, self.probs, self.loss = z(e + 1, dtype=torch.int32, **kw), z(e, **kw), z(1, **kw)
        self.dn, self.dgamma, self.dwr = z(n, c, dtype=L.dtype, **kw), z(c, **kw), z(c, e, **kw)
        self.q, self.scales = z(n, c, dtype=torch.uint8, **kw), z(n, M.row8_scales(1, c, 128), **kw)
        self.grads = [self.dgamma, self.dwr, L.dw1, L.db1, L.dw2]
        total = sum(g.numel() for g in self.grads)
        self.flat, at, outs = z(total, **kw), 0, []
        for g in self.grads:
            outs.append(self.flat[at:at + g.numel()])
            at += g.numel()
        self.list = M.TensorList(self.grads, outs)
        self.norm_sq, self.clip, self.one = z(1, **kw), z(1, **kw), torch.ones(1, **kw)
        self.param, self.m, self.v = d(r.standard_normal(total)), z(total, **kw), z(total, **kw)

    def norm(self):
        L = self.L
        M.residual_rmsnorm_forward(self.a, self.b, self.gamma, self.x, L.x, self.inv, L.n, L.c, EPS)

    def balance(self):
        L = self.L
        M.moe_balance_forward(L.logits, L.ids, self.valid, self.counts, self.probs, self.loss, L.n,
                              L.e, L.k, COEF)

    def balance_back(self):
        L = self.L
        M.moe_balance_backward(L.logits, self.valid, self.counts, None, L.dlogits, L.n, L.e, L.k,
                               COEF, True)

    def norm_back(self):
        L = self.L
        self.dgamma.fill_(0.0)
        self.dstream.copy_(L.dout)  # the way past the experts
        M.rmsnorm_backward_residual(self.dn, self.x, self.inv, self.gamma, self.dstream, self.dgamma,
                                    L.n, L.c)

    def update(self):
        M.tensors_clip(self.list, MAX_NORM, self.norm_sq, self.clip)
        M.adam_clipped(self.param, self.flat, self.m, self.v, self.one, 1e-3, 0.9, 0.95, 1e-8, 0.1,
                       0.05, 1.0, self.flat.numel())

    def step(self):
        L = self.L
        self.norm()
        L.logits.copy_(L.x.float() @ self.wr)
        L.route()
        self.balance()
        ends = L.offsets.tolist()
        L.forward(ends)
        L.backward(ends)
        self.routed = L.dlogits.clone()  # the router's own gradient
        self.balance_back()
        self.dwr.copy_(L.x.float().t().contiguous() @ L.dlogits)
        self.dn.copy_(L.dx.float() + L.dlogits @ self.wr.t().contiguous())
        self.norm_back()
        self.update()


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,c,f,e,k", [(96, 48, 80, 5, 2), (1, 64, 128, 8, 2), (300, 72, 200, 16, 4)])
def test_step(dev, n, c, f, e, k, t):
    note(f"moe step {n}x{c}x{f} e={e} k={k} {t}")
    B = Block(n, c, f, e, k, t, n + c)
    L = B.L
    before = _h64(B.param)
    B.step()
    # the norm
    x, r, y, rel_r, rel_y = S.rms(_h64(B.a), _h64(B.b), _h64(B.gamma), EPS)
    R.near("x", _h64(B.x), x, S.U * np.abs(x) + R.half_step(t, x) * (1 + 2.0 ** -9))
    R.near("inv", _h64(B.inv), r, rel_r * r)
    R.near("n", _h64(L.x), y, rel_y * np.abs(y) * (1 + 2.0 ** -7) + R.half_step(t, y) * (1 + 2.0 ** -9))
    # the layer, by the bound of its own test
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[t]
    full = L.dlogits
    L.dlogits = B.routed
    ref, ids = _reference(L)
    for name in OUTPUTS:
        got = _h64(getattr(L, name))
        rel = np.linalg.norm(got - ref[name]) / max(np.linalg.norm(ref[name]), 1e-300)
        assert rel <= 7 * half + 200 * S.U, (name, rel)
    L.dlogits = full
    # the balance loss and its gradient on top of the router's
    l = _h64(L.logits)
    counts, probs, p_bound, loss, l_bound = S.balance(l, ids, host(B.valid), k, COEF)
    assert np.array_equal(host(B.counts), counts)
    R.near("probs", _h64(B.probs), probs, p_bound)
    R.near("loss", _h64(B.loss), [loss], [l_bound])
    g, g_bound = S.balance_back(l, host(B.valid), counts, 1.0, k, COEF)
    both = _h64(B.routed) + g
    R.near("dlogits", _h64(full), both, g_bound + 2 * S.U * np.abs(both))
    # the norm's gradient onto the residual stream's
    dx, bound, dg, dg_bound = S.rms_back(_h64(B.dn), _h64(B.x), _h64(B.inv), _h64(B.gamma), _h64(L.dout))
    R.near("dstream", _h64(B.dstream), dx, bound + R.half_step(t, dx) * (1 + 2.0 ** -9))
    R.near("dgamma", _h64(B.dgamma), dg, dg_bound + S.U * np.abs(dg))
    # clipping and Adam
    grads = np.concatenate([_h64(x).reshape(-1) for x in B.grads])
    want = (grads ** 2).sum()
    rel = (S.norm_chain(grads.size) + 4) * S.U
    assert abs(_h64(B.norm_sq)[0] - want) <= rel * want
    scale = min(1.0, MAX_NORM / np.sqrt(want))
    assert abs(_h64(B.clip)[0] - scale) <= (rel / 2 + 3 * S.U) * scale
    R.near("flat", _h64(B.flat), grads * _h64(B.clip)[0], S.U * np.abs(grads))
    flat = _h64(B.flat)
    m, v = np.float32(1 - np.float32(0.9)) * flat, np.float32(1 - np.float32(0.95)) * flat * flat
    step = np.float32(1e-3) * (m / np.float32(0.1)) / (np.sqrt(v / np.float32(0.05)) + np.float32(1e-8))
    # some ten roundings of the step, one of the parameter
    R.near("param", _h64(B.param), before - step, 12 * S.U * np.abs(step) + S.U * np.abs(before) +
           1e-12)


def test_step_replayed_from_a_graph(dev):
    """The framework's calls of a step, captured (the products' buffers stay as they are): every
    replay gives the eager calls' bits, with eager steps between the replays."""
    B = Block(2100, 128, 96, 6, 2, "bf16", 7)
    L = B.L
    M.workspace_reserve(32 << 20)
    B.step()
    param, m, v = B.param.clone(), B.m.clone(), B.v.clone()
    router = L.dlogits.clone()

    def calls():
        for a, b in ((B.param, param), (B.m, m), (B.v, v), (L.dlogits, router)):
            a.copy_(b)
        B.norm()
        L.route()
        B.balance()
        B.balance_back()
        B.norm_back()
        M.rmsnorm_forward_row8(B.x, B.gamma, B.q, B.scales, None, None, L.n, L.c, EPS, 128)
        B.update()
    names = [B.x, L.x, B.inv, L.ids, L.weights, B.counts, B.probs, B.loss, L.dlogits, B.dstream,
             B.dgamma, B.q, B.scales, B.norm_sq, B.clip, B.flat, B.param, B.m, B.v]
    calls()
    torch.cuda.synchronize()
    ref = [x.clone() for x in names]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for rep in range(3):
        for x in names:
            x.fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(names, ref)), rep
        B.step()
        calls()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(names, ref)), rep


def test_two_graphs_share_the_workspace(dev):
    """Two captured graphs of different shapes, replayed one after the other in either order:
    what one leaves in the workspace does not reach the other."""
    M.workspace_reserve(32 << 20)
    graphs = []
    for n, c, e, k, count in ((3000, 200, 24, 3, 300), (9001, 72, 160, 8, 500)):
        r = np.random.default_rng(n)

        def d(*shape, scale=1.0):
            return dev_t((r.standard_normal(shape) * scale).astype(np.float32))
        x, dy, gamma, logits = d(n, c), d(n, c), d(c), d(n, e)
        ids = dev_t(r.integers(0, e, (n, k)).astype(np.int32))
        grads = [d(1 + i * 97 % 500) for i in range(count)]
        flat = torch.zeros(sum(g.numel() for g in grads), device=dev)
        tensors = M.TensorList(grads, list(flat.split([g.numel() for g in grads])))
        inv, dx, dg, dl = torch.ones(n, device=dev), torch.empty_like(x), torch.empty(c, device=dev), torch.empty_like(logits)
        counts, probs = torch.empty(e + 1, dtype=torch.int32, device=dev), torch.empty(e, device=dev)
        loss, n2, clip = torch.empty(3, 1, device=dev)

        def step(n=n, c=c, e=e, k=k, x=x, dy=dy, gamma=gamma, logits=logits, ids=ids, tensors=tensors,
                 inv=inv, dx=dx, dg=dg, dl=dl, counts=counts, probs=probs, loss=loss, n2=n2, clip=clip):
            dg.fill_(0.0)
            M.rmsnorm_backward(dy, x, inv, gamma, dx, dg, n, c)
            M.moe_balance_forward(logits, ids, None, counts, probs, loss, n, e, k, COEF)
            M.moe_balance_backward(logits, None, counts, loss, dl, n, e, k, COEF, False)
            M.tensors_clip(tensors, 1.0, n2, clip)
        step()
        torch.cuda.synchronize()
        results = [dx, dg, dl, counts, probs, loss, n2, clip, flat]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append((graph, results, [t.clone() for t in results], step))
    for order in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for _, results, _, _ in graphs:
            for t in results:
                t.fill_(1)
        for i in order:
            graphs[i][0].replay()
        torch.cuda.synchronize()
        for _, results, want, step in graphs:
            assert all(torch.equal(t, w) for t, w in zip(results, want)), order
            step()
        torch.cuda.synchronize()
        for _, results, want, _ in graphs:
            assert all(torch.equal(t, w) for t, w in zip(results, want)), order
