"""GPU parity of the calls on many tensors (norm, scaling, clipping) against 64 bits:
lists of one to hundreds of tensors of three types, empty ones and single elements among
them, off any alignment, in place and into fp32, norms below and above the limit, at it,
infinite and NaN."""
import numpy as np
import pytest
import torch

import cme213_amd as M
import moe_ref as R
import step_ref as S
from gpu_util import host, note

pytestmark = pytest.mark.gpu

# elements of each tensor: around the unit of 8192 and a step of 1024 or 2048
LISTS = {"one": [1], "none": [0], "empty": [], "odd": [7, 0, 1, 8191, 8192, 8193, 3, 0],
         "one large": [300_001], "many": [5 + 37 * i % 3000 for i in range(500)],
         "a batch with outs": [100] * 192, "and one": [100] * 193, "a batch": [100] * 320,
         "a batch and one": [100] * 321, "three batches": [1 + 53 * i % 700 for i in range(700)],
         "batches, large": [40_000 + 97 * i for i in range(400)], "mixed": [1 << 20, 5, 99_999, 17, 1025] * 7}


def _h64(t):
    return host(t.double())


def _tensors(sizes, seed, scale=1.0, types=("f32", "bf16", "f16")):
    """Tensors at odd places of one buffer for each type, with 77 around them."""
    r = np.random.default_rng(seed)
    got, guards = [], {}
    for t in types:
        mine = [i for i in range(len(sizes)) if types[i % len(types)] == t]
        room = sum(sizes[i] + 1 for i in mine) + 1
        guards[t] = torch.full((room,), 77.0, dtype=R.TYPES[t], device="cuda:0")
    at = dict.fromkeys(types, 1)
    for i, n in enumerate(sizes):
        t = types[i % len(types)]
        v = guards[t][at[t]:at[t] + n]
        v.copy_(torch.from_numpy(r.standard_normal(n) * scale).to(R.TYPES[t]))
        at[t] += n + 1
        got.append(v)
    return got, guards


def _norm_sq(tensors):
    return sum(float((_h64(x) ** 2).sum()) for x in tensors)


def _one(v):
    return torch.full((1,), float(v), device="cuda:0")


def _type(x):
    return {v: k for k, v in R.TYPES.items()}[x.dtype]


@pytest.mark.parametrize("name", list(LISTS))
def test_norm_sq(dev, name):
    note(f"tensors norm {name}")
    xs, _ = _tensors(LISTS[name], 1)
    want, total = _norm_sq(xs), sum(LISTS[name])
    rel = (S.norm_chain(total) + 4) * S.U
    got = _one(3.0)
    M.tensors_norm_sq_acc(M.TensorList(xs), got)
    assert abs(host(got)[0] - (want + 3)) <= rel * want + 2 * S.U * (want + 3)
    first = host(got)[0]
    got = _one(3.0)
    M.tensors_norm_sq_acc(M.TensorList(xs), got)
    assert host(got)[0] == first


@pytest.mark.parametrize("where", ["inplace", "elsewhere"])
@pytest.mark.parametrize("scale", [0.37, 1.0, 0.0, -2.5])
@pytest.mark.parametrize("name", list(LISTS))
def test_scale(dev, name, scale, where):
    note(f"tensors scale {name} {scale} {where}")
    xs, guards = _tensors(LISTS[name], 2)
    before = [x.clone() for x in xs]
    s32 = float(np.float32(scale))
    if where == "inplace":
        M.tensors_scale(M.TensorList(xs), _one(scale))
        for x, b in zip(xs, before):
            # the product in fp32, rounded to the type
            want = (b.float() * _one(scale)).to(b.dtype)
            assert torch.equal(x, want)
        for t, n in ((t, sum(LISTS[name][i] for i in range(len(xs)) if i % 3 == j))
                     for j, t in enumerate(guards)):
            assert int((guards[t] == 77).sum()) >= guards[t].numel() - n
    else:
        flat = torch.full((sum(LISTS[name]) + 2,), 77.0, device=dev)
        outs, at = [], 1
        for x in xs:
            outs.append(flat[at:at + x.numel()])
            at += x.numel()
        M.tensors_scale(M.TensorList(xs, outs), _one(scale))
        for x, b, o in zip(xs, before, outs):
            assert torch.equal(x, b) and torch.equal(o, b.float() * s32)
        assert flat[0] == 77 and flat[-1] == 77


@pytest.mark.parametrize("where", ["inplace", "elsewhere"])
@pytest.mark.parametrize("limit", [0.5, 2.0, 0.0])
@pytest.mark.parametrize("name", list(LISTS))
def test_clip(dev, name, limit, where):
    """The limit as a multiple of the norm."""
    note(f"tensors clip {name} {limit} {where}")
    xs, _ = _tensors(LISTS[name], 3)
    before = [x.clone() for x in xs]
    want = _norm_sq(xs)
    max_norm = float(np.float32(limit * np.sqrt(want)))
    outs = [torch.full((x.numel(),), 77.0, device=dev) for x in xs] if where == "elsewhere" else None
    n2, c = _one(77), _one(77)
    M.tensors_clip(M.TensorList(xs, outs), max_norm, n2, c)
    rel = (S.norm_chain(sum(LISTS[name])) + 4) * S.U
    assert abs(host(n2)[0] - want) <= rel * want
    scale = limit if limit < 1 and want > 0 else 1.0
    # half the norm's error, the root and the division
    assert abs(host(c)[0] - scale) <= (rel / 2 + 3 * S.U) * scale
    if scale == 1.0:
        assert host(c)[0] == 1.0
    for i, (x, b) in enumerate(zip(xs, before)):
        if outs is not None:
            assert torch.equal(x, b) and torch.equal(outs[i], b.float() * c)
        else:
            assert torch.equal(x, (b.float() * c).to(b.dtype))


def test_the_limit_itself(dev):
    x = torch.full((4,), 0.5, device=dev)  # norm 1, exactly
    n2, c = _one(0), _one(0)
    M.tensors_clip(M.TensorList([x]), 1.0, n2, c)
    assert host(n2)[0] == 1 and host(c)[0] == 1 and (host(x) == 0.5).all()


@pytest.mark.parametrize("bad,norm,scale", [(np.inf, np.inf, 0.0), (np.nan, np.nan, 1.0)])
def test_infinity_and_nan(dev, bad, norm, scale):
    """As compute_clip_scale has it: an infinite norm gives the scale 0, a NaN the scale 1."""
    xs, _ = _tensors([100, 20_000, 5], 4)
    xs[1][7] = bad
    before = [x.clone() for x in xs]
    n2, c = _one(0), _one(0)
    M.tensors_clip(M.TensorList(xs), 1.0, n2, c)
    assert host(c)[0] == scale and (np.isnan(host(n2)[0]) if np.isnan(norm) else host(n2)[0] == norm)
    for x, b in zip(xs, before):
        assert torch.equal(torch.nan_to_num(x.float(), 9.0), torch.nan_to_num(b.float() * scale, 9.0))


def test_wide_range(dev):
    """fp16's and bf16's largest and smallest values: the squares are formed in fp32."""
    big = torch.full((1000,), 65504.0, dtype=torch.float16, device=dev)
    tiny = torch.full((1000,), 2.0 ** -24, dtype=torch.float16, device=dev)
    n2 = _one(0)
    M.tensors_norm_sq_acc(M.TensorList([big, tiny]), n2)
    want = 1000 * 65504.0 ** 2
    assert abs(host(n2)[0] - want) <= 50 * S.U * want
    n2 = _one(0)
    M.tensors_norm_sq_acc(M.TensorList([tiny]), n2)
    want = 1000 * 2.0 ** -48
    assert abs(host(n2)[0] - want) <= 50 * S.U * want


def test_views_and_refused_lists(dev):
    x = torch.zeros(8, 8, device=dev)
    with pytest.raises(ValueError, match="contiguous"):
        M.TensorList([x.t()[1:]])
    with pytest.raises(ValueError, match="elements"):
        M.TensorList([x], [torch.zeros(63, device=dev)])
    with pytest.raises(ValueError, match="dtype"):
        M.TensorList([x], [x.half()])
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        M.TensorList([x.double()])
    # what is written may overlap nothing: two calls' worth of scaling could meet in one element
    twice = M.TensorList([x, x.view(-1)[60:]])
    for call in (lambda: M.tensors_scale(twice, _one(2)),
                 lambda: M.tensors_clip(twice, 1.0, _one(0), _one(0)),
                 lambda: M.tensors_scale(M.TensorList([x], [x]), _one(2))):
        with pytest.raises(ValueError, match="overlap"):
            call()
    M.tensors_norm_sq_acc(twice, _one(0))
    # the same tensor twice counts twice in the norm, and may be read twice into other buffers
    y = torch.full((10,), 2.0, device=dev)
    a, b = torch.empty(2, 10, device=dev)
    n2, c = _one(0), _one(0)
    M.tensors_clip(M.TensorList([y, y], [a, b]), 1e9, n2, c)
    assert host(n2)[0] == 80 and torch.equal(a, y) and torch.equal(b, y)


def test_same_bits_again_and_from_a_graph(dev):
    """The list is baked into the graph: the host arrays may go afterwards."""
    sizes = LISTS["mixed"] + LISTS["many"]
    xs, _ = _tensors(sizes, 5)
    src = [x.clone() for x in xs]
    n2, c = _one(0), _one(0)
    outs = [torch.empty(x.numel(), device=dev) for x in xs]
    lists = [M.TensorList(xs, outs), M.TensorList(xs)]

    def step():
        for x, s in zip(xs, src):
            x.copy_(s)
        M.tensors_clip(lists[0], 3.0, n2, c)
        M.tensors_clip(lists[1], 3.0, n2, c)
    step()
    torch.cuda.synchronize()
    ref = [t.clone() for t in xs + outs + [n2, c]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(xs + outs + [n2, c], ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lists[:] = [M.TensorList(xs, outs), M.TensorList(xs)]
    other = M.TensorList([torch.ones(100, device=dev)])
    for rep in range(3):
        for t in xs + outs + [n2, c]:
            t.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(xs + outs + [n2, c], ref)), rep
        M.tensors_clip(other, 1.0, n2, c)
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(xs + outs + [n2, c], ref)), rep


def test_past_2_31_elements(dev):
    n = 2 ** 31 + 5003
    note(f"tensors clip {n}")
    x = torch.full((n,), 0.5, dtype=torch.bfloat16, device=dev)
    x[-1] = 2.0
    small = torch.ones(3, device=dev)
    n2, c = _one(0), _one(0)
    M.tensors_clip(M.TensorList([small, x, small.clone()]), 1.0, n2, c)
    want = (n - 1) / 4 + 4 + 6
    assert abs(host(n2)[0] - want) <= (S.norm_chain(n) + 4) * S.U * want
    for part in (slice(0, 9000), slice(n - 9000, n - 1)):
        assert torch.equal(x[part], (torch.full((1,), 0.5, device=dev) * c).bfloat16().expand(len(x[part])))
    assert x[-1] == (2 * c).bfloat16()


@pytest.mark.parametrize("again", [False, True])
def test_gradients_of_several_steps(dev, again):
    """A list is of the memory that the gradients had when it was made: made once for gradients
    that are cleared where they are, or made again each step for gradients that are dropped."""
    r = np.random.default_rng(8)
    params = [torch.from_numpy(r.standard_normal(s).astype(np.float32)).to(dev, t).requires_grad_()
              for s, t in (((30, 7), torch.float32), ((501,), torch.bfloat16), ((3, 3000), torch.float32))]
    optimizer = torch.optim.SGD(params, lr=0.1)
    flat = torch.zeros(sum(p.numel() for p in params), device=dev)
    n2, c = _one(0), _one(0)
    grads = None
    for step in range(3):
        optimizer.zero_grad(set_to_none=again)
        x = [torch.from_numpy(r.standard_normal(p.shape).astype(np.float32)).to(dev, p.dtype) for p in params]
        sum((p * y).float().sum() for p, y in zip(params, x)).backward()
        if again or grads is None:
            grads = M.TensorList([p.grad for p in params],
                                 list(flat.split([p.numel() for p in params])))
        M.tensors_clip(grads, 1.0, n2, c)
        want = _norm_sq(x)  # the gradients of this step are x
        assert abs(host(n2)[0] - want) <= (S.norm_chain(flat.numel()) + 4) * S.U * want
        assert torch.equal(flat, torch.cat([y.float().reshape(-1) for y in x]) * c)
