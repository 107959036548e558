"""What a mixture-of-experts feed-forward layer does outside its matrix products,
trained with the hidden activation kept in 8 bits: the router's choice, the rows
sorted by expert and brought back with their weights, and bias + GELU whose backward
pass reads an 8-bit checkpoint.

listed() holds fixed cases, draw(rng) gives more of the same ranges.  A case is a
dict of plain values with an "op" and a "dir":

  gate      forward: the k largest logits of each token and their softmax weights;
            backward: the logits' gradient from the weights'
  dispatch  forward: slots sorted by expert, token rows copied to their experts;
            backward: the rows' gradients summed per token
  combine   forward: each token's expert rows summed with its weights;
            backward: the rows' and the weights' gradients
  gelu8     step: bias + GELU of rows grouped by expert, its input kept in 8 bits,
            then the gradient from the checkpoint; backward: the gradient alone

Rows are fp32, fp16 or bf16; weights, biases and their gradients fp32.  Bias
gradients accumulate (`+=`), as the framework's do.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32       # columns that share a scale in a checkpoint
LEAST_EXP = -118  # the smallest exponent a scale takes


def listed():
    return [
        # A serving step's router: 16 sequences, one token each, 8 experts.
        {"name": "gate_16x8", "op": "gate", "dir": "forward", "N": 16, "E": 8, "k": 2,
         "renorm": True, "type": "f32", "masked": 0.0},
        # Training, B=8 T=1024, many small experts, weights over all of them.
        {"name": "gate_8192x64", "op": "gate", "dir": "forward", "N": 8192, "E": 64, "k": 6,
         "renorm": False, "type": "f32", "masked": 0.0},
        # A ragged batch and an expert number that is no power of two, some experts
        # masked out, 16-bit logits.
        {"name": "gate_back_8191x160", "op": "gate", "dir": "backward", "N": 8191, "E": 160,
         "k": 8, "renorm": False, "type": "bf16", "masked": 0.1},
        # The serving step's rows to their experts, 768 wide.
        {"name": "dispatch_16x768", "op": "dispatch", "dir": "forward", "N": 16, "E": 8, "k": 2,
         "C": 768, "type": "f32", "dropped": 0.0},
        # Training rows of the 1600-wide model, 64 experts.
        {"name": "dispatch_8192x1600", "op": "dispatch", "dir": "forward", "N": 8192, "E": 64,
         "k": 4, "C": 1600, "type": "bf16", "dropped": 0.02},
        # Its gradient on an odd number of tokens and an odd width.
        {"name": "dispatch_back_4095x769", "op": "dispatch", "dir": "backward", "N": 4095,
         "E": 16, "k": 2, "C": 769, "type": "f32", "dropped": 0.02},
        # The largest rows back: 8 experts of 128 a token, 4096 wide.
        {"name": "combine_8192x4096", "op": "combine", "dir": "forward", "N": 8192, "E": 128,
         "k": 8, "C": 4096, "type": "bf16", "dropped": 0.0},
        # Their gradients at the 768-wide model.
        {"name": "combine_back_8192x768", "op": "combine", "dir": "backward", "N": 8192, "E": 8,
         "k": 2, "C": 768, "type": "f32", "dropped": 0.0},
        # Three choices, a width that is no multiple of 4, dropped slots, fp16.
        {"name": "combine_back_3001x1026", "op": "combine", "dir": "backward", "N": 3001,
         "E": 24, "k": 3, "C": 1026, "type": "f16", "dropped": 0.05},
        # The reference's default FFN (B=32, T=64, 4 * 128), one bias: the smallest step.
        {"name": "gelu8_2048x512", "op": "gelu8", "dir": "step", "R": 2048, "F": 512, "G": 1,
         "type": "f32", "format": "int8", "act": False, "dropped": 0.0},
        # Two choices for each of 8192 tokens, 6400 wide, 32 experts, the activation
        # computed again for the second product's weight gradient.
        {"name": "gelu8_16384x6400", "op": "gelu8", "dir": "step", "R": 16384, "F": 6400, "G": 32,
         "type": "bf16", "format": "int8", "act": True, "dropped": 0.0},
        # The gradient alone, odd sizes, the floating 8-bit format.
        {"name": "gelu8_back_6007x2049", "op": "gelu8", "dir": "backward", "R": 6007, "F": 2049,
         "G": 5, "type": "f16", "format": "e4m3", "act": True, "dropped": 0.02},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row width: half the time a multiple of 64, else whatever comes."""
    w = _log(rng, lo, hi)
    return max(64, w // 64 * 64) if rng.random() < 0.5 else w


def draw(rng):
    op = rng.choice(["gate", "dispatch", "combine", "gelu8"])
    type_ = rng.choice(["f32", "f16", "bf16"])
    if op == "gelu8":
        cols, groups = _width(rng, 64, 8192), rng.choice([1, 1, _log(rng, 2, 128)])
        rows = max(1, min(_log(rng, 1, 32768), (200 << 20) // (cols * SIZE[type_])))
        return {"op": op, "dir": rng.choice(["step", "step", "backward"]), "R": rows, "F": cols,
                "G": groups, "type": type_, "format": rng.choice(["int8", "e4m3"]),
                "act": rng.random() < 0.5,
                "dropped": rng.choice([0.0, 0.03]) if groups > 1 else 0.0}
    experts = rng.choice([8, 16, 64, 128, 256, _log(rng, 2, 384)])
    k = min(experts, rng.choice([1, 2, 2, 3, 4, 6, 8]))
    tokens = _log(rng, 1, 32768)
    if op == "gate":
        return {"op": op, "dir": rng.choice(["forward", "backward"]), "N": tokens, "E": experts,
                "k": k, "renorm": rng.random() < 0.5, "type": type_,
                "masked": rng.choice([0.0, 0.1])}
    cols = _width(rng, 64, 8192)
    tokens = max(1, min(tokens, (400 << 20) // (k * cols * SIZE[type_])))
    return {"op": op, "dir": rng.choice(["forward", "backward"]), "N": tokens, "E": experts,
            "k": k, "C": cols, "type": type_, "dropped": rng.choice([0.0, 0.03])}


# ----- inputs -------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=g).mul_(scale).to(dtype)


def _rand(g, *shape):
    return torch.rand(shape, device="cuda", generator=g)


def _router(g, tokens, experts):
    """A router's logits: some experts are liked more than others."""
    return _randn(g, tokens, experts, scale=1.5) + _randn(g, experts, scale=0.7)


def _chosen(g, c):
    """Expert ids of a router's choice, a share of the slots dropped (-1)."""
    top = torch.sort(_router(g, c["N"], c["E"]), dim=1, descending=True, stable=True)[1]
    ids = top[:, :c["k"]].to(torch.int32).contiguous()
    ids[_rand(g, *ids.shape) < c["dropped"]] = -1
    return ids.reshape(-1)


def _position(ids, experts):
    """The row of each slot in the buffer sorted by expert, -1 where dropped."""
    key = torch.where(ids < 0, experts, ids)
    order = torch.sort(key, stable=True)[1]
    position = torch.empty_like(ids)
    position[order] = torch.arange(ids.numel(), device="cuda", dtype=torch.int32)
    return torch.where(ids < 0, -1, position).contiguous()


def _zeros(*shape, dtype=torch.float32):
    return torch.zeros(shape, device="cuda", dtype=dtype)


def prepare(c, seed):
    """The inputs, and the output buffers that a program keeps from step to step."""
    g, t, i32 = _gen(seed), TYPES[c["type"]], torch.int32
    s = {"case": c}
    if c["op"] == "gelu8":
        R, F, G = c["R"], c["F"], c["G"]
        # pre-activations: a few columns are far larger than the rest
        loud = torch.where(_rand(g, F) < 0.01, 6.0, 1.0)
        h = (_randn(g, R, F, scale=1.5) * loud).to(t)
        s["bias"], s["dbias"] = _randn(g, G, F, scale=0.1), _zeros(G, F)
        s["grad_out"] = _randn(g, R, F, dtype=t)
        s["offsets"] = None
        if G > 1:
            share = torch.cumsum(_rand(g, G) ** 2 + 0.01, 0)
            ends = (share / share[-1] * (R * (1 - c["dropped"]))).round()
            s["offsets"] = torch.cat([_zeros(1), ends]).to(i32)
        for name in ("out", "grad_in", "act"):
            s[name] = _zeros(R, F, dtype=t)
        s["q"] = _zeros(R, F, dtype=torch.uint8)
        s["scales"] = _zeros(R, -(-F // BLOCK), dtype=torch.uint8)
        if c["dir"] == "step":
            s["in"] = h
        else:
            q, s["scales"] = _to_ckpt8(h.float(), c["format"])
            s["q"] = _code(q, c["format"])
        return s
    N, E, k = c["N"], c["E"], c["k"]
    if c["op"] == "gate":
        logits = _router(g, N, E)
        logits[_rand(g, N, E) < c["masked"]] = -math.inf
        s["logits"] = logits.to(t)
        if c["dir"] == "forward":
            s["ids"], s["weights"] = _zeros(N, k, dtype=i32), _zeros(N, k)
        else:
            s["ids"], s["weights"] = _gate(s["logits"], k, c["renorm"])
            s["dweights"], s["dlogits"] = _randn(g, N, k), _zeros(N, E, dtype=t)
        return s
    C, M = c["C"], N * k
    ids = _chosen(g, c)
    if c["op"] == "dispatch" and c["dir"] == "forward":
        s["ids"], s["x"] = ids, _randn(g, N, C, dtype=t)
        s["offsets"], s["order"] = _zeros(E + 1, dtype=i32), _zeros(M, dtype=i32)
        s["position"], s["out"] = _zeros(M, dtype=i32), _zeros(M, C, dtype=t)
        return s
    s["position"] = _position(ids, E)
    if c["op"] == "dispatch":
        s["dout"], s["dx"] = _randn(g, M, C, dtype=t), _zeros(N, C, dtype=t)
        return s
    s["y"] = _randn(g, M, C, dtype=t)
    w = _rand(g, N, k) + 0.1
    s["weights"] = w / w.sum(1, keepdim=True)
    if c["dir"] == "forward":
        s["out"] = _zeros(N, C, dtype=t)
    else:
        s["dout"], s["dy"], s["dweights"] = _randn(g, N, C, dtype=t), _zeros(M, C, dtype=t), _zeros(N, k)
    return s


# ----- one pass -----------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] == "gate":
        if c["dir"] == "forward":
            ids, weights = _gate(s["logits"], c["k"], c["renorm"])
            return {"ids": ids, "weights": weights}
        return {"dlogits": _gate_back(s["logits"], s["ids"], s["weights"], s["dweights"],
                                      c["renorm"])}
    if c["op"] == "dispatch":
        return _dispatch(s) if c["dir"] == "forward" else {"dx": _gather_sum(s["dout"], s, None)}
    if c["op"] == "combine":
        if c["dir"] == "forward":
            return {"out": _gather_sum(s["y"], s, s["weights"])}
        return _combine_back(s)
    return _gelu8(s)


def _gate(logits, k, renorm):
    l = logits.float()
    value, at = torch.sort(l, dim=1, descending=True, stable=True)
    value, at = value[:, :k], at[:, :k]
    none = value == -math.inf
    top = value[:, :1]
    e = torch.where(none, 0.0, torch.exp(value - top))
    if renorm:
        total = e.sum(1, keepdim=True)
    else:
        total = torch.where(l == -math.inf, 0.0, torch.exp(l - top)).sum(1, keepdim=True)
    return (torch.where(none, -1, at).to(torch.int32).contiguous(),
            torch.where(none, 0.0, e / total).contiguous())


def _gate_back(logits, ids, w, dw, renorm):
    l, chosen = logits.float(), ids >= 0
    wd = torch.where(chosen, w * dw, 0.0)
    d = wd.sum(1, keepdim=True)
    if renorm:
        return _zeros(*l.shape).scatter_add_(1, ids.clamp(min=0).long(),
                                             torch.where(chosen, w * (dw - d), 0.0)).to(logits.dtype)
    top = l.amax(1, keepdim=True)
    e = torch.where(l == -math.inf, 0.0, torch.exp(l - top))
    p = e / torch.where(top == -math.inf, 1.0, e.sum(1, keepdim=True))
    return (-p * d).scatter_add_(1, ids.clamp(min=0).long(), wd).to(logits.dtype)


def _dispatch(s):
    c = s["case"]
    E, k, ids = c["E"], c["k"], s["ids"]
    M = ids.numel()
    key = torch.where((ids < 0) | (ids >= E), E, ids)
    count = (key[:, None] == torch.arange(E, device="cuda")).sum(0)
    offsets = torch.cat([_zeros(1, dtype=torch.int64), torch.cumsum(count, 0)])
    order = torch.sort(key, stable=True)[1]
    row = torch.arange(M, device="cuda")
    position = torch.empty_like(row)
    position[order] = row
    used = row < offsets[E]
    return {"offsets": offsets.to(torch.int32),
            "order": torch.where(used, order.to(torch.int32), s["order"]),
            "position": torch.where(key == E, -1, position).to(torch.int32),
            "out": torch.where(used[:, None], s["x"][order // k], s["out"])}


def _gather_sum(rows, s, weights):
    """sum over a token's slots of [its weight times] its row."""
    c = s["case"]
    at = s["position"].long()
    there = (at >= 0).view(-1, 1)
    r = torch.where(there, rows[at.clamp(min=0)].float(), 0.0)
    if weights is not None:
        r = r * weights.reshape(-1, 1)
    return r.view(c["N"], c["k"], c["C"]).sum(1).to(rows.dtype)


def _combine_back(s):
    c = s["case"]
    at = s["position"].long()
    there = at >= 0
    g = s["dout"].float().repeat_interleave(c["k"], 0)
    dw = torch.where(there, (g * s["y"][at.clamp(min=0)].float()).sum(1), 0.0)
    dy = (g * s["weights"].reshape(-1, 1)).to(s["y"].dtype)
    slot = _zeros(at.numel() + 1, dtype=torch.int64)
    slot[torch.where(there, at, at.numel())] = torch.arange(at.numel(), device="cuda")
    used = torch.arange(at.numel(), device="cuda") < there.sum()
    return {"dy": torch.where(used[:, None], dy[slot[:-1]], s["dy"]),
            "dweights": dw.view(c["N"], c["k"])}


def _blocks(x):
    """Columns in blocks of 32, the last one filled with zeros: [rows, blocks, 32]."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK))
    return x.view(x.shape[0], -1, BLOCK)


def _to_ckpt8(x, fmt):
    """The scaled values rounded to their 8-bit format (still floats), and the scales' bytes."""
    b = _blocks(x)
    e = (torch.frexp(b.abs().amax(2))[1] - 1).clamp(min=LEAST_EXP)
    e = torch.where(b.abs().amax(2) == 0, LEAST_EXP, e)
    if fmt == "int8":
        q = torch.ldexp(b, (6 - e)[:, :, None]).round().clamp(max=127.0)
    else:
        q = torch.ldexp(b, (8 - e)[:, :, None]).clamp(-448.0, 448.0)
        q = q.to(torch.float8_e4m3fn).float()
    bad = ~torch.isfinite(b).all(2)
    q = torch.where(bad[:, :, None], 0.0, q).reshape(x.shape[0], -1)[:, :x.shape[1]]
    return q.contiguous(), torch.where(bad, 255, e + 127).to(torch.uint8)


def _code(q, fmt):
    """The bytes of rounded values."""
    return (q.to(torch.int8) if fmt == "int8" else q.to(torch.float8_e4m3fn)).view(torch.uint8)


def _from_ckpt8(q, scales, fmt):
    v = (q.view(torch.int8) if fmt == "int8" else q.view(torch.float8_e4m3fn)).float()
    step = torch.ldexp(_zeros(1) + 1.0, scales.to(torch.int32) - (133 if fmt == "int8" else 135))
    step = torch.where(scales == 255, math.nan, step)
    return v * step.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _gelu(u):
    """Half tanh GELU's slope terms: 1 / (1 + exp(-2 z)) and dz/du."""
    z = math.sqrt(2 / math.pi) * (u + 0.044715 * u * u * u)
    return torch.sigmoid(2 * z), math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * u * u)


def _gelu8(s):
    c = s["case"]
    R, G, t = c["R"], c["G"], TYPES[c["type"]]
    row = torch.arange(R, device="cuda")
    if G > 1:
        group = (row[:, None] >= s["offsets"][None, 1:]).sum(1)
        used = group < G
        bias = s["bias"][group.clamp(max=G - 1)]
        member = (group[None, :] == torch.arange(G, device="cuda")[:, None]).float()
    else:
        used, bias, member = row >= 0, s["bias"], torch.ones(1, R, device="cuda")
    used = used[:, None]
    r = {}
    if c["dir"] == "step":
        u = s["in"].float() + bias
        r["out"] = torch.where(used, (u * _gelu(u)[0]).to(t), s["out"])
        q, scales = _to_ckpt8(s["in"].float(), c["format"])
        q = _code(q, c["format"])
    else:
        q, scales = s["q"], s["scales"]
    u = _from_ckpt8(q, scales, c["format"]) + bias
    p, dz = _gelu(u)
    grad = s["grad_out"].float() * (p + 2 * u * p * (1 - p) * dz)
    r["grad_in"] = torch.where(used, grad.to(t), s["grad_in"])
    if c["act"]:
        r["act"] = torch.where(used, (u * p).to(t), s["act"])
    s["dbias"] = s["dbias"] + member @ torch.where(used, grad, 0.0)
    r["dbias"] = s["dbias"]
    return r


def _run_own(s):
    """The framework's calls, bound once to the program's buffers."""
    if "calls" not in s:
        s["calls"] = _bind(s)
    for call in s["calls"]:
        call()
    return s["returns"]


def _bind(s):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    if os.path.join(root, "cme213-final-project_amd") not in sys.path:
        sys.path.insert(0, os.path.join(root, "cme213-final-project_amd"))
    import cme213_amd as M
    c, bind = s["case"], M.bind
    t = {"f32": M.TYPE_F32, "f16": M.TYPE_F16, "bf16": M.TYPE_BF16}[c["type"]]
    if c["op"] == "gelu8":
        f = {"int8": M.CKPT8_INT8, "e4m3": M.CKPT8_E4M3}[c["format"]]
        size = (c["R"], c["F"], c["G"], f, t)
        act = s["act"] if c["act"] else None
        calls = []
        if c["dir"] == "step":
            calls.append(bind("mi_bias_gelu_forward_ckpt8", s["in"], s["bias"], s["offsets"],
                              s["out"], s["q"], s["scales"], *size))
        calls.append(bind("mi_gelu_backward_with_bias_backward_ckpt8", s["q"], s["scales"],
                          s["bias"], s["offsets"], s["grad_out"], s["grad_in"], act, s["dbias"],
                          *size))
        names = ["grad_in", "dbias"] + ["out"] * (c["dir"] == "step") + ["act"] * c["act"]
    elif c["op"] == "gate":
        size = (c["N"], c["E"], c["k"], int(c["renorm"]), t)
        if c["dir"] == "forward":
            calls = [bind("mi_moe_gate_forward", s["logits"], s["ids"], s["weights"], *size)]
            names = ["ids", "weights"]
        else:
            calls = [bind("mi_moe_gate_backward", s["logits"], s["ids"], s["weights"],
                          s["dweights"], s["dlogits"], *size)]
            names = ["dlogits"]
    else:
        slots = c["N"] * c["k"]
        size = (c["N"], c["k"], slots, c["C"], t)
        if c["op"] == "dispatch" and c["dir"] == "forward":
            calls = [bind("mi_moe_sort", s["ids"], s["offsets"], s["order"], s["position"], slots,
                          c["E"]),
                     bind("mi_moe_dispatch_forward", s["x"], s["position"], s["out"], *size)]
            names = ["offsets", "order", "position", "out"]
        elif c["op"] == "dispatch":
            calls = [bind("mi_moe_dispatch_backward", s["dout"], s["position"], s["dx"], *size)]
            names = ["dx"]
        elif c["dir"] == "forward":
            calls = [bind("mi_moe_combine_forward", s["y"], s["position"], s["weights"], s["out"],
                          *size)]
            names = ["out"]
        else:
            calls = [bind("mi_moe_combine_backward", s["dout"], s["y"], s["position"],
                          s["weights"], s["dy"], s["dweights"], *size)]
            names = ["dy", "dweights"]
    s["returns"] = {n: s[n] for n in names}
    return calls


# ----- what a pass cannot do without ----------------------------------------------

def work(c):
    b = SIZE[c["type"]]
    if c["op"] == "gelu8":
        n = c["R"] * c["F"] * (1 - c["dropped"])
        code = n + c["R"] * -(-c["F"] // BLOCK)
        small = 4 * c["G"] * c["F"]
        if c["dir"] == "step":  # in, out, codes written and read, both gradients, sums
            return {"bytes": (4 + c["act"]) * n * b + 2 * code + 4 * small, "flops": 40 * n}
        return {"bytes": (2 + c["act"]) * n * b + code + 3 * small, "flops": 25 * n}
    N, E, k = c["N"], c["E"], c["k"]
    if c["op"] == "gate":
        if c["dir"] == "forward":
            return {"bytes": N * E * b + 8 * N * k, "flops": 4 * N * E}
        return {"bytes": N * E * b * (1 if c["renorm"] else 2) + 12 * N * k, "flops": 4 * N * E}
    row, used = c["C"] * b, N * k * (1 - c["dropped"])
    if c["op"] == "dispatch":
        index = 12 * N * k + 4 * (E + 1) if c["dir"] == "forward" else 4 * N * k
        return {"bytes": (N + used) * row + index, "flops": used * c["C"]}
    if c["dir"] == "forward":
        return {"bytes": (N + used) * row + 8 * N * k, "flops": 2 * used * c["C"]}
    return {"bytes": (N + 2 * used) * row + 12 * N * k, "flops": 3 * used * c["C"]}


# ----- the definition, in 64 bits ---------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "gate":
        return _exact_gate(c, s)
    if c["op"] == "gelu8":
        return _exact_gelu8(c, s)
    if c["op"] == "dispatch" and c["dir"] == "forward":
        return _exact_dispatch(c, s)
    N, k, C = c["N"], c["k"], c["C"]
    at = s["position"].view(N, k)
    if c["op"] == "dispatch" or c["dir"] == "forward":
        rows = s["dout"] if c["op"] == "dispatch" else s["y"]
        total = torch.zeros(N, C, device="cuda", dtype=torch.float64)
        for j in range(k):
            t = (at[:, j] >= 0).nonzero()[:, 0]
            r = rows[at[t, j].long()].double()
            total[t] += r if c["op"] == "dispatch" else r * s["weights"][t, j, None].double()
        return {"dx" if c["op"] == "dispatch" else "out": total}
    dy = s["dy"].double()
    dw = torch.zeros(N, k, device="cuda", dtype=torch.float64)
    for j in range(k):
        t = (at[:, j] >= 0).nonzero()[:, 0]
        r, g = at[t, j].long(), s["dout"][t].double()
        dy[r] = g * s["weights"][t, j, None].double()
        dw[t, j] = (g * s["y"][r].double()).sum(1)
    return {"dy": dy, "dweights": dw}


def _exact_gate(c, s):
    l, k = s["logits"].double(), c["k"]
    N, E = l.shape
    e = torch.exp(l)  # a router's logits are small: no maximum is needed
    if c["dir"] == "backward":
        dl = torch.zeros_like(l)
        w, dw, ids = s["weights"].double(), s["dweights"].double(), s["ids"].long()
        d = (w * dw).sum(1)
        for j in range(k):
            t = (ids[:, j] >= 0).nonzero()[:, 0]
            dl[t, ids[t, j]] += w[t, j] * (dw[t, j] - (d[t] if c["renorm"] else 0))
        if not c["renorm"]:
            dl -= e / e.sum(1, keepdim=True).clamp(min=1e-300) * d[:, None]
        return {"dlogits": dl}
    ids = torch.full((N, k), -1, device="cuda", dtype=torch.int32)
    w = torch.zeros(N, k, device="cuda", dtype=torch.float64)
    index = torch.arange(E, device="cuda")
    left = l.clone()
    for j in range(k):
        top = left.amax(1, keepdim=True)
        first = torch.where(left == top, index, E).amin(1)  # ties: the lowest expert
        fine = (top[:, 0] > -math.inf).nonzero()[:, 0]
        ids[fine, j] = first[fine].to(torch.int32)
        w[fine, j] = e[fine, first[fine]]
        left[fine, first[fine]] = -math.inf
    total = w.sum(1, keepdim=True) if c["renorm"] else e.sum(1, keepdim=True)
    return {"ids": ids, "weights": w / total.clamp(min=1e-300)}


def _exact_dispatch(c, s):
    out, order = s["out"].double(), s["order"].clone()
    position, offsets, row = torch.full_like(s["ids"], -1), [0], 0
    for expert in range(c["E"]):
        slots = (s["ids"] == expert).nonzero()[:, 0]
        n = slots.numel()
        order[row:row + n] = slots.to(torch.int32)
        position[slots] = torch.arange(row, row + n, device="cuda", dtype=torch.int32)
        out[row:row + n] = s["x"][torch.div(slots, c["k"], rounding_mode="floor")].double()
        row += n
        offsets.append(row)
    return {"offsets": torch.tensor(offsets, device="cuda", dtype=torch.int32), "order": order,
            "position": position, "out": out}


def _exact_read(c, s):
    """What the checkpoint of the input stands for, from the format's definition."""
    if c["dir"] == "backward":
        q, byte = s["q"], s["scales"].double()
        if c["format"] == "int8":
            v = q.double() - 256.0 * (q >= 128)
            step = torch.exp2(byte - 133)
        else:  # 1 sign, 4 exponent and 3 fraction bits, exponent bias 7
            b = q.to(torch.int32)
            exp, frac = (b >> 3) & 15, (b & 7).double()
            v = torch.where(exp == 0, frac / 512, (1 + frac / 8) * torch.exp2(exp.double() - 7))
            v = torch.where(b >= 128, -v, v)
            step = torch.exp2(byte - 135)
        return v * step.repeat_interleave(BLOCK, 1)[:, :c["F"]]
    x = s["in"].double()
    big = torch.zeros(x.shape[0], s["scales"].shape[1] * BLOCK, device="cuda", dtype=torch.float64)
    big[:, :c["F"]] = x.abs()
    big = big.view(x.shape[0], -1, BLOCK).amax(2).clamp(min=2.0 ** LEAST_EXP)
    e = torch.floor(torch.log2(big))
    e = torch.where(torch.exp2(e) > big, e - 1, torch.where(torch.exp2(e + 1) <= big, e + 1, e))
    e = e.repeat_interleave(BLOCK, 1)[:, :c["F"]]
    if c["format"] == "int8":
        return torch.clamp(torch.round(x / torch.exp2(e - 6)), max=127) * torch.exp2(e - 6)
    v = torch.clamp(x / torch.exp2(e - 8), -448, 448)
    own_e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    ulp = torch.exp2(own_e - 3)
    return torch.round(v / ulp) * ulp * torch.exp2(e - 8)


def _exact_gelu(u):
    z = math.sqrt(2 / math.pi) * (u + 0.044715 * u ** 3)
    t = torch.tanh(z)
    d = 0.5 * (1 + t) + 0.5 * u * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * u * u)
    return 0.5 * u * (1 + t), d


def _exact_gelu8(c, s):
    R, G = c["R"], c["G"]
    ends = [0, R] if G == 1 else s["offsets"].tolist()
    kept = _exact_read(c, s)
    r = {"grad_in": s["grad_in"].double(), "dbias": s["dbias"].double()}
    if c["dir"] == "step":
        r["out"] = s["out"].double()
    if c["act"]:
        r["act"] = s["act"].double()
    for i in range(G):
        a, b = ends[i], ends[i + 1]
        bias = s["bias"][i].double()
        if c["dir"] == "step":
            r["out"][a:b] = _exact_gelu(s["in"][a:b].double() + bias)[0]
        y, d = _exact_gelu(kept[a:b] + bias)
        g = s["grad_out"][a:b].double() * d
        r["grad_in"][a:b] = g
        r["dbias"][i] += g.sum(0)
        if c["act"]:
            r["act"][a:b] = y
    return r
