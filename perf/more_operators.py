"""What a training or serving step of a mixture-of-experts layer does beside its
products and its router: the root-mean-square norm in front of it, the balance loss
of the router, and the clipping of its many gradients by their global norm.

listed() holds fixed cases, draw(rng) gives more of the same ranges.  A case is a
dict of plain values with an "op" and a "dir":

  rms      forward: rows [plus the residual's rows] normalised, as rows of their type
           ("out": "row") or in 8 bits with a scale for each row or each 128 columns;
           backward: the rows' gradient [added to the residual stream's] and gamma's
  balance  forward: per-expert counts, mean probabilities and the loss;
           backward: the logits' gradient [added to what is there]
  clip     elsewhere: the norm of all gradients, and the gradients times the clip
           scale as fp32 pieces of one flat buffer, as the optimizer takes it;
           inplace: the same in place, with a norm below the limit

Rows, logits and weights' gradients are fp32, fp16 or bf16; gamma, statistics and
scales fp32.  Gamma's gradient accumulates (`+=`), as the framework's do.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
LARGEST_CODE = {"int8": 127.0, "e4m3": 448.0}
LEAST = 2.0 ** -100  # a row or block counts as at least this large
EPS = 1e-5
COEF = 0.01


def listed():
    return [
        # A decoding step of 16 sequences in the 1600-wide model: the residual's addition,
        # the norm, and the product's input in 8 bits.
        {"name": "rms_16x1600_e4m3", "op": "rms", "dir": "forward", "R": 16, "C": 1600,
         "type": "bf16", "residual": True, "out": "e4m3", "block": 0},
        # The same model's training batch, B=8 T=1024.
        {"name": "rms_8192x1600", "op": "rms", "dir": "forward", "R": 8192, "C": 1600,
         "type": "bf16", "residual": True, "out": "row", "block": 0},
        # The widest rows, a long batch's prefill, a scale for each 128 columns.
        {"name": "rms_32768x4096_e4m3", "op": "rms", "dir": "forward", "R": 32768, "C": 4096,
         "type": "bf16", "residual": True, "out": "e4m3", "block": 128},
        # A ragged batch and an odd width, no residual, integer codes.
        {"name": "rms_6007x769_int8", "op": "rms", "dir": "forward", "R": 6007, "C": 769,
         "type": "f16", "residual": False, "out": "int8", "block": 0},
        # The 768-wide model's gradient into the residual stream's, B=8 T=1024.
        {"name": "rms_back_8192x768", "op": "rms", "dir": "backward", "R": 8192, "C": 768,
         "type": "f32", "residual": True},
        # An odd number of rows, an odd width.
        {"name": "rms_back_4095x769", "op": "rms", "dir": "backward", "R": 4095, "C": 769,
         "type": "f16", "residual": False},
        # Wide rows of a large batch.
        {"name": "rms_back_16384x4096", "op": "rms", "dir": "backward", "R": 16384, "C": 4096,
         "type": "bf16", "residual": True},
        # The smallest router's loss.
        {"name": "balance_16x8", "op": "balance", "dir": "forward", "N": 16, "E": 8, "k": 2,
         "type": "f32", "padded": 0.0, "masked": 0.0},
        # Many small experts, 16-bit logits, a batch padded to its longest sequence.
        {"name": "balance_32768x256", "op": "balance", "dir": "forward", "N": 32768, "E": 256,
         "k": 8, "type": "bf16", "padded": 0.2, "masked": 0.0},
        # The gradient onto the router's own, a ragged batch, an expert number that is no
        # power of two, some experts masked out.
        {"name": "balance_back_8191x160", "op": "balance", "dir": "backward", "N": 8191,
         "E": 160, "k": 8, "type": "f32", "padded": 0.0, "masked": 0.1, "add": True},
        # Four layers of the reference's default width (128, 4 * 128), fp32: below the limit, in
        # place.
        {"name": "clip_4x128", "op": "clip", "dir": "inplace", "L": 4, "d": 128, "f": 512,
         "V": 1000, "E": 1, "type": "f32"},
        # The 48-layer 1600-wide model, bf16 gradients over the limit, into fp32.
        {"name": "clip_48x1600", "op": "clip", "dir": "elsewhere", "L": 48, "d": 1600, "f": 6400,
         "V": 50257, "E": 1, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row width: half the time a multiple of 64, else whatever comes."""
    w = _log(rng, lo, hi)
    return max(64, w // 64 * 64) if rng.random() < 0.5 else w


def draw(rng):
    op = rng.choice(["rms", "rms", "balance", "clip"])
    type_ = rng.choice(["f32", "f16", "bf16"])
    if op == "rms":
        cols = _width(rng, 64, 8192)
        rows = max(1, min(_log(rng, 1, 262144), (200 << 20) // (cols * SIZE[type_])))
        c = {"op": op, "dir": rng.choice(["forward", "backward"]), "R": rows, "C": cols,
             "type": type_, "residual": rng.random() < 0.5}
        if c["dir"] == "forward":
            c["out"] = rng.choice(["row", "row", "e4m3", "e4m3", "e4m3", "int8"])
            c["block"] = rng.choice([0, 128]) if c["out"] != "row" else 0
        return c
    if op == "balance":
        experts = rng.choice([8, 16, 64, 128, 256, _log(rng, 2, 384)])
        c = {"op": op, "dir": rng.choice(["forward", "backward"]), "N": _log(rng, 1, 65536),
             "E": experts, "k": min(experts, rng.choice([1, 2, 2, 3, 4, 6, 8])), "type": type_,
             "padded": rng.choice([0.0, 0.2]), "masked": rng.choice([0.0, 0.1])}
        if c["dir"] == "backward":
            c["add"] = rng.random() < 0.5
        return c
    d, experts = _width(rng, 64, 1600), rng.choice([1, 1, 8])
    c = {"op": op, "dir": rng.choice(["elsewhere", "inplace"]), "L": _log(rng, 1, 48), "d": d,
         "f": rng.choice([2 * d, 4 * d]), "V": _log(rng, 100, 50257), "E": experts,
         "type": type_}
    c["L"] = max(1, min(c["L"], 400000000 // (4 * d * d + 2 * experts * d * c["f"])))
    return c


# ----- inputs -------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=g).mul_(scale).to(dtype)


def _rand(g, *shape):
    return torch.rand(shape, device="cuda", generator=g)


def _zeros(*shape, dtype=torch.float32):
    return torch.zeros(shape, device="cuda", dtype=dtype)


def _blocks(c):
    return -(-c["C"] // c["block"]) if c["block"] else 1


def _sizes(c):
    """The model's weights, as (elements, always fp32)."""
    d, f, E = c["d"], c["f"], c["E"]
    layer = [(d, True)] + [(d * d, False)] * 4 + [(d, True)]
    if E > 1:
        layer.append((E * d, True))  # the router
    layer += [(E * d * f, False), (E * f, True), (E * f * d, False)]
    return [(c["V"] * d, False)] + layer * c["L"] + [(d, True)]


def prepare(c, seed):
    """The inputs, and the output buffers that a program keeps from step to step."""
    g, t, i32 = _gen(seed), TYPES[c["type"]], torch.int32
    s = {"case": c}
    if c["op"] == "clip":
        return _prepare_clip(s, c, g, t)
    if c["op"] == "balance":
        N, E, k = c["N"], c["E"], c["k"]
        # some experts are liked more than others
        logits = _randn(g, N, E, scale=1.5) + _randn(g, E, scale=0.7)
        logits[_rand(g, N, E) < c["masked"]] = -math.inf
        s["logits"] = logits.to(t)
        value, at = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
        ids = torch.where(value == -math.inf, -1, at)[:, :k].to(i32).contiguous()
        s["valid"] = None
        if c["padded"]:
            s["valid"] = (_rand(g, N) >= c["padded"]).to(torch.uint8)
        if c["dir"] == "forward":
            s["ids"], s["loss"] = ids, _zeros(1)
            s["counts"], s["probs"] = _zeros(E + 1, dtype=i32), _zeros(E)
        else:
            live = _valid(s)
            counts = ((ids[:, :, None] == torch.arange(E, device="cuda")).sum(1) * live).sum(0)
            s["counts"] = torch.cat([counts, live.sum()[None]]).to(i32)
            # the loss's own gradient: fp16 is trained with a loss scale
            s["dloss"] = _zeros(1) + (65536.0 if c["type"] == "f16" else 1.0)
            scale = float(s["dloss"]) * COEF / N
            s["dlogits"] = _randn(g, N, E, scale=scale, dtype=t) if c["add"] else _zeros(N, E, dtype=t)
        return s
    R, C = c["R"], c["C"]
    # a few columns of a residual stream are far larger than the rest
    loud = torch.where(_rand(g, C) < 0.005, 8.0, 1.0)
    s["gamma"] = 1 + _randn(g, C, scale=0.1)
    x = (_randn(g, R, C) * loud).to(t)
    if c["dir"] == "backward":
        s["x"], s["dy"], s["dgamma"] = x, _randn(g, R, C, dtype=t), _zeros(C)
        s["inv_rms"] = torch.rsqrt(x.float().square().mean(1) + EPS)
        s["dx"] = _randn(g, R, C, dtype=t) if c["residual"] else _zeros(R, C, dtype=t)
        return s
    s["x"] = x
    if c["residual"]:
        s["residual"], s["sum"] = _randn(g, R, C, scale=0.5, dtype=t), _zeros(R, C, dtype=t)
    if c["out"] == "row":
        s["out"], s["inv_rms"] = _zeros(R, C, dtype=t), _zeros(R)
    else:
        s["q"], s["scales"] = _zeros(R, C, dtype=torch.uint8), _zeros(R, _blocks(c))
    return s


def _prepare_clip(s, c, g, t):
    """Gradients of two types, each at a place that an allocator would give it (a multiple of
    512 bytes) in the memory that the program's gradients take; their norm is 3, or 0.3."""
    sizes = _sizes(c)
    total = sum(n for n, _ in sizes)
    std = (3.0 if c["dir"] == "elsewhere" else 0.3) / math.sqrt(total)
    at, used = [], {False: 0, True: 0}
    for n, small in sizes:
        at.append(used[small])
        used[small] += -(-n // 256) * 256
    s["memory"] = [_randn(g, used[False], scale=std, dtype=t), _randn(g, used[True], scale=std)]
    s["grads"] = [s["memory"][small][a:a + n] for (n, small), a in zip(sizes, at)]
    behind = [torch.ones(m.numel(), dtype=torch.bool, device="cuda") for m in s["memory"]]
    for (n, small), a in zip(sizes, at):
        behind[small][a:a + n] = False
    for m, b in zip(s["memory"], behind):
        m.masked_fill_(b, 0.0)
    if c["dir"] == "elsewhere":
        s["flat"] = _zeros(total)
    s["norm_sq"], s["clip"] = _zeros(1), _zeros(1)
    return s


# ----- one pass -----------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] == "rms":
        return _rms(s) if c["dir"] == "forward" else _rms_back(s)
    if c["op"] == "balance":
        return _balance(s) if c["dir"] == "forward" else _balance_back(s)
    return _clip(s)


def _rms(s):
    c = s["case"]
    t = TYPES[c["type"]]
    h, r = s["x"].float(), {}
    if c["residual"]:
        h = h + s["residual"].float()
        r["sum"] = h.to(t)
    inv = torch.rsqrt(h.square().mean(1) + EPS)
    y = h * inv[:, None] * s["gamma"]
    if c["out"] == "row":
        return {**r, "out": y.to(t), "inv_rms": inv}
    block, blocks = c["block"] or c["C"], _blocks(c)
    y = torch.nn.functional.pad(y, (0, block * blocks - c["C"])).view(c["R"], blocks, block)
    scales = y.abs().amax(2).clamp(min=LEAST) / LARGEST_CODE[c["out"]]
    q = (y / scales[:, :, None]).reshape(c["R"], -1)[:, :c["C"]]
    if c["out"] == "int8":
        return {**r, "q": q.round().to(torch.float16), "scales": scales}
    return {**r, "q": q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), "scales": scales}


def _rms_back(s):
    c = s["case"]
    inv, dy = s["inv_rms"][:, None], s["dy"].float()
    n = s["x"].float() * inv
    g = dy * s["gamma"]
    dx = inv * (g - n * (g * n).mean(1, keepdim=True))
    if c["residual"]:
        dx = s["dx"].float() + dx
    s["dx"], s["dgamma"] = dx.to(s["dx"].dtype), s["dgamma"] + (dy * n).sum(0)
    return {"dx": s["dx"], "dgamma": s["dgamma"]}


def _valid(s):
    if s["valid"] is None:
        return torch.ones(s["case"]["N"], 1, dtype=torch.int64, device="cuda")
    return (s["valid"] != 0).to(torch.int64)[:, None]


def _softmax(logits):
    l = logits.float()
    top = l.amax(1, keepdim=True)
    e = torch.where(l == -math.inf, 0.0, torch.exp(l - top))
    return e / torch.where(top == -math.inf, 1.0, e.sum(1, keepdim=True))


def _balance(s):
    c = s["case"]
    live = _valid(s)
    n = live.sum()
    p = torch.where(live != 0, _softmax(s["logits"]), 0.0).sum(0) / n.clamp(min=1)
    slots = torch.where((live != 0) & (s["ids"] >= 0) & (s["ids"] < c["E"]), s["ids"], c["E"])
    counts = _zeros(c["E"] + 1, dtype=torch.int64).scatter_add_(
        0, slots.reshape(-1).long(), torch.ones_like(slots, dtype=torch.int64).reshape(-1))
    loss = COEF * c["E"] / c["k"] * (counts[:-1].float() * p).sum() / n.clamp(min=1)
    counts[-1] = n
    return {"counts": counts.to(torch.int32), "probs": p, "loss": loss[None]}


def _balance_back(s):
    c = s["case"]
    p, n = _softmax(s["logits"]), s["counts"][-1].float()
    counts = s["counts"][:-1].float() / n.clamp(min=1)
    d = p * (counts - (p * counts).sum(1, keepdim=True))
    d = torch.where(_valid(s) != 0, d * (s["dloss"] * COEF * c["E"] / c["k"] / n.clamp(min=1)), 0.0)
    if c["add"]:
        d = s["dlogits"].float() + d
    s["dlogits"] = d.to(s["dlogits"].dtype)
    return {"dlogits": s["dlogits"]}


def _clip(s):
    if s["case"]["dir"] == "inplace":
        wide = [m.float() for m in s["memory"]]
        norm_sq = wide[0].square().sum() + wide[1].square().sum()
    else:
        flat = torch.cat([x.float() for x in s["grads"]])
        norm_sq = flat.square().sum()
    norm = torch.sqrt(norm_sq)
    scale = torch.where(norm > 1.0, 1.0 / norm, 1.0)
    r = {"norm_sq": norm_sq[None], "clip": scale[None]}
    if s["case"]["dir"] == "inplace":
        s["memory"] = [(w * scale).to(m.dtype) for w, m in zip(wide, s["memory"])]
        return {**r, "weights": s["memory"][0], "vectors": s["memory"][1]}
    return {**r, "flat": flat * scale}


def _run_own(s):
    """The framework's calls, bound once to the program's buffers."""
    if "call" not in s:
        _bind(s)
    s["call"]()
    if s["case"].get("out") == "int8":  # the codes as the numbers that they are
        return {**s["returns"], "q": s["q"].view(torch.int8).to(torch.float16)}
    return s["returns"]


def _bind(s):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    if os.path.join(root, "cme213-final-project_amd") not in sys.path:
        sys.path.insert(0, os.path.join(root, "cme213-final-project_amd"))
    import cme213_amd as M
    c, bind = s["case"], M.bind
    t = {"f32": M.TYPE_F32, "f16": M.TYPE_F16, "bf16": M.TYPE_BF16}[c["type"]]
    if c["op"] == "clip":
        flat, at = None, 0
        if c["dir"] == "elsewhere":
            flat = []
            for x in s["grads"]:
                flat.append(s["flat"][at:at + x.numel()])
                at += x.numel()
        s["list"] = M.TensorList(s["grads"], flat)
        s["call"] = bind("mi_tensors_clip", *s["list"].args(), 1.0, s["norm_sq"], s["clip"])
        s["returns"] = {"norm_sq": s["norm_sq"], "clip": s["clip"]}
        if flat is None:
            s["returns"].update(weights=s["memory"][0], vectors=s["memory"][1])
        else:
            s["returns"]["flat"] = s["flat"]
        return
    if c["op"] == "balance":
        size = (c["N"], c["E"], c["k"], COEF)
        if c["dir"] == "forward":
            s["call"] = bind("mi_moe_balance_forward", s["logits"], s["ids"], s["valid"],
                             s["counts"], s["probs"], s["loss"], *size, t)
            names = ["counts", "probs", "loss"]
        else:
            s["call"] = bind("mi_moe_balance_backward", s["logits"], s["valid"], s["counts"],
                             s["dloss"], s["dlogits"], *size, int(c["add"]), t)
            names = ["dlogits"]
    elif c["dir"] == "backward":
        name = "mi_rmsnorm_backward_residual" if c["residual"] else "mi_rmsnorm_backward"
        s["call"] = bind(name, s["dy"], s["x"], s["inv_rms"], s["gamma"], s["dx"], s["dgamma"],
                         c["R"], c["C"], t)
        names = ["dx", "dgamma"]
    else:
        rows = (s["x"], s["residual"], s["gamma"], s["sum"]) if c["residual"] else (s["x"], s["gamma"])
        name = "mi_residual_rmsnorm_forward" if c["residual"] else "mi_rmsnorm_forward"
        names = ["sum"] * c["residual"]
        if c["out"] == "row":
            s["call"] = bind(name, *rows, s["out"], s["inv_rms"], c["R"], c["C"], EPS, t)
            names += ["out", "inv_rms"]
        else:
            f = {"int8": M.ROW8_INT8, "e4m3": M.ROW8_E4M3}[c["out"]]
            s["call"] = bind(name + "_row8", *rows, s["q"], s["scales"], None, None, c["R"],
                             c["C"], EPS, c["block"], f, t)
            names += ["scales"]
    s["returns"] = {n: s[n] for n in names}
    if c.get("out") == "e4m3":
        s["returns"]["q"] = s["q"].view(torch.float8_e4m3fn)


# ----- what a pass cannot do without ----------------------------------------------

def work(c):
    b = SIZE[c["type"]]
    if c["op"] == "clip":
        n = sum(n for n, _ in _sizes(c))
        held = sum(n * (4 if small else b) for n, small in _sizes(c))
        return {"bytes": held + 4 * n * (c["dir"] == "elsewhere"),
                "flops": 2 * n + n * (c["dir"] == "elsewhere")}
    if c["op"] == "balance":
        n, small = c["N"] * c["E"] * b, c["N"] * (c["padded"] > 0)
        if c["dir"] == "forward":
            return {"bytes": n + small + 4 * c["N"] * c["k"] + 8 * c["E"],
                    "flops": 4 * c["N"] * c["E"]}
        return {"bytes": n * (2 + c["add"]) + small + 4 * c["E"], "flops": 7 * c["N"] * c["E"]}
    n = c["R"] * c["C"]
    if c["dir"] == "backward":
        return {"bytes": n * b * (3 + c["residual"]) + 4 * c["R"] + 12 * c["C"], "flops": 9 * n}
    out = n * b + 4 * c["R"] if c["out"] == "row" else n + 4 * c["R"] * _blocks(c)
    return {"bytes": n * b * (1 + 2 * c["residual"]) + out + 4 * c["C"],
            "flops": (4 + c["residual"] + 2 * (c["out"] != "row")) * n}


# ----- the definition, in 64 bits ---------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "clip":
        return _exact_clip(c, s)
    if c["op"] == "balance":
        return _exact_balance(c, s)
    parts = []
    step = max(1, (1 << 26) // c["C"])  # rows at a time
    for a in range(0, c["R"], step):
        rows = slice(a, a + step)
        parts.append(_exact_rms_back(c, s, rows) if c["dir"] == "backward" else _exact_rms(c, s, rows))
    r = {k: torch.cat([p[k] for p in parts]) for k in parts[0] if k != "dgamma"}
    if c["dir"] == "backward":
        r["dgamma"] = s["dgamma"].double() + sum(p["dgamma"] for p in parts)
    return r


def _exact_rms(c, s, rows):
    h, r = s["x"][rows].double(), {}
    if c["residual"]:
        h = h + s["residual"][rows].double()
        r["sum"] = h
    size = torch.sqrt((h * h).sum(1) / c["C"] + EPS)
    y = s["gamma"].double() * (h / size[:, None])
    if c["out"] == "row":
        return {**r, "out": y, "inv_rms": 1 / size}
    block = c["block"] or c["C"]
    scales = torch.stack([y[:, i:i + block].abs().max(1)[0] for i in range(0, c["C"], block)], 1)
    scales = scales.clamp(min=LEAST) / LARGEST_CODE[c["out"]]
    v = y / scales.repeat_interleave(block, 1)[:, :c["C"]]
    if c["out"] == "int8":
        return {**r, "q": torch.round(v), "scales": scales}
    # 3 fraction bits, the smallest exponent -6
    ulp = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return {**r, "q": torch.clamp(torch.round(v / ulp) * ulp, -448, 448), "scales": scales}


def _exact_rms_back(c, s, rows):
    x, dy, inv = s["x"][rows].double(), s["dy"][rows].double(), s["inv_rms"][rows].double()
    g = dy * s["gamma"].double()
    dot = (g * x).sum(1) / c["C"]
    dx = g * inv[:, None] - x * (dot * inv ** 3)[:, None]
    if c["residual"]:
        dx = dx + s["dx"][rows].double()
    return {"dx": dx, "dgamma": inv.unsqueeze(0).mm(dy * x)[0]}


def _exact_balance(c, s):
    keep = torch.arange(c["N"], device="cuda") if s["valid"] is None else s["valid"].nonzero()[:, 0]
    l = s["logits"][keep].double()
    e = torch.exp(l)  # a router's logits are small: no maximum is needed
    p = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    n, scale = keep.numel(), COEF * c["E"] / c["k"]
    if c["dir"] == "backward":
        counts = s["counts"][:-1].double()
        inner = p.mv(counts)
        out = s["dlogits"].double() if c["add"] else torch.zeros_like(s["dlogits"], dtype=torch.float64)
        out[keep] += p * (counts[None] - inner[:, None]) * (s["dloss"].double() * scale / max(n, 1) ** 2)
        return {"dlogits": out}
    ids = s["ids"][keep]
    counts = torch.stack([(ids == i).sum() for i in range(c["E"])] + [torch.tensor(n, device="cuda")])
    probs = p.sum(0) / max(n, 1)
    loss = scale * (counts[:-1].double() * probs).sum() / max(n, 1)
    return {"counts": counts.to(torch.int32), "probs": probs, "loss": loss[None]}


def _exact_clip(c, s):
    norm = math.sqrt(sum(float(x.double().square().sum()) for x in s["grads"]))
    scale = 1.0 / norm if norm > 1 else 1.0
    one = torch.ones(1, device="cuda", dtype=torch.float64)
    r = {"norm_sq": one * norm ** 2, "clip": one * scale}
    if c["dir"] == "inplace":
        return {**r, "weights": s["memory"][0].double() * scale,
                "vectors": s["memory"][1].double() * scale}
    flat = torch.empty_like(s["flat"], dtype=torch.float64)
    at = 0
    for x in s["grads"]:
        flat[at:at + x.numel()] = x.double() * scale
        at += x.numel()
    return {**r, "flat": flat}
