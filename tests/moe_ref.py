"""Plain implementations, in 64 bits and on the host, of the mixture-of-experts
and 8-bit checkpoint entry points, and the error bounds their tests use.

Bounds.  U = 2^-24 is half a step of fp32; `half_step` the half step of the row
type, relative to the value (fp32 2^-24, fp16 2^-11, bf16 2^-8), plus half of
the smallest subnormal.  A sum of n fp32 terms is off by at most about n U times
the sum of their magnitudes."""
import numpy as np
import torch

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(t, ref):
    """Half a step of type t at the values ref."""
    fi = torch.finfo(TYPES[t])
    return np.abs(ref) * fi.eps / 2 + float(fi.smallest_normal) * fi.eps / 2


def near(name, got, want, bound):
    """|got - want| <= bound; NaN and infinities in the same places."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, f"{name}: {got.shape} and {want.shape}"
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{name}: NaN in other places"
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), name
    err = np.abs(np.where(fine, got - np.where(fine, want, 0), 0))
    over = err > np.where(fine, bound, 1)
    if over.any():
        i = np.unravel_index(np.argmax(np.where(fine, err - bound, -1)), err.shape)
        raise AssertionError(f"{name}: {over.sum()} of {err.size} off; at {i} got {got[i]!r}, "
                             f"want {want[i]!r}, bound {np.broadcast_to(bound, err.shape)[i]:.3e}")


# ----- router ------------------------------------------------------------------------

def gate(l, k, renorm):
    """ids, weights and a relative bound on the weights, of logits l (float64)."""
    n, e = l.shape
    ids, w = np.full((n, k), -1, np.int32), np.zeros((n, k))
    rel = np.zeros((n, k))
    for i in range(n):
        # NaN above all, then falling, equal ones by rising expert; -inf never
        rank = sorted((j for j in range(e) if l[i, j] != -np.inf),
                      key=lambda j: (0 if np.isnan(l[i, j]) else 1,
                                     0.0 if np.isnan(l[i, j]) else -l[i, j], j))
        chosen = rank[:k]
        ids[i, :len(chosen)] = chosen
        part = l[i, chosen if renorm else rank]
        if not len(chosen):
            continue
        top = l[i, rank[0]]
        with np.errstate(invalid="ignore"):
            w[i, :len(chosen)] = np.exp(l[i, chosen] - top) / np.exp(part - top).sum()
            # the difference to the top is rounded (U of it), exp is good to a
            # few U, the sum of at most e terms to e U, and their own errors
            # (x e^-x <= 0.37 each) enter the total once more
            rel[i, :len(chosen)] = U * (np.abs(l[i, chosen] - top) + 2 * e + 16)
    return ids, w, rel


def gate_back(l, ids, w, dw, renorm):
    """dlogits and an absolute bound on the fp32 computation of them."""
    n, e = l.shape
    k = ids.shape[1]
    out, bound = np.zeros((n, e)), np.zeros((n, e))
    for i in range(n):
        live = ids[i] >= 0
        wd = np.where(live, w[i] * dw[i], 0)
        d, size = wd.sum(), np.abs(wd).sum()
        if not renorm:
            fin = l[i][l[i] != -np.inf]
            if len(fin):
                with np.errstate(invalid="ignore"):
                    top = np.nan if np.isnan(fin).any() else fin.max()
                    ex = np.where(l[i] == -np.inf, 0, np.exp(l[i] - top))
                    p = ex / ex.sum()
                out[i] -= p * d
                spread = np.abs(fin - top).max() if np.isfinite(fin).all() else 0
                bound[i] += U * (spread + 2 * e + k + 24) * p * size
        for j in range(k):
            if live[j]:
                out[i, ids[i, j]] += w[i, j] * (dw[i, j] - d) if renorm else wd[j]
                # one more rounding for each term added to the same logit
                bound[i, ids[i, j]] += U * (k + 8) * (abs(wd[j]) + abs(w[i, j]) * size)
    return out, bound


# ----- sort and rows ---------------------------------------------------------------------

def sort(ids, experts):
    key = np.where((ids < 0) | (ids >= experts), experts, ids)
    order = np.argsort(key, kind="stable").astype(np.int32)
    offsets = np.searchsorted(key[order], np.arange(experts + 1)).astype(np.int32)
    position = np.full(len(ids), -1, np.int32)
    used = offsets[experts]
    position[order[:used]] = np.arange(used)
    return offsets, order[:used], position


def there(position, rows):
    return (position >= 0) & (position < rows)


def gather_sum(src, position, weights, n, k, rows):
    """sum over j of [w] src[position], and the sum of the terms' magnitudes."""
    out, size = np.zeros((n, src.shape[1])), np.zeros((n, src.shape[1]))
    pos, ok = position.reshape(n, k), there(position, rows).reshape(n, k)
    for t in range(n):
        for j in range(k):
            if ok[t, j]:
                term = src[pos[t, j]] * (1.0 if weights is None else weights[t, j])
                out[t] += term
                size[t] += np.abs(term)
    return out, size


# ----- 8-bit checkpoints ------------------------------------------------------------------

BLOCK = 32


def _e4m3_table():
    v = np.empty(256)
    for b in range(256):
        exp, frac = (b >> 3) & 15, b & 7
        m = frac / 8 * 2.0 ** -6 if exp == 0 else (1 + frac / 8) * 2.0 ** (exp - 7)
        if exp == 15 and frac == 7:
            m = np.nan
        v[b] = -m if b >= 128 else m
    return v


E4M3 = _e4m3_table()


def to_ckpt8(x, fmt):
    """Codes and scale bytes of x (float64 values of the row type)."""
    rows, cols = x.shape
    nb = -(-cols // BLOCK)
    pad = np.zeros((rows, nb * BLOCK))
    pad[:, :cols] = x
    b = pad.reshape(rows, nb, BLOCK)
    bad = ~np.isfinite(b).all(2)
    b = np.where(bad[:, :, None], 0, b)
    big = np.abs(b).max(2)
    e = np.where(big > 0, np.frexp(np.where(big > 0, big, 1))[1] - 1, -118)
    e = np.maximum(e, -118)
    if fmt == "int8":
        q = np.minimum(np.rint(np.ldexp(b, (6 - e)[:, :, None])), 127).astype(np.int8)
        code = q.view(np.uint8)
    else:
        s = np.clip(np.ldexp(b, (8 - e)[:, :, None]), -448, 448)
        # nearest code, ties to the even one; the sign of a zero is kept
        pos = E4M3[:127]
        i = np.clip(np.searchsorted(pos, np.abs(s)), 1, 126)
        lo, hi = pos[i - 1], pos[i]
        d = (np.abs(s) - lo) - (hi - np.abs(s))
        i = np.where(d < 0, i - 1, np.where(d > 0, i, np.where((i - 1) % 2 == 0, i - 1, i)))
        code = (i + np.where(np.signbit(s), 128, 0)).astype(np.uint8)
    scale = np.where(bad, 255, e + 127).astype(np.uint8)
    return np.ascontiguousarray(code.reshape(rows, -1)[:, :cols]), scale


def from_ckpt8(code, scale, fmt):
    if fmt == "int8":
        v, s = code.view(np.int8).astype(np.float64), scale.astype(np.int32) - 133
    else:
        v, s = E4M3[code], scale.astype(np.int32) - 135
    step = np.where(scale == 255, np.nan, np.ldexp(1.0, s))
    return v * np.repeat(step, BLOCK, 1)[:, :code.shape[1]]


def gelu(u):
    """gelu(u) and gelu'(u), tanh form, through the logistic function of 2z."""
    c = np.sqrt(2 / np.pi)
    z = c * (u + 0.044715 * u ** 3)
    with np.errstate(over="ignore", invalid="ignore"):
        s = 1 / (1 + np.exp(-2 * z))
        y = np.where(np.isneginf(u), 0.0, u * s)
        d = s + 2 * u * s * (1 - s) * c * (1 + 3 * 0.044715 * u * u)
    return y, np.where(np.isinf(u), (u > 0) * 1.0, d)


def groups_of(offsets, rows, groups):
    """The group of each row, -1 for none."""
    g = np.full(rows, -1)
    if offsets is None:
        g[:] = 0
        return g
    for i in range(groups):
        g[max(0, offsets[i]):min(rows, offsets[i + 1])] = i
    return g
