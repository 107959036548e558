"""Plain implementations, in 64 bits and on the host, of RMS norm, rows in 8 bits, the
router's balance loss and clipping, and the error bounds their tests use.

Bounds.  U = 2^-24 is half a step of fp32.  A sum of positive terms in which no term goes
through more than `chain` additions is off by at most chain U of itself; a sum of any terms
by chain U times the sum of their magnitudes.  Roundings are counted one U each, products of
errors are left out and covered by rounding the counts up."""
import numpy as np

import moe_ref as R

U = R.U


def row_chain(cols):
    """Additions a column's term goes through in a row's sum, at most: in a thread's registers
    (32 elements) or, where a workgroup walks the row, cols / 256 of them, then over lanes and
    waves (16 or fewer)."""
    return min(cols, 32 + cols // 256) + 16


# ----- RMS norm ----------------------------------------------------------------------

def rms(a, b, gamma, eps):
    """h, r, y in 64 bits, and the relative bounds of r and y as fp32 numbers."""
    h = a if b is None else a + b
    cols = h.shape[1]
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        r = 1 / np.sqrt((h * h).mean(1) + eps)
        y = h * gamma * r[:, None]
    # sum of squares: h's rounding twice, the square's, the chain; the division by cols, eps's
    # rounding and addition 3; halved by the root; the root and the division 2 more
    rel_r = ((row_chain(cols) + 6) / 2 + 2) * U
    # h's rounding, two products
    return h, r, y, rel_r, rel_r + 3 * U


def scales_of(y, block, largest):
    """Scales [rows, blocks] and v = y / scale, in 64 bits; NaN where a value is none."""
    rows, cols = y.shape
    width = block or cols
    scales = np.empty((rows, -(-cols // width)))
    for i in range(scales.shape[1]):
        part = y[:, i * width:(i + 1) * width]
        scales[:, i] = np.maximum(np.abs(part).max(1), 2.0 ** -100) / largest
        scales[~np.isfinite(part).all(1), i] = np.nan
    with np.errstate(invalid="ignore"):
        v = y / np.repeat(scales, width, 1)[:, :cols]
    return scales, np.where(np.isnan(v), 0.0, v)


def code_values(q, fmt):
    return q.view(np.int8).astype(np.float64) if fmt == "int8" else R.E4M3[q.view(np.uint8)]


def code_bound(v, fmt):
    """Half a step at v, and the error of v in fp32: h gamma twice (its own and the largest
    one's), the quotient, the product, h's own twice: 6 U of v."""
    v = np.abs(v)
    if fmt == "int8":
        half = np.full(v.shape, 0.5)
    else:  # 4 significant bits, the smallest exponent -6: half a step
        half = np.exp2(np.floor(np.log2(np.maximum(v, 2.0 ** -6))) - 4)
        # just below a power of two the error of v may reach the next, wider step
        half = np.maximum(half, np.exp2(np.floor(np.log2(np.maximum(v * (1 + 8 * U), 2.0 ** -6))) - 4))
    return half + 8 * U * v


def rms_back(dy, x, r, gamma, old):
    """dx, dgamma in 64 bits and absolute bounds of both as fp32 computations."""
    rows, cols = x.shape
    n = x * r[:, None]
    g = dy * gamma
    m = (g * n).mean(1, keepdims=True)
    dx = r[:, None] * (g - n * m)
    # m: three roundings a term and the chain, the division
    em = (row_chain(cols) + 4) * U * np.abs(g * n).mean(1, keepdims=True)
    # r (g - n m): g 1, n 1, n m 1, the difference 1, the product 1
    b = np.abs(r)[:, None] * (5 * U * (np.abs(g) + np.abs(n * m)) + np.abs(n) * em)
    out = dx if old is None else old + dx
    if old is not None:
        b = b + U * np.abs(out)
    t = dy * n
    # n and the product 2; the rows of a group one after another, 512 / 16 groups and 32 + 16
    # partial rows at most, then the old value
    chain = rows // 256 + 100
    return out, b, t.sum(0), (chain + 3) * U * np.abs(t).sum(0)


# ----- balance loss -----------------------------------------------------------------------

def softmax(l):
    """p and a relative bound on it as an fp32 computation: the difference to the top and its
    product with log2 e are rounded (2 U of their size each way), exp2 is good to 2 U; their
    average enters through the sum, which has 16 additions in a lane and 6 over lanes."""
    p, rel = np.zeros(l.shape), np.zeros(l.shape)
    for i, row in enumerate(l):
        if np.isneginf(row).all():
            continue
        top = np.nan if np.isnan(row).any() else row.max()
        with np.errstate(invalid="ignore"):
            e = np.where(np.isneginf(row), 0.0, np.exp(row - top))
            p[i] = e / e.sum()
            d = np.where(np.isneginf(row), 0.0, np.abs(row - top))
            rel[i] = U * (4 * d + 4 * (np.where(p[i] > 0, p[i] * d, 0)).sum() + 32)
    return p, rel


def balance(l, ids, valid, k, coef):
    """counts, probs, loss, and bounds of the last two."""
    n_tokens, experts = l.shape
    live = np.ones(n_tokens, bool) if valid is None else valid != 0
    n = int(live.sum())
    p, rel = softmax(l)
    p, rel = p[live], rel[live]
    some = ids[live].reshape(-1)
    some = some[(some >= 0) & (some < experts)]
    counts = np.bincount(some, minlength=experts)
    probs = p.sum(0) / max(n, 1)
    # tokens of a lane one after another (16 or 64 a trip of each of 256 workgroups, of which 8 are
    # counted here), 4 + 8 lanes and waves, 256 partial rows
    chain = n_tokens // (256 * 8) + 280
    bound = (p * rel).sum(0) / max(n, 1) + (chain + 3) * U * probs
    scale = coef * experts / (k * max(n, 1))
    loss = scale * (counts * probs).sum()
    return (np.append(counts, n).astype(np.int32), probs, bound, loss,
            scale * (counts * bound).sum() + 4 * U * abs(loss))


def balance_back(l, valid, counts, dloss, k, coef):
    """dlogits (0 where a token is not valid) and a bound."""
    n_tokens, experts = l.shape
    live = np.ones(n_tokens, bool) if valid is None else valid != 0
    n = int(counts[-1])
    p, rel = softmax(l)
    c = counts[:-1].astype(np.float64)
    left = c - np.rint(c.mean())  # what the calls compute with: p adds up to 1
    d = (p * left).sum(1, keepdims=True)
    scale = dloss * coef * experts / k / max(n, 1) ** 2 if n else 0.0
    g = scale * p * (left - d)
    # left to within 1 (its mean may be rounded to either side) is exact; d by p's errors and
    # its sum's (24 additions); the difference, the factors 8
    ed = (p * (np.abs(left) + 1) * (rel + 32 * U)).sum(1, keepdims=True)
    size = np.abs(left).max() + 1
    b = abs(scale) * p * (ed + (rel + 12 * U) * (np.abs(left - d)) + 4 * U * size)
    g, b = np.where(live[:, None], g, 0), np.where(live[:, None], b, 0)
    return g, b


# ----- clipping ---------------------------------------------------------------------------

def norm_chain(total):
    """Additions of a square in fp32: a thread's part of its workgroup's elements (at least 2048
    workgroups, or 1024 over the launches of fewer than 2^24 elements, 256 where these are four and
    one has all; 256 threads with 4 sums each; whole units of 8192 elements), 8 sums, lanes and
    waves."""
    workgroups = 2048 if total >= 1 << 24 else 256
    return total // (workgroups * 256 * 4) + 8192 // (256 * 4) + 8 + 16
