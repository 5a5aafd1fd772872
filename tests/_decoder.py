"""Plain 64-bit forms of rotary positions, dropout, gated linear layers and cross entropy over a vocabulary, and bounds on
the rounding errors of float32 kernels."""
import math

import numpy as np

U32 = 2.0 ** -24  # half a step of float32, relative to the value
GATES = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")
_erfc = np.vectorize(math.erfc, otypes=[float])


# ------------------------------------------------------------------ rotary

def rotary(x, heads, dim, turned, interleaved, positions, frequencies, scale, inverse=False):
    y = x.astype(np.float64)
    angle = positions.astype(np.float64)[:, None, None] * frequencies
    c, s = scale * np.cos(angle), scale * np.sin(angle) * (-1 if inverse else 1)
    part = y[:, :heads * dim].reshape(len(y), heads, dim)[:, :, :turned].copy()
    u, v = (part[:, :, 0::2], part[:, :, 1::2]) if interleaved else (part[:, :, :turned // 2], part[:, :, turned // 2:])
    pair = u * c - v * s, v * c + u * s
    turned_part = np.stack(pair, 3).reshape(part.shape) if interleaved else np.concatenate(pair, 2)
    y[:, :heads * dim].reshape(len(y), heads, dim)[:, :, :turned] = turned_part
    return y


def rotary_bound(x, heads, dim, turned, interleaved, positions, frequencies, scale, unit=U32):
    """A value of float32 errs by: the angle's rounding, pi / 2 2^-26 < 0.4 units, and 2^-51 of the angle; 8 units for a
    sine or cosine (4 units in the last place are 8 halves), two for its scale and factor, two for product and sum: 16 in
    all, of u and v both.  In float64 (unit 2^-53) the same with numpy's own function in the place of the angle's error,
    and angles that round as numpy's do."""
    a = np.abs(x.astype(np.float64))
    angle = np.abs(positions.astype(np.float64)[:, None, None] * frequencies)
    part = a[:, :heads * dim].reshape(len(a), heads, dim)[:, :, :turned].copy()
    u, v = (part[:, :, 0::2], part[:, :, 1::2]) if interleaved else (part[:, :, :turned // 2], part[:, :, turned // 2:])
    e = abs(scale) * (u + v) * (16 * unit + (angle * 2.0 ** -51 if unit == U32 else 0))
    out = np.zeros(a.shape)
    out[:, :heads * dim].reshape(len(a), heads, dim)[:, :, :turned] = \
        np.stack((e, e), 3).reshape(part.shape) if interleaved else np.concatenate((e, e), 2)
    return out


# ----------------------------------------------------------------- dropout

def philox(counter, key):
    """Philox4x32-10 of arrays of four 32-bit words."""
    c, (k0, k1) = [np.asarray(w, np.uint64) for w in counter], key
    mask, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> half) ^ c[1] ^ np.uint64(k0), q & mask, (p >> half) ^ c[3] ^ np.uint64(k1), p & mask]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def kept(n, rate, seed, call):
    unit = np.arange(-(-n // 4), dtype=np.uint64)
    call = call % (1 << 64)
    words = philox((unit & np.uint64(0xFFFFFFFF), unit >> np.uint64(32), np.full(unit.shape, call & 0xFFFFFFFF, np.uint64),
                    np.full(unit.shape, call >> 32, np.uint64)), (seed & 0xFFFFFFFF, seed >> 32))
    return np.stack(words, 1).reshape(-1)[:n] >= np.uint64(round(rate * 2 ** 32))


# ------------------------------------------------------------ gated linear

def gate(name, a):
    """(act(a), act'(a), the magnitude of what the logistic or error function is taken of)"""
    if name == "gelu":
        s = 0.5 * _erfc(-a / math.sqrt(2))
        return a * s, s + a * np.exp(-a * a / 2) / math.sqrt(2 * math.pi), a * a
    if name == "relu":
        return np.maximum(a, 0), (a > 0) * 1.0, 0 * a
    c = math.sqrt(2 / math.pi)
    v = 2 * c * (a + 0.044715 * a ** 3) if name == "gelu_tanh" else a
    with np.errstate(over="ignore"):
        s, rest = 1 / (1 + np.exp(-v)), 1 / (1 + np.exp(v))
    if name == "sigmoid":
        return s, s * rest, np.abs(v)
    slope = 2 * c * (1 + 3 * 0.044715 * a * a) if name == "gelu_tanh" else 1
    return a * s, s + a * s * rest * slope, np.abs(v)


def gated(name, x, w, b, g=None):
    """h, and with g also dx, dw and db."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    pre = x @ w + (0 if b is None else b.astype(np.float64))
    n = w.shape[1] // 2
    a, u = pre[:, :n], pre[:, n:]
    act, slope, _ = gate(name, a)
    if g is None:
        return act * u
    g = g.astype(np.float64)
    d = np.concatenate((g * u * slope, g * act), 1)
    return act * u, d @ w.T, x.T @ d, d.sum(0)


def gated_bounds(name, x, w, b, g):
    """Bounds on the errors of (h, dx, dw, db) by counting roundings.

    A sum of k products errs by at most k + 16 units of its magnitudes: a rounding a term and 8 units for operands held
    in parts.  act and act' have slopes of at most 1.2 (except ReLU's act', whose inputs have to keep away from 0); they
    err besides by 64 units of |a| s or s, and where the function falls steeply by 4 units of its argument's magnitude
    (a^2 for the error function) of themselves."""
    x, w, g = (t.astype(np.float64) for t in (x, w, g))
    n = w.shape[1] // 2
    pre = x @ w + (0 if b is None else b.astype(np.float64))
    e = (x.shape[1] + 16) * U32 * (np.abs(x) @ np.abs(w)) + U32 * np.abs(pre)
    a, u, ea, eu = pre[:, :n], pre[:, n:], e[:, :n], e[:, n:]
    act, slope, steep = gate(name, a)
    unit = (64 + 4 * steep) * U32
    eact = 1.2 * ea + unit * np.abs(act)
    # act' is a sum of two terms: s, and one that is at most |a| (1 + |act'|) as large
    eslope = (0 if name == "relu" else 1.2 * ea) + unit * (np.abs(slope) + np.abs(act) * (1 + np.abs(a)))
    eh = eact * np.abs(u) + np.abs(act) * eu + 4 * U32 * np.abs(act * u)
    ga = np.abs(g)
    d = np.abs(np.concatenate((g * u * slope, g * act), 1))
    ed = np.concatenate((ga * (eu * np.abs(slope) + np.abs(u) * eslope), ga * eact), 1) * 1.01 + 4 * U32 * d
    wa, xa = np.abs(w), np.abs(x)
    return (eh, ed @ wa.T + (w.shape[1] + 16) * U32 * (d @ wa.T), xa.T @ ed + (len(x) + 16) * U32 * (xa.T @ d),
            ed.sum(0) + (len(x) + 16) * U32 * d.sum(0))


# ----------------------------------------------------------- cross entropy

def cross_entropy(x, w, b, targets, weights=None):
    """(loss, dx, dw, db) of the weighted sum of the losses.  Rows with a negative target take no part at all."""
    n, vocab = len(x), w.shape[1]
    rows = np.nonzero(targets >= 0)[0]
    loss, dx = np.zeros(n), np.zeros((n, x.shape[1]))
    with np.errstate(all="ignore"):
        xs, w = x[rows].astype(np.float64), w.astype(np.float64)
        z = xs @ w + (0 if b is None else b.astype(np.float64))
        top = z.max(1, keepdims=True)
        p = np.exp(z - top)
        total = p.sum(1, keepdims=True)
        t = targets[rows]
        bad = t >= vocab
        at = np.where(bad, 0, t)[:, None]
        loss[rows] = np.where(bad, np.nan, (np.log(total) - (np.take_along_axis(z, at, 1) - top))[:, 0])
        wt = np.ones(len(rows)) if weights is None else weights[rows].astype(np.float64)
        d = p / total * wt[:, None]
        np.put_along_axis(d, at, np.take_along_axis(d, at, 1) - wt[:, None], 1)
        d[bad] = np.nan
        dx[rows] = d @ w.T
        return loss, dx, xs.T @ d, d.sum(0)


def cross_entropy_bounds(x, w, b, targets, weights=None):
    """Bounds on the errors of (loss, dx, dw, db) for finite operands and targets inside the vocabulary.

    A logit errs as a sum of k products does (gated_bounds).  Exponents and their sum err by the logits' error, the
    rounding of z - max (a unit of it) and at most vocab / 64 + 64 roundings: a lane's terms, the lanes, the waves and
    the parts of a row."""
    rows = np.nonzero(targets >= 0)[0]
    out = np.zeros(len(x)), np.zeros(x.shape)
    xs, w = x[rows].astype(np.float64), w.astype(np.float64)
    z = xs @ w + (0 if b is None else b.astype(np.float64))
    xa, wa, k = np.abs(xs), np.abs(w), w.shape[0]
    ez = (k + 16) * U32 * (xa @ wa) + 2 * U32 * np.abs(z)
    top = z.max(1, keepdims=True)
    p = np.exp(z - top)
    total = p.sum(1, keepdims=True)
    p = p / total
    worst, spread = ez.max(1), (top - z).max(1)
    rel = worst + (w.shape[1] / 64 + 64 + spread) * U32
    t = targets[rows][:, None]
    loss = (np.log(total) - (np.take_along_axis(z, t, 1) - top))[:, 0]
    away = np.abs(np.take_along_axis(z, t, 1) - top)[:, 0]
    out[0][rows] = worst + rel + 4 * U32 * (loss + away)
    wt = np.ones(len(rows)) if weights is None else np.abs(weights[rows].astype(np.float64))
    d = p * wt[:, None]
    ed = d * (2 * rel + 8 * U32)[:, None]
    hit = np.zeros_like(d)
    np.put_along_axis(hit, t, wt[:, None], 1)
    ed, d = ed + 2 * U32 * hit, d + hit
    out[1][rows] = ed @ wa.T + (w.shape[1] + 16) * U32 * (d @ wa.T)
    return out[0], out[1], xa.T @ ed + (len(rows) + 16) * U32 * (xa.T @ d), ed.sum(0) + (len(rows) + 16) * U32 * d.sum(0)
