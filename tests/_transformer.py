"""Plain 64-bit forms of layer norm, AdamW and packed attention, and bounds on the rounding errors of float32 kernels."""
import numpy as np

U32 = 2.0 ** -24  # half a step of float32, relative to the value


def layer_norm(x, w, b, eps):
    x = x.astype(np.float64)
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    z = (x - mean) * rstd
    y = z * (1 if w is None else w.astype(np.float64)) + (0 if b is None else b.astype(np.float64))
    return y, mean[:, 0], rstd[:, 0]


def layer_norm_backward(g, x, w, eps):
    g, x = g.astype(np.float64), x.astype(np.float64)
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    z = (x - mean) * rstd
    u = g * (1 if w is None else w.astype(np.float64))
    dx = rstd * (u - u.mean(1, keepdims=True) - z * (u * z).mean(1, keepdims=True))
    return dx, (g * z).sum(0), g.sum(0)


def adamw(p, g, m, v, t, lr, beta1, beta2, eps, decay):
    p, g, m, v = (a.astype(np.float64) for a in (p, g, m, v))
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    mh, vh = m / (1 - beta1 ** t), v / (1 - beta2 ** t)
    return p * (1 - lr * decay) - lr * mh / (np.sqrt(vh) + eps), m, v


def mixed(x):
    """MurmurHash3's 32-bit finalizer."""
    x = np.asarray(x, np.uint64) & 0xFFFFFFFF
    x ^= x >> 16
    x = (x * 0x85EBCA6B) & 0xFFFFFFFF
    x ^= x >> 13
    x = (x * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(n, tensor, t, seed):
    key = mixed((t ^ (seed & 0xFFFFFFFF)) & 0xFFFFFFFF)
    key = mixed((int(key) + 0x9E3779B9 * (tensor + 1)) & 0xFFFFFFFF)
    return mixed(np.arange(n, dtype=np.uint64) ^ key)


def blocks(x, size=256):
    n = -(-len(x) // size) * size
    return np.pad(x, (0, n - len(x))).reshape(-1, size)


def decode(codes, scales, q):
    c = blocks(codes).astype(np.float64)
    return (np.sign(c) * (c / q) ** 2 * scales.astype(np.float64)[:, None]).reshape(-1)[:len(codes)]


def attention(q, k, v, ql, kl, heads, kv_heads, scale, causal, g=None):
    """o, lse and, with g, dq, dk and dv.  Rows of sequences one after another, [rows, heads * d].  Masked places take no
    part at all: what they hold, infinities and NaN too, reaches nothing."""
    d = q.shape[1] // heads
    q, k, v = (a.astype(np.float64).reshape(len(a), a.shape[1] // d, d) for a in (q, k, v))
    o, lse = np.zeros_like(q), np.full((len(q), heads), -np.inf)
    if g is not None:
        g = g.astype(np.float64).reshape(q.shape)
        dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    q0 = k0 = 0
    with np.errstate(all="ignore"):
        for lq, lk in zip(ql, kl):
            for h in range(heads):
                c = h // (heads // kv_heads)
                for i in range(lq):
                    n = min(max(i + 1 + lk - lq, 0), lk) if causal else lk
                    if n == 0:
                        continue
                    ks, vs, qi = k[k0:k0 + n, c], v[k0:k0 + n, c], q[q0 + i, h]
                    s = ks @ qi * scale
                    top = s.max() if s.max() > -np.inf else 0.0
                    p = np.exp(s - top)
                    z = p.sum()
                    lse[q0 + i, h] = top + np.log(z)
                    p = p / z if z != 0 else p
                    o[q0 + i, h] = p @ vs
                    if g is not None:
                        gi = g[q0 + i, h]
                        dp = vs @ gi
                        ds = p * (dp - gi @ o[q0 + i, h]) * scale
                        dq[q0 + i, h] = ds @ ks
                        dk[k0:k0 + n, c] += np.outer(ds, qi)
                        dv[k0:k0 + n, c] += np.outer(p, gi)
            q0, k0 = q0 + lq, k0 + lk
    flat = lambda a: a.reshape(len(a), a.shape[1] * d)  # noqa: E731
    return (flat(o), lse) if g is None else (flat(o), lse, flat(dq), flat(dk), flat(dv))


def layer_norm_bounds(g, x, w, b, eps):
    """Bounds on the float32 errors of (y, mean, rstd, dx, dw, db), by counting roundings.

    A row's sum of n values runs over at most 32 values of a lane, 6 lane exchanges, 8 waves, and a multiplication by the
    rounded 1 / n: fewer than 56 roundings, each at most half a step of the sum of magnitudes; 64 below leaves 8 for what
    is done to the sum next.  z inherits the mean's error times rstd."""
    x = x.astype(np.float64)
    w64 = np.ones(x.shape[1]) if w is None else np.abs(w.astype(np.float64))
    b64 = np.zeros(x.shape[1]) if b is None else np.abs(b.astype(np.float64))
    e = 64 * U32
    xa = np.abs(x).mean(1, keepdims=True)
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    z = np.abs(x - mean) * rstd
    dz = e * (rstd * xa + z)                       # of z, whose rstd errs by e z at most too
    out = dict(y=dz * w64 + e * (z * w64 + b64), mean=e * xa[:, 0],
               rstd=rstd[:, 0] * e * (2 + rstd * xa)[:, 0])
    if g is not None:
        ga = np.abs(g.astype(np.float64))
        u = ga * w64
        av = lambda t: t.mean(1, keepdims=True)  # noqa: E731
        e2 = e * av(u * z) + av(u * dz)            # of avg(u z)
        out["dx"] = rstd * (e * (u + 2 * av(u)) + z * e2 + dz * av(u * z) + 2 * e * z * av(u * z)) \
            + e * (2 + rstd * xa) * rstd * (u + av(u) + z * av(u * z))
        # rows add up in a lane (at most rows / 256 + 1 of them), then 16 groups, 16 partials a lane, 5 halvings
        er = (64 + len(x) / 256) * U32
        out["dw"] = (ga * dz).sum(0) + er * (ga * z).sum(0)
        out["db"] = er * ga.sum(0)
    return out


def attention_bounds(q, k, v, ql, kl, heads, kv_heads, scale, causal, g=None):
    """Bounds on the errors of (o, lse, dq, dk, dv) for finite inputs, by counting roundings.

    A score is a sum of d products; each product may lose 8 units (two operands held to 2^-23 and a term of 2^-22 left
    out, the split-fp16 form) and the sum d; 16 in all besides d.  A weight 2^(s - base) errs by the error of its exponent
    and 4 roundings; sums over n keys or queries add n."""
    d = q.shape[1] // heads
    shape = lambda a: np.asarray(a, np.float64).reshape(len(a), a.shape[1] // d, d)  # noqa: E731
    q, k, v = shape(q), shape(k), shape(v)
    g = None if g is None else shape(g)
    eo, el = np.zeros_like(q), np.zeros((len(q), heads))
    eq, ek, ev = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    u, q0, k0 = U32, 0, 0
    for lq, lk in zip(ql, kl):
        if lq and lk:
            seen = np.arange(lk)[None] <= np.arange(lq)[:, None] + lk - lq if causal else np.ones((lq, lk), bool)
            for h in range(heads):
                c = h // (heads // kv_heads)
                qs, ks, vs = q[q0:q0 + lq, h], k[k0:k0 + lk, c], v[k0:k0 + lk, c]
                s = np.where(seen, qs @ ks.T * scale, -np.inf)
                top = s.max(1, keepdims=True)
                top = np.where(np.isfinite(top), top, 0)
                p = np.exp(s - top)
                z = p.sum(1, keepdims=True)
                p = p / np.where(z > 0, z, 1)
                ds = scale * (d + 16) * u * (np.abs(qs) @ np.abs(ks).T) + 4 * u * (np.abs(np.where(seen, s, 0)) + np.abs(top))
                worst = np.where(seen, ds, 0).max(1, keepdims=True)
                rel = 2 * worst + (lk + 16) * u       # of a normalised weight, p's own error and the sum's
                va = np.abs(vs)
                eo[q0:q0 + lq, h] = rel * (p @ va) + (lk + 16) * u * (p @ va)
                el[q0:q0 + lq, h] = (worst + (lk + 16) * u + 4 * u * (np.abs(top) + np.log(np.maximum(z, 1))))[:, 0]
                if g is not None:
                    gs = g[q0:q0 + lq, h]
                    ga, o = np.abs(gs), p @ vs
                    relp = rel + worst + el[q0:q0 + lq, h][:, None]   # of p formed again from lse
                    ev[k0:k0 + lk, c] += (p * (relp + (lq * heads + 16) * u)).T @ ga
                    dp = gs @ vs.T
                    delta = (gs * o).sum(1, keepdims=True)
                    edp = (d + 16) * u * (ga @ va.T)
                    ede = (d + 16) * u * (ga * np.abs(o)).sum(1, keepdims=True) + (ga * eo[q0:q0 + lq, h]).sum(1, keepdims=True)
                    size = p * (np.abs(dp) + np.abs(delta))
                    eds = p * (edp + ede) + size * (relp + 16 * u)
                    eq[q0:q0 + lq, h] = scale * (eds @ np.abs(ks) + (lk + 16) * u * (size @ np.abs(ks)))
                    ek[k0:k0 + lk, c] += scale * (eds + (lq * heads + 16) * u * size).T @ np.abs(qs)
        q0, k0 = q0 + lq, k0 + lk
    flat = lambda a: a.reshape(len(a), a.shape[1] * d)  # noqa: E731
    return (flat(eo), el) if g is None else (flat(eo), el, flat(eq), flat(ek), flat(ev))
