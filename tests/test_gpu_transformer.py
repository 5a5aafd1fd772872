"""Layer norm, AdamW and packed attention through the C ABI, against plain 64-bit forms (tests/_transformer.py).

Tolerances count roundings (the bounds in _transformer.py); codes of 8-bit states have to be equal, since they are a
function of float32 operations that round once each."""
import ctypes as C

import numpy as np
import pytest

import _transformer as T

pytestmark = pytest.mark.gpu


def up(hip, a):
    return hip.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


def padded(a, ld, fill=np.nan):
    """The rows of `a` in rows of ld values; what lies between them must not be read into results or written."""
    out = np.full((a.shape[0], ld), fill, a.dtype)
    out[:, :a.shape[1]] = a
    return out


def close(got, want, bound, what=""):
    err = np.abs(got.astype(np.float64) - want)
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(err[bad].max()), float(np.broadcast_to(bound, err.shape)[bad].min()))


# ------------------------------------------------------------- layer norm

NORM_SHAPES = [(1, 1), (3, 2), (5, 7), (1, 16), (33, 64), (19, 65), (130, 200), (64, 256), (9, 257), (40, 768), (17, 1000),
               (4, 1024), (6, 1031), (3, 2048), (5, 2049), (7, 3001), (2, 4096), (3, 5000), (2, 8192), (3, 8193),
               (2, 16384), (3, 16385), (1, 40000), (4097, 64), (2000, 768), (1500, 1030)]


def norm(hip, x, w, b, eps, ldx=None, ldy=None):
    rows, n = x.shape
    ldx, ldy = ldx or n, ldy or n
    dx, dw, db = up(hip, padded(x, ldx)), None if w is None else up(hip, w), None if b is None else up(hip, b)
    y = up(hip, np.full((rows, ldy), 7, x.dtype))
    mean, rstd = (hip.DeviceBuffer((rows,), x.dtype) for _ in range(2))
    hip.check(hip.lib().lmp_k_layer_norm(dx.code, rows, n, dx.ptr, ldx, dw and dw.ptr, db and db.ptr, eps, y.ptr, ldy,
                                         mean.ptr, rstd.ptr))
    out = y.numpy()
    assert (out[:, n:] == 7).all()
    return out[:, :n], mean, rstd, dx, dw


def norm_back(hip, g, dx, ldx, dw, mean, rstd, ldg=None, lddx=None, want=(True, True, True)):
    rows, n = g.shape
    ldg, lddx = ldg or n, lddx or n
    dg = up(hip, padded(g, ldg))
    outs = [up(hip, np.full(s, 7, g.dtype)) for s in ((rows, lddx), (n,), (n,))]
    ptr = [o.ptr if t else None for o, t in zip(outs, want)]
    hip.check(hip.lib().lmp_k_layer_norm_backward(dg.code, rows, n, dg.ptr, ldg, dx.ptr, ldx, dw and dw.ptr, mean.ptr,
                                                  rstd.ptr, ptr[0], lddx, ptr[1], ptr[2]))
    got = [o.numpy() for o in outs]
    assert (got[0][:, n:] == 7).all()
    for o, t in zip(got, want):
        assert t or (o == 7).all()
    return got[0][:, :n], got[1], got[2]


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,n", NORM_SHAPES)
def test_layer_norm(hip, rows, n, dtype):
    rng = np.random.default_rng(rows * 100003 + n)
    x = (rng.standard_normal((rows, n)) + 0.5).astype(dtype)
    w, b = (1 + 0.1 * rng.standard_normal(n)).astype(dtype), (0.1 * rng.standard_normal(n)).astype(dtype)
    g = (0.1 * rng.standard_normal((rows, n))).astype(dtype)
    eps, scale = 1e-5, 1 if dtype == np.float32 else 2.0 ** -29  # half a step of float64 is 2^-53
    ldx, ldy = n + rows % 3, n + n % 2
    y, mean, rstd, dx, dw = norm(hip, x, w, b, eps, ldx, ldy)
    bound = T.layer_norm_bounds(g, x, w, b, eps)
    wy, wm, wr = T.layer_norm(x, w, b, eps)
    long = 1 + n / 16384  # rows past the registers: more values a lane
    # The 64-bit form rounds too, by what numpy's pairwise sums lose.
    slack = 64 * 2.0 ** -53 if dtype == np.float64 else 0
    close(y, wy, long * scale * bound["y"] + slack * np.abs(wy), "y")
    close(mean.numpy(), wm, long * scale * bound["mean"], "mean")
    close(rstd.numpy(), wr, long * scale * bound["rstd"] + slack * wr, "rstd")
    gx, gw, gb = norm_back(hip, g, dx, ldx, dw, mean, rstd, n + 1, n + 2)
    wx, ww, wb = T.layer_norm_backward(g, x, w, eps)
    close(gx, wx, long * scale * bound["dx"], "dx")
    rows_long = 1 + (rows / 64 if n > 8192 else 0)  # long rows: a lane per column runs over its rows
    close(gw, ww, rows_long * long * scale * bound["dw"], "dw")
    close(gb, wb, rows_long * scale * bound["db"], "db")


def test_layer_norm_without_weights_in_place_and_parts_of_the_backward(hip):
    rng = np.random.default_rng(5)
    for rows, n in ((6, 40), (5, 700), (3, 9000), (2, 20000)):
        x, g = rng.standard_normal((rows, n)).astype(np.float32), rng.standard_normal((rows, n)).astype(np.float32)
        bound = T.layer_norm_bounds(g, x, None, None, 0.0)
        y, mean, rstd, dx, _ = norm(hip, x, None, None, 0.0)
        close(y, T.layer_norm(x, None, None, 0.0)[0], 2 * bound["y"])
        full = norm_back(hip, g, dx, n, None, mean, rstd)
        for want in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
            got = norm_back(hip, g, dx, n, None, mean, rstd, want=want)
            for a, f, t in zip(got, full, want):
                assert not t or np.array_equal(a, f)
        # y over x, statistics not asked for; dx over g, all gradients asked for
        hip.check(hip.lib().lmp_k_layer_norm(hip.FLOAT32, rows, n, dx.ptr, n, None, None, 0.0, dx.ptr, n, None, None))
        assert np.array_equal(dx.numpy(), y)
        dx, dg = up(hip, x), up(hip, g)
        hip.check(hip.lib().lmp_k_layer_norm_backward(hip.FLOAT32, rows, n, dg.ptr, n, dx.ptr, n, None, mean.ptr, rstd.ptr,
                                                      dg.ptr, n, None, None))
        assert np.array_equal(dg.numpy(), full[0])
        dw, db = hip.DeviceBuffer((n,)), hip.DeviceBuffer((n,))
        for over in (up(hip, x), up(hip, g)):
            dx, dg = (over, up(hip, g)) if np.array_equal(over.numpy(), x) else (up(hip, x), over)
            hip.check(hip.lib().lmp_k_layer_norm_backward(hip.FLOAT32, rows, n, dg.ptr, n, dx.ptr, n, None, mean.ptr,
                                                          rstd.ptr, over.ptr, n, dw.ptr, db.ptr))
            for a, f in zip((over, dw, db), full):
                assert np.array_equal(a.numpy(), f)


def test_layer_norm_constant_and_special_rows(hip):
    """A constant row has var 0 exactly where its sum is exact; a row with an infinity or NaN is NaN and touches no other."""
    for n in (8, 300, 3000, 20000):
        x = np.random.default_rng(n).standard_normal((6, n)).astype(np.float32)
        x[1] = 2.0
        x[2, n // 2] = np.inf
        x[3, n - 1] = np.nan
        y, mean, rstd, _, _ = norm(hip, x, None, None, 1e-5)
        assert (y[1] == 0).all() and mean.numpy()[1] == 2.0
        assert abs(rstd.numpy()[1] - 1e5 ** 0.5) < 1e5 ** 0.5 * 4 * T.U32
        assert np.isnan(y[2]).all() and np.isnan(y[3]).all()
        for r in (0, 4, 5):
            assert np.array_equal(y[r], norm(hip, x[r:r + 1], None, None, 1e-5)[0][0])


def test_layer_norm_gradients_of_a_row_of_67_million(hip):
    """Past 2^26 columns a lane per value and partial would pass 2^32 threads a grid."""
    n = (1 << 26) + 70
    rng = np.random.default_rng(1)
    x, g = rng.standard_normal((1, n), np.float32), rng.standard_normal((1, n), np.float32)
    dx, dg, dw, db = up(hip, x), up(hip, g), hip.DeviceBuffer((n,)), hip.DeviceBuffer((n,))
    mean, rstd = up(hip, np.array([0.25], np.float32)), up(hip, np.array([2.0], np.float32))
    hip.check(hip.lib().lmp_k_layer_norm_backward(hip.FLOAT32, 1, n, dg.ptr, n, dx.ptr, n, None, mean.ptr, rstd.ptr, None, 0,
                                                  dw.ptr, db.ptr))
    assert np.array_equal(db.numpy(), g[0])
    want = g[0].astype(np.float64) * (x[0].astype(np.float64) - 0.25) * 2
    bound = 3 * T.U32 * np.abs(g[0]) * (np.abs(x[0]) + 0.25) * 2
    close(dw.numpy(), want, bound)


def test_layer_norm_backward_of_no_rows(hip):
    out = [up(hip, np.full(700, 7, np.float32)) for _ in range(2)]
    hip.check(hip.lib().lmp_k_layer_norm_backward(hip.FLOAT32, 0, 700, None, 0, None, 0, None, None, None, None, 0,
                                                  out[0].ptr, out[1].ptr))
    assert not out[0].numpy().any() and not out[1].numpy().any()


# ------------------------------------------------------------------ AdamW

HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)


def adamw_case(rng, n):
    return ((0.02 * rng.standard_normal(n)).astype(np.float32), (2e-3 * rng.standard_normal(n)).astype(np.float32),
            (1e-3 * rng.standard_normal(n)).astype(np.float32), ((1e-3 * rng.standard_normal(n)) ** 2 + 1e-8).astype(np.float32))


def adamw_call(hip, bits, tensors, decays, step, seed=0, hyper=HYPER):
    """tensors: lists of device buffers (p, g, m, v[, m_scale, v_scale]) and value counts."""
    arr = (hip.AdamWTensor * max(1, len(tensors)))(*[
        hip.AdamWTensor(*[b.ptr for b in t[0][:4]], *([b.ptr for b in t[0][4:]] or [None, None]), t[1], d)
        for t, d in zip(tensors, decays)])
    hip.check(hip.lib().lmp_k_adamw_f32(bits, len(tensors), C.cast(arr, C.c_void_p), hyper["lr"], hyper["beta1"],
                                        hyper["beta2"], hyper["eps"], seed, step.ptr))


@pytest.mark.parametrize("sizes", [[1], [5, 0, 3], [4096], [4097, 1, 255, 256, 257], list(range(1, 120)),
                                   [1 << 20, 7, (1 << 20) + 3]], ids=lambda s: f"{len(s)}x{max(s)}")
def test_adamw_32(hip, sizes):
    rng = np.random.default_rng(len(sizes) * 7 + max(sizes))
    host = [adamw_case(rng, n) for n in sizes]
    # the third tensor on is one value into its allocation: no alignment beyond a value's own
    dev = [([up(hip, np.concatenate([[9], a]).astype(np.float32)) for a in h], n) for h, n in zip(host, sizes)]
    for i, (bufs, _) in enumerate(dev):
        for b in bufs:
            b.base, b.ptr = b.ptr, b.ptr + 4
    decays = [0.01 * (i % 2) for i in range(len(sizes))]
    step = up(hip, np.array([4, 0], np.int64))
    state = [tuple(a.astype(np.float64) for a in h) for h in host]
    bounds = [[np.zeros(n) for _ in range(3)] for n in sizes]
    for t in (5, 6):
        adamw_call(hip, 32, dev, decays, step)
        for i, (p, g, m, v) in enumerate(state):
            p2, m2, v2 = T.adamw(p, g, m, v, t, decay=decays[i], **HYPER)
            bp, bm, bv = bounds[i]
            bm = 0.9 * bm + 4 * T.U32 * (0.9 * abs(m) + 0.1 * abs(g))
            bv = 0.999 * bv + 5 * T.U32 * v2
            den = np.sqrt(v2 / (1 - 0.999 ** t)) + 1e-8
            size = 1e-3 / (1 - 0.9 ** t)
            bp = bp + 3 * T.U32 * (abs(p) + abs(p2)) + size / den * (bm + abs(m2) * (8 * T.U32 + 0.51 * bv / v2))
            bounds[i], state[i] = [bp, bm, bv], (p2, g, m2, v2)
        assert step.numpy().tolist() == [t, 0]
    for i, (bufs, n) in enumerate(dev):
        for j, which in ((0, 0), (2, 1), (3, 2)):
            b = bufs[j]
            b.ptr = b.base
            got = b.numpy()
            assert got[0] == 9
            close(got[1:], state[i][j], bounds[i][which], (i, j))
            b.ptr = b.base + 4
        bufs[1].ptr = bufs[1].base
    for bufs, _ in dev:
        for b in bufs:
            b.ptr = b.base


def encode32(x, q, r):
    """The codes' definition in float32, each operation rounded once, as the header words it."""
    f = np.float32
    xb, rb = T.blocks(x), T.blocks(r)
    with np.errstate(all="ignore"):
        top = np.abs(xb).max(1)
        live = (top >= f(1e-30)) & (top < np.inf)
        scale = np.where(live, top, np.where(top < f(1e-30), f(0), f(np.nan))).astype(f)
        inv = np.where(live, (f(1) / np.where(live, top, f(1))) * f(q * q), f(0)).astype(f)
        t = np.where(live[:, None], np.minimum(np.abs(xb) * inv[:, None], f(q * q)), f(0)).astype(f)
        c = np.floor(np.sqrt(t))
        c = np.where(c * c > t, c - 1, c)
        c = np.where((c + 1) * (c + 1) <= t, c + 1, c)
        c = np.where(rb.astype(f) * f(1 / 65536) * (2 * c + 1) < t - c * c, c + 1, c)
        if q == 255:
            c = np.where((c == 0) & (t > 0), f(1), c)
        c = np.where(xb < 0, -c, c)
    return np.clip(c, -q, q).reshape(-1)[:len(x)].astype(np.int64), scale


def states8(rng, n):
    p, g, m, v = adamw_case(rng, n)
    mc, ms = encode32(m, 127, np.zeros(n, np.uint64))
    vc, vs = encode32(v, 255, np.zeros(n, np.uint64))
    return p, g, mc.astype(np.int8), vc.astype(np.uint8), ms, vs


class Bytes:
    """Codes on the device (the binding's buffers are of the framework's own types)."""

    def __init__(self, hip, a, offset=0):
        self.n, self.offset, self.dtype = len(a), offset, a.dtype
        raw = np.concatenate([np.full(offset, 77, np.uint8), a.view(np.uint8), np.full(8, 77, np.uint8)])
        raw = np.pad(raw, (0, -len(raw) % 4), constant_values=77)
        self.buf = up(hip, raw.view(np.int32))
        self.ptr = self.buf.ptr + offset

    def numpy(self):
        raw = self.buf.numpy().view(np.uint8)
        assert (raw[:self.offset] == 77).all() and (raw[self.offset + self.n:] == 77).all()
        return raw[self.offset:self.offset + self.n].view(self.dtype)


@pytest.mark.parametrize("sizes", [[1], [255, 0, 256], [257, 4096, 4099], list(range(200, 260)), [100003]],
                         ids=lambda s: f"{len(s)}x{max(s)}")
def test_adamw_8(hip, sizes):
    f = np.float32
    rng = np.random.default_rng(11 + len(sizes) + max(sizes))
    host = [states8(rng, n) for n in sizes]
    host = [list(h) for h in host]
    dev = [([up(hip, h[0]), up(hip, h[1]), Bytes(hip, h[2], i % 3), Bytes(hip, h[3], i % 2), up(hip, h[4]), up(hip, h[5])], n)
           for i, (h, n) in enumerate(zip(host, sizes))]
    step = up(hip, np.array([9, 0], np.int64))
    for t in (10, 11):
        adamw_call(hip, 8, dev, [0.0] * len(sizes), step, seed=12345678901)
        for i, (h, (bufs, n)) in enumerate(zip(host, dev)):
            if n == 0:
                continue
            p, g, mc, vc, ms, vs = h
            unit = lambda codes, s, q: ((codes * np.abs(codes)).astype(f)  # noqa: E731
                                        * np.repeat(s * f(1 / (q * q)), 256)[:n])
            m = unit(mc.astype(f), ms, 127) * f(0.9) + g * f(1 - 0.9)
            v = unit(vc.astype(f), vs, 255) * f(0.999) + (g * g) * f(1 - 0.999)
            r = T.random_bits(n, i, t, 12345678901)
            mc2, ms2 = encode32(m, 127, r & 0xFFFF)
            vc2, vs2 = encode32(v, 255, r >> 16)
            want = T.adamw(p, g, T.decode(mc, ms, 127), T.decode(vc, vs, 255), t, decay=0.0, **HYPER)
            got = [b.numpy() for b in bufs]
            assert np.array_equal(got[4], ms2) and np.array_equal(got[5], vs2), (t, i)
            assert np.array_equal(got[2].astype(np.int64), mc2), (t, i)
            assert np.array_equal(got[3].astype(np.int64), vc2), (t, i)
            # the parameter sees the moments before they are rounded to codes
            den = np.sqrt(want[2] / (1 - 0.999 ** t)) + 1e-8
            em = 6 * T.U32 * (0.9 * np.abs(T.decode(mc, ms, 127)) + 0.1 * np.abs(g))
            close(got[0], want[0], 3 * T.U32 * (abs(p) + abs(want[0])) + 1e-3 / (1 - 0.9 ** t) / den * (em + 16 * T.U32 * abs(want[1])), (t, i))
            for j, (code, scale, q) in enumerate(((2, 4, 127), (3, 5, 255))):
                out = hip.DeviceBuffer((n,), f)
                hip.check(hip.lib().lmp_k_adamw_decode(int(j == 0), bufs[code].ptr, bufs[scale].ptr, n, out.ptr))
                full = T.decode(got[code], got[scale], q)
                close(out.numpy(), full, 4 * T.U32 * np.abs(full), "decode")
            h[0], h[2], h[3], h[4], h[5] = got[0].copy(), got[2].copy(), got[3].copy(), got[4], got[5]
        assert step.numpy().tolist() == [t, 0]


def test_adamw_8_rounding_is_fair(hip):
    """One gradient of many equal values below a step of the codes: the mean of the decoded first moments is the value."""
    n = 1 << 16
    g = np.full(n, 1e-4, np.float32)
    g[::256] = 1e-2  # each block's scale
    zeros = np.zeros(n, np.float32)
    dev = [([up(hip, zeros), up(hip, g), Bytes(hip, np.zeros(n, np.int8)), Bytes(hip, np.zeros(n, np.uint8)),
             up(hip, zeros[:n // 256]), up(hip, zeros[:n // 256])], n)]
    step = up(hip, np.zeros(2, np.int64))
    adamw_call(hip, 8, dev, [0.0], step, seed=3)
    small = np.arange(n) % 256 != 0
    m = T.decode(dev[0][0][2].numpy(), dev[0][0][4].numpy(), 127)[small]
    # values at c^2 or (c + 1)^2 steps of 1e-3 / 127^2 around 1e-5: spread below half their distance
    c = np.floor(127 * 0.1)
    spread = (2 * c + 1) / 127 ** 2 * 1e-3 / 2
    assert abs(m.mean() - 1e-5) < 5 * spread / np.sqrt(small.sum())
    # a second moment above zero is never lost
    assert (dev[0][0][3].numpy() > 0).all()


def test_adamw_8_special_blocks(hip):
    """Blocks of zeros keep scale 0; a block whose gradient holds a NaN or infinity stores NaN; its neighbours do not see it."""
    n = 256 * 4
    rng = np.random.default_rng(2)
    p, g, mc, vc, ms, vs = states8(rng, n)
    g[256:512] = 0
    mc[256:512] = vc[256:512] = 0
    ms[1] = vs[1] = 0
    g[512] = np.inf
    g[800] = np.nan
    dev = [([up(hip, p), up(hip, g), Bytes(hip, mc), Bytes(hip, vc), up(hip, ms), up(hip, vs)], n)]
    adamw_call(hip, 8, dev, [0.0], up(hip, np.zeros(2, np.int64)), seed=3)
    got = [b.numpy() for b in dev[0][0]]
    assert np.array_equal(got[0][256:512], p[256:512]) and got[4][1] == 0 and got[5][1] == 0
    for b in (2, 3):
        assert np.isnan(got[4][b]) and np.isnan(got[5][b])
        assert not got[2][b * 256:(b + 1) * 256].any() and not got[3][b * 256:(b + 1) * 256].any()
    assert np.isfinite(got[0][:512]).all() and np.isfinite(got[4][:2]).all()


def test_adamw_step_of_nothing_counts(hip):
    step = up(hip, np.array([7, 0], np.int64))
    hip.check(hip.lib().lmp_k_adamw_f32(32, 0, None, 1e-3, 0.9, 0.999, 1e-8, 0, step.ptr))
    assert step.numpy().tolist() == [8, 0]


# -------------------------------------------------------------- attention

def attend(hip, ql, kl, heads, kv, d, causal, q, k, v, scale, g=None, pad=0):
    """(o, lse[, dq, dk, dv]) with rows `pad` values longer than their heads; what lies between rows stays as it was."""
    plan = hip.AttentionPlan(ql, kl, heads=heads, kv_heads=kv, head_dim=d, causal=causal)
    L, qw, kw = hip.lib(), heads * d, kv * d
    dq_, dk_, dv_ = (up(hip, padded(a, w + pad)) for a, w in ((q, qw), (k, kw), (v, kw)))
    new = lambda rows, w: up(hip, np.full((rows, w + pad), 7, np.float32))  # noqa: E731
    o, lse = new(len(q), qw), up(hip, np.full((len(q), heads), 7, np.float32))
    hip.check(L.lmp_k_attention_f32(plan.handle, dq_.ptr, qw + pad, dk_.ptr, kw + pad, dv_.ptr, kw + pad, scale, o.ptr,
                                    qw + pad, lse.ptr))
    outs = [o]
    if g is not None:
        dg, gq, gk, gv = up(hip, padded(g, qw + pad)), new(len(q), qw), new(len(k), kw), new(len(k), kw)
        hip.check(L.lmp_k_attention_backward_f32(
            plan.handle, dq_.ptr, qw + pad, dk_.ptr, kw + pad, dv_.ptr, kw + pad, scale, o.ptr, qw + pad, lse.ptr, dg.ptr,
            qw + pad, gq.ptr, qw + pad, gk.ptr, kw + pad, gv.ptr, kw + pad))
        outs += [gq, gk, gv]
    got = []
    for a, w in zip(outs, (qw, qw, kw, kw)):
        a = a.numpy()
        assert (a[:, w:] == 7).all()
        got.append(a[:, :w])
    return [got[0], lse.numpy()] + got[1:]


def attention_inputs(rng, ql, kl, heads, kv, d):
    f = lambda rows, w: rng.standard_normal((rows, w)).astype(np.float32)  # noqa: E731
    return f(sum(ql), heads * d), f(sum(kl), kv * d), f(sum(kl), kv * d), f(sum(ql), heads * d)


ATTENTION = [
    # query lengths, key lengths, heads, kv heads, dim, causal
    ([1], [1], 1, 1, 1, True), ([1], [1], 4, 2, 64, True), ([2], [2], 1, 1, 3, True), ([16], [16], 2, 2, 32, True),
    ([17], [17], 3, 1, 80, True), ([33], [33], 4, 4, 64, False), ([100], [100], 6, 2, 96, True),
    ([130], [130], 2, 2, 128, True), ([65], [65], 2, 1, 33, True), ([40], [40], 1, 1, 130, True),
    ([20], [20], 2, 1, 256, False), ([31], [31], 5, 1, 48, True), ([24], [24], 2, 2, 100, True),
    # packed batches, sequences without queries or keys among them
    ([5, 0, 64, 1, 33], [5, 0, 64, 1, 33], 4, 2, 64, True), ([3, 0, 7], [0, 5, 7], 2, 2, 16, True),
    ([0, 0], [0, 0], 2, 1, 8, True), ([4], [0], 2, 1, 8, False),
    # chunks: the last query sees every key; more queries than keys: the first see none
    ([7, 20], [300, 21], 4, 1, 64, True), ([50], [20], 2, 2, 64, True), ([70, 3], [17, 1], 3, 3, 32, True),
    ([9], [200], 2, 2, 40, False),
    # single tokens against long keys, split over several workgroups
    ([1, 1, 1], [1000, 3, 257], 8, 2, 128, True), ([1], [2049], 1, 1, 64, True), ([1] * 5, [700, 1, 64, 65, 300], 4, 4, 80, True),
    ([2], [1500], 16, 1, 32, True),
]


@pytest.mark.parametrize("case", range(len(ATTENTION)), ids=lambda i: str(ATTENTION[i]).replace(" ", ""))
def test_attention(hip, case):
    ql, kl, heads, kv, d, causal = ATTENTION[case]
    q, k, v, g = attention_inputs(np.random.default_rng(case), ql, kl, heads, kv, d)
    scale = d ** -0.5
    got = attend(hip, ql, kl, heads, kv, d, causal, q, k, v, scale, g, pad=case % 4)
    want = T.attention(q, k, v, ql, kl, heads, kv, scale, causal, g)
    bound = T.attention_bounds(q, k, v, ql, kl, heads, kv, scale, causal, g)
    empty = want[1] == -np.inf
    assert np.array_equal(got[1][empty], want[1][empty])
    got[1] = np.where(empty, 0, got[1])
    for a, w, b, what in zip(got, (want[0], np.where(empty, 0, want[1]), *want[2:]), bound, ("o", "lse", "dq", "dk", "dv")):
        close(a, w, b, what)


def test_attention_slices_of_one_projection_and_no_lse(hip):
    """q, k and v side by side in the rows of one projection, gradients into the rows of another; lse not asked for."""
    ql, heads, kv, d = [30, 45], 4, 2, 16
    q, k, v, g = attention_inputs(np.random.default_rng(1), ql, ql, heads, kv, d)
    want = attend(hip, ql, ql, heads, kv, d, True, q, k, v, 0.3, g)
    rows, width = up(hip, np.concatenate([q, k, v], 1)), (heads + 2 * kv) * d
    plan = hip.AttentionPlan(ql, heads=heads, kv_heads=kv, head_dim=d)
    at = [0, 4 * heads * d, 4 * (heads + kv) * d]
    o, lse, dg = hip.DeviceBuffer((75, heads * d)), hip.DeviceBuffer((75, heads)), up(hip, g)
    grads = up(hip, np.full((75, width), 7, np.float32))
    L, ptr = hip.lib(), [rows.ptr + a for a in at]
    call = lambda stats: hip.check(L.lmp_k_attention_f32(  # noqa: E731
        plan.handle, ptr[0], width, ptr[1], width, ptr[2], width, 0.3, o.ptr, heads * d, stats))
    call(None)
    assert np.array_equal(o.numpy(), want[0])
    call(lse.ptr)
    hip.check(L.lmp_k_attention_backward_f32(plan.handle, ptr[0], width, ptr[1], width, ptr[2], width, 0.3, o.ptr, heads * d,
                                             lse.ptr, dg.ptr, heads * d, grads.ptr, width, grads.ptr + at[1], width,
                                             grads.ptr + at[2], width))
    assert np.array_equal(grads.numpy(), np.concatenate(want[2:], 1))


@pytest.mark.parametrize("n,d,heads,kv", [(48, 32, 2, 1), (200, 64, 2, 2), (300, 128, 4, 1)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
def test_attention_masked_places_reach_nothing(hip, n, d, heads, kv, bad):
    """Infinities, NaN and huge values in keys and values that a row must not see, and in queries and output gradients of
    rows that a key must not see."""
    rng = np.random.default_rng(n)
    q, k, v, g = attention_inputs(rng, [n], [n], heads, kv, d)
    at, scale = n // 2 + 3, d ** -0.5
    clean = T.attention(q, k, v, [n], [n], heads, kv, scale, True, g)
    bound = T.attention_bounds(q, k, v, [n], [n], heads, kv, scale, True, g)
    k2, v2 = k.copy(), v.copy()
    k2[at, 1] = bad
    v2[at, :] = bad
    got = attend(hip, [n], [n], heads, kv, d, True, q, k2, v2, scale, g)
    for i, what in ((0, "o"), (1, "lse"), (2, "dq")):
        close(got[i][:at], clean[i][:at], bound[i][:at], what)
    q2, g2 = q.copy(), g.copy()
    q2[at, ::5] = bad
    g2[at, 1::3] = bad
    got = attend(hip, [n], [n], heads, kv, d, True, q2, k, v, scale, g2)
    keep = np.arange(n) != at
    for i, what in ((0, "o"), (1, "lse"), (2, "dq")):
        close(got[i][keep], clean[i][keep], bound[i][keep], what)
    for i, what in ((3, "dk"), (4, "dv")):
        close(got[i][at + 1:], clean[i][at + 1:], bound[i][at + 1:], what)


def test_attention_special_values_in_sight(hip):
    """An infinite value in sight gives that infinity (weights are positive), a NaN gives NaN, a key of -inf weight 0."""
    n, d = 40, 16
    q, k, v, _ = attention_inputs(np.random.default_rng(8), [n], [n], 1, 1, d)
    v[7, 3], v[9, 4] = np.inf, np.nan
    q[:, 0] = np.abs(q[:, 0])
    k[12, 0] = -np.inf
    got = attend(hip, [n], [n], 1, 1, d, True, q, k, v, 0.25)[0]
    want = T.attention(q, k, v, [n], [n], 1, 1, 0.25, True)[0]
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isposinf(got), np.isposinf(want))
    fine = np.isfinite(want)
    assert np.abs(got[fine] - want[fine]).max() < 1e-5


def launches(hip):
    n = C.c_uint64()
    hip.check(hip.lib().lmp_rt_kernel_launch_count(C.byref(n)))
    return n.value


def check_split(hip, ql, kl, heads, kv, d, causal, q, k, v, g, scale, pad=0, split=True):
    """Both passes against 64 bits; `split`: by the split-fp16 kernels, which launch nine or more where the fp32
    ones launch four at most."""
    before = launches(hip)
    got = attend(hip, ql, kl, heads, kv, d, causal, q, k, v, scale, g, pad=pad)
    assert (launches(hip) - before >= 9) == split
    want = T.attention(q, k, v, ql, kl, heads, kv, scale, causal, g)
    bound = T.attention_bounds(q, k, v, ql, kl, heads, kv, abs(scale), causal, g) if scale > 0 else \
        T.attention_bounds(-q, k, v, ql, kl, heads, kv, -scale, causal, g)
    empty = want[1] == -np.inf
    assert np.array_equal(got[1][empty], want[1][empty])
    got[1] = np.where(empty, 0, got[1])
    for a, w, b, what in zip(got, (want[0], np.where(empty, 0, want[1]), *want[2:]), bound, ("o", "lse", "dq", "dk", "dv")):
        close(a, w, b, what)
    return got


SPLIT = [
    ([700, 333], [700, 333], 16, 4, 64, True), ([513], [513], 32, 8, 128, True), ([1000], [1000], 16, 2, 80, True),
    ([600, 37, 0, 450], [600, 37, 5, 450], 12, 4, 96, True), ([640], [640], 16, 16, 33, False), ([777], [777], 16, 1, 100, True),
    # the last query sees every key; the first see none
    ([300, 1], [1200, 64], 16, 4, 128, True), ([900], [500], 16, 4, 64, True), ([257, 400], [90, 1100], 16, 8, 48, False),
    # few blocks: keys and steps in parts that are joined
    ([200], [3000], 8, 2, 128, True), ([1500], [1500], 2, 1, 128, True),
]


@pytest.mark.parametrize("case", range(len(SPLIT)), ids=lambda i: str(SPLIT[i]).replace(" ", ""))
def test_attention_of_long_batches(hip, case):
    ql, kl, heads, kv, d, causal = SPLIT[case]
    q, k, v, g = attention_inputs(np.random.default_rng(50 + case), ql, kl, heads, kv, d)
    check_split(hip, ql, kl, heads, kv, d, causal, q, k, v, g, d ** -0.5, pad=case % 3)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1.0, 1e-6])
def test_attention_of_long_batches_any_scale(hip, scale):
    q, k, v, g = attention_inputs(np.random.default_rng(3), [640], [640], 16, 4, 64)
    if scale == 0:  # every visible key weighs the same; the fp32 kernels run it
        got = attend(hip, [640], [640], 16, 4, 64, True, q, k, v, 0.0, g)
        mean = np.cumsum(v.astype(np.float64), 0) / np.arange(1, 641)[:, None]
        want = np.repeat(mean.reshape(640, 4, 64), 4, 1).reshape(640, -1)
        close(got[0], want, 700 * T.U32 * np.abs(v).max())
        assert not got[2].any() and not got[3].any()
        return
    check_split(hip, [640], [640], 16, 4, 64, True, q, k, v, g, scale)


@pytest.mark.parametrize("what", ["rows", "tiny", "huge", "columns", "zeros"])
def test_attention_of_long_batches_ranges(hip, what):
    """Operands of one power of two per tile: rows further apart than that carries, and largest values outside its range,
    go to the fp32 kernels; columns apart and rows of zeros stay."""
    n, heads, kv, d = 600, 16, 4, 64
    q, k, v, g = attention_inputs(np.random.default_rng(4), [n], [n], heads, kv, d)
    scale = d ** -0.5
    if what == "rows":
        for a in (q, k, v, g):
            a[::7] *= np.float32(2.0 ** -16)
            a[5] *= np.float32(8)
    elif what == "tiny":
        q *= np.float32(2.0 ** -70)
        g *= np.float32(2.0 ** -70)
        scale = float(2.0 ** 67)
    elif what == "huge":
        k *= np.float32(2.0 ** 45)
        scale = float(2.0 ** -48)
    elif what == "columns":
        for a in (q, k):
            a[:, 3::64] *= np.float32(64)
        scale /= 512
    else:
        for a in (q, k, v, g):
            a[64:128] = 0
            a[200] = 0
    check_split(hip, [n], [n], heads, kv, d, True, q, k, v, g, scale)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
def test_attention_of_long_batches_masked_places_reach_nothing(hip, bad):
    """As above, at sizes of the split kernels: sequences and key heads without such a value stay bit for bit as they were,
    those with one are as the fp32 kernels have them."""
    ql, heads, kv, d = [500, 400], 16, 4, 64
    q, k, v, g = attention_inputs(np.random.default_rng(12), ql, ql, heads, kv, d)
    clean = check_split(hip, ql, ql, heads, kv, d, True, q, k, v, g, 0.125)
    want = T.attention(q, k, v, ql, ql, heads, kv, 0.125, True, g)
    bound = T.attention_bounds(q, k, v, ql, ql, heads, kv, 0.125, True, g)
    at, width = 300, d * heads // kv  # in key head 1 of the first sequence
    k2, v2 = k.copy(), v.copy()
    k2[at, d + 3] = bad
    v2[at, d:2 * d] = bad
    got = attend(hip, ql, ql, heads, kv, d, True, q, k2, v2, 0.125, g)
    hit = np.zeros((900, heads * d), bool)
    hit[at:500, width:2 * width] = True
    for i in (0, 2):
        close(np.where(hit, 0, got[i]), np.where(hit, 0, want[i]), bound[i])
        other = np.ones_like(hit)
        other[:500, width:2 * width] = False
        assert np.array_equal(got[i][other], clean[i][other])
    q2, g2 = q.copy(), g.copy()
    q2[at, width:width + 5] = bad
    g2[at, width + 64:width + 70] = bad
    got = attend(hip, ql, ql, heads, kv, d, True, q2, k, v, 0.125, g2)
    for i in (3, 4):
        seen = np.zeros((900, kv * d), bool)
        seen[:at + 1, d:2 * d] = True
        close(np.where(seen, 0, got[i]), np.where(seen, 0, want[i]), bound[i])
        other = np.ones_like(seen)
        other[:500, d:2 * d] = False
        assert np.array_equal(got[i][other], clean[i][other])


def test_attention_of_long_batches_special_values_in_sight(hip):
    n, heads, kv, d = 600, 16, 4, 64
    q, k, v, g = attention_inputs(np.random.default_rng(8), [n], [n], heads, kv, d)
    v[200, 70], v[300, 5] = np.inf, np.nan
    k[250, 2 * d] = -np.inf
    q[:, 8 * d] = np.abs(q[:, 8 * d])
    got = attend(hip, [n], [n], heads, kv, d, True, q, k, v, 0.125, g)[0]
    want = T.attention(q, k, v, [n], [n], heads, kv, 0.125, True)[0]
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isposinf(got), np.isposinf(want))
    fine = np.isfinite(want)
    assert np.abs(got[fine] - want[fine]).max() < 1e-5


def test_attention_plans_are_refused_inside_a_capture(hip):
    hip.check(hip.lib().lmp_rt_graph_begin())
    try:
        with pytest.raises(hip.LmpError):
            hip.AttentionPlan([3], heads=1, head_dim=8)
    finally:
        hip.check(hip.lib().lmp_rt_graph_abort())


def test_recorded_step_replays(hip):
    """Norm, attention and AdamW recorded once: every replay equals the eager calls on the same state, and the step counts."""
    L, ql, heads, kv, d = hip.lib(), [40, 23], 4, 2, 32
    rng = np.random.default_rng(4)
    rows, width = 63, (heads + 2 * kv) * d
    x = up(hip, rng.standard_normal((rows, width)).astype(np.float32))
    plan = hip.AttentionPlan(ql, heads=heads, kv_heads=kv, head_dim=d)
    y, mean, rstd = hip.DeviceBuffer((rows, width)), hip.DeviceBuffer((rows,)), hip.DeviceBuffer((rows,))
    o, lse, grads = hip.DeviceBuffer((rows, heads * d)), hip.DeviceBuffer((rows, heads)), hip.DeviceBuffer((rows, width))
    dx, dw, db = hip.DeviceBuffer((rows, width)), hip.DeviceBuffer((width,)), hip.DeviceBuffer((width,))
    p = [rng.standard_normal(width).astype(np.float32) for _ in range(2)]

    def state():
        return ([[up(hip, a)] + [None] + [up(hip, np.zeros(width, np.float32)) for _ in range(2)] for a in p],
                up(hip, np.zeros(2, np.int64)))

    def step(tensors, count):
        at = [0, 4 * heads * d, 4 * (heads + kv) * d]
        hip.check(L.lmp_k_layer_norm(hip.FLOAT32, rows, width, x.ptr, width, tensors[0][0].ptr, tensors[1][0].ptr, 1e-5, y.ptr,
                                     width, mean.ptr, rstd.ptr))
        s = [y.ptr + a for a in at]
        hip.check(L.lmp_k_attention_f32(plan.handle, s[0], width, s[1], width, s[2], width, 0.2, o.ptr, heads * d, lse.ptr))
        hip.check(L.lmp_k_attention_backward_f32(plan.handle, s[0], width, s[1], width, s[2], width, 0.2, o.ptr, heads * d,
                                                 lse.ptr, o.ptr, heads * d, grads.ptr, width, grads.ptr + at[1], width,
                                                 grads.ptr + at[2], width))
        hip.check(L.lmp_k_layer_norm_backward(hip.FLOAT32, rows, width, grads.ptr, width, x.ptr, width, tensors[0][0].ptr,
                                              mean.ptr, rstd.ptr, dx.ptr, width, dw.ptr, db.ptr))
        adamw_call(hip, 32, [([t[0], gr, t[2], t[3]], width) for t, gr in zip(tensors, (dw, db))], [0.0, 0.0], count)

    (eager, n_eager), (kept, n_kept) = state(), state()
    graph = C.c_void_p()
    hip.check(L.lmp_rt_graph_begin())
    try:
        step(kept, n_kept)
    except BaseException:
        hip.check(L.lmp_rt_graph_abort())
        raise
    hip.check(L.lmp_rt_graph_end(C.byref(graph)))
    for i in range(4):
        step(eager, n_eager)
        want = [dx.numpy(), dw.numpy()] + [t[j].numpy() for t in eager for j in (0, 2, 3)]
        hip.check(L.lmp_rt_graph_launch(graph))
        got = [dx.numpy(), dw.numpy()] + [t[j].numpy() for t in kept for j in (0, 2, 3)]
        for a, b in zip(got, want):
            assert np.array_equal(a, b), i
        assert n_kept.numpy().tolist() == [i + 1, 0]
    hip.check(L.lmp_rt_graph_destroy(graph))


def test_attention_without_queries_or_keys(hip):
    """A million keys that no query sees, and queries without keys: zeros, whatever form the sizes ask for."""
    heads, kv, d = 2, 1, 64
    for ql, kl in (([0], [1 << 20]), ([5000], [0])):
        q, k, v, g = attention_inputs(np.random.default_rng(0), ql, kl, heads, kv, d)
        o, lse, dq, dk, dv = attend(hip, ql, kl, heads, kv, d, True, q, k, v, 0.1, g)
        assert (lse == -np.inf).all()
        for a in (o, dq, dk, dv):
            assert not a.any()


def test_recorded_long_attention_replays(hip):
    """The split kernels, their workspaces and joins recorded once; replays with new operands in the same buffers, eager work
    between them, one of them with a NaN that sends a key head to the fp32 kernels."""
    L, ql, heads, kv, d = hip.lib(), [700, 350], 16, 4, 64
    plan = hip.AttentionPlan(ql, heads=heads, kv_heads=kv, head_dim=d)
    sizes = [heads * d, kv * d, kv * d, heads * d]
    held = [hip.DeviceBuffer((1050, w)) for w in sizes]
    outs = [hip.DeviceBuffer((1050, w)) for w in (heads * d, heads, heads * d, kv * d, kv * d)]

    def step():
        q, k, v, g = (b.ptr for b in held)
        o, lse, dq, dk, dv = (b.ptr for b in outs)
        qw, kw = heads * d, kv * d
        hip.check(L.lmp_k_attention_f32(plan.handle, q, qw, k, kw, v, kw, 0.125, o, qw, lse))
        hip.check(L.lmp_k_attention_backward_f32(plan.handle, q, qw, k, kw, v, kw, 0.125, o, qw, lse, g, qw, dq, qw, dk, kw,
                                                 dv, kw))

    graph = C.c_void_p()
    hip.check(L.lmp_rt_graph_begin())
    try:
        step()
    except BaseException:
        hip.check(L.lmp_rt_graph_abort())
        raise
    hip.check(L.lmp_rt_graph_end(C.byref(graph)))
    for i in range(4):
        host = attention_inputs(np.random.default_rng(i), ql, ql, heads, kv, d)
        if i == 2:
            host[2][900, 70] = np.nan
        for b, a in zip(held, host):
            hip.check(L.lmp_rt_memcpy_h2d(b.ptr, a.ctypes.data, a.nbytes))
        step()
        want = [o.numpy() for o in outs]
        for o in outs:
            hip.check(L.lmp_k_fill(hip.FLOAT32, o.ptr, o.nbytes // 4, 7.0))
        hip.check(L.lmp_rt_graph_launch(graph))
        for o, w in zip(outs, want):
            assert np.array_equal(o.numpy(), w, equal_nan=True), i
    hip.check(L.lmp_rt_graph_destroy(graph))


def test_calls_repeat_bit_for_bit(hip):
    for ql, kl, heads, kv, d in (([1, 300, 40], [900, 300, 400], 4, 2, 64), ([1000, 300], [1000, 300], 16, 2, 64)):
        q, k, v, g = attention_inputs(np.random.default_rng(6), ql, kl, heads, kv, d)
        first = attend(hip, ql, kl, heads, kv, d, True, q, k, v, 0.125, g)
        for _ in range(3):
            for a, b in zip(attend(hip, ql, kl, heads, kv, d, True, q, k, v, 0.125, g), first):
                assert np.array_equal(a, b)


def one_power_a_tile(a, lengths, d):
    """Whether every tile of 32 rows of one head is one the split-fp16 kernels keep (include/lmp_hip_transformer.h)."""
    first = 0
    for n in lengths:
        for at in range(first, first + n, 32):
            rows = np.abs(a[at:min(at + 32, first + n)].reshape(-1, a.shape[1] // d, d)).max(2)
            top = rows.max(0)
            least = np.where(rows > 0, rows, np.inf).min(0)
            if not ((top == 0) | ((top >= 2.0 ** -60) & (top < 2.0 ** 41) & (least * 2 ** 11 >= top))).all():
                return False
        first += n
    return True


def attend_split(hip, n, heads, kv, d, q, k, v, scale):
    """The forward pass of one causal sequence, by the split kernels alone."""
    assert all(one_power_a_tile(a, [n], d) for a in (q, k, v))
    before = launches(hip)
    got = attend(hip, [n], [n], heads, kv, d, True, q, k, v, scale)
    assert launches(hip) - before >= 4  # the fp32 kernels launch two at most
    return got


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [8, 11, 15])
def test_attention_of_long_batches_scores_past_24_bits(hip, power, sign):
    """Scores of up to 2^25, 2^31 and 2^39, formed without an error and further apart than float32's steps at their size:
    each row is its best key's value.

    Rounding: the value's two parts hold it to 2 u, their sum rounds once, and 2^-39 of the tile's largest is lost where
    a value is small; the weight is exactly 1.  lse: the constant log2 e, the product with it and the product with ln 2."""
    n, heads, kv, d, scale = 1000, 16, 4, 64, 0.125
    rng = np.random.default_rng(power)
    q, k, v, _ = attention_inputs(rng, [n], [n], heads, kv, d)
    q[:], k[:] = 0, 0
    order = rng.permutation(n) - n / 2 + 0.5
    q[:, ::d] = (sign * 2.0 ** power * (1 + np.arange(n) % 7))[:, None]
    k[:, ::d] = (2.0 ** power * order)[:, None]
    o, lse = attend_split(hip, n, heads, kv, d, q, k, v, scale)
    best = np.array([(sign * order[:i + 1]).argmax() for i in range(n)])
    want = np.repeat(v[best].reshape(n, kv, d), heads // kv, 1).reshape(n, -1).astype(np.float64)
    close(o, want, 4 * T.U32 * np.abs(want) + 2.0 ** -39 * np.abs(v).max(), "o")
    top = (q[:, 0].astype(np.float64) * k[best, 0] * scale)[:, None].repeat(heads, 1)
    close(lse, top, 4 * T.U32 * np.abs(top), "lse")


@pytest.mark.parametrize("size", [2e3, 1e4])
def test_attention_of_long_batches_large_random_scores(hip, size):
    """Scores of some 10^7 and 10^9: a row whose best key leads by more than the scores' rounding and 60 is that key's value,
    every other one lies among the values that it sees."""
    n, heads, kv, d, scale = 1000, 16, 4, 64, 0.125
    q, k, v, _ = attention_inputs(np.random.default_rng(11), [n], [n], heads, kv, d)
    q, k = (q * np.float32(size)), (k * np.float32(size))
    o, lse = attend_split(hip, n, heads, kv, d, q, k, v, scale)
    assert np.isfinite(o).all() and np.isfinite(lse).all()
    alone = 0
    for h in range(heads):
        qs, ks, vs = (a.reshape(n, -1, d)[:, i].astype(np.float64) for a, i in ((q, h), (k, h // 4), (v, h // 4)))
        s = np.where(np.tri(n, dtype=bool), qs @ ks.T * scale, -np.inf)
        # of a score: d sums and 16 roundings as in attention_bounds, and those of its product with the constant
        err = (d + 20) * T.U32 * scale * (np.abs(qs) @ np.abs(ks).T).max(1)
        ranks = np.sort(s, 1)
        lead = ranks[:, -1] - ranks[:, -2] > 2 * err + 60
        alone += int(lead.sum())
        got, want = o.reshape(n, heads, d)[:, h], vs[s.argmax(1)]
        close(got[lead], want[lead], 4 * T.U32 * np.abs(want[lead]) + 2.0 ** -39 * np.abs(v).max(), "o")
        slack = 64 * T.U32 * np.abs(v).max()
        low, high = np.minimum.accumulate(vs, 0), np.maximum.accumulate(vs, 0)
        assert (got >= low - slack).all() and (got <= high + slack).all()
    assert alone > n * heads // 2


@pytest.mark.parametrize("at", [0, 288])
@pytest.mark.parametrize("weight", ["negligible", "even"])
@pytest.mark.parametrize("power", [28, 40, 64])
def test_attention_of_long_batches_values_of_different_sizes(hip, power, weight, at):
    """A tile of 32 keys whose values are 2^power as large as the others', with weights that make up for it or go 2^16
    below: the other keys' weights keep their digits."""
    n, heads, kv, d, scale = 1000, 16, 4, 64, 0.125
    q, k, v, g = attention_inputs(np.random.default_rng(power + at), [n], [n], heads, kv, d)
    v *= np.float32(2.0 ** -30)
    v[at:at + 32] *= np.float32(2.0 ** power)
    q[:, ::d] = 8
    k[at:at + 32, ::d] = np.float32(-np.log(2) * (power + (16 if weight == "negligible" else 0)))
    attend_split(hip, n, heads, kv, d, q, k, v, scale)
    check_split(hip, [n], [n], heads, kv, d, True, q, k, v, g, scale)


def test_attention_of_long_batches_weights_that_rise_by_less_than_a_bit(hip):
    """Every tile of keys weighs 2^0.95 as much as the one before it, and the first one's values are 2^44 as large: the power
    of two that the weights take falls with its weight, by parts of a bit at a time.  Heads enough that no row's keys are
    split into parts."""
    n, heads, kv, d, scale = 1600, 64, 16, 32, 0.125
    q, k, v, _ = attention_inputs(np.random.default_rng(5), [n], [n], heads, kv, d)
    q, k, v = q / 32, k / 32, v / 1024
    v[:32] *= np.float32(2.0 ** 44)
    q[:, ::d] = 8
    k[:, ::d] = (np.log(2) * 0.95 * (1 + np.arange(n) // 32)).astype(np.float32)[:, None]
    o, lse = attend_split(hip, n, heads, kv, d, q, k, v, scale)
    for h in (0, heads - 1):
        own, keys = slice(h * d, h * d + d), slice(h // 4 * d, h // 4 * d + d)
        one = (q[:, own], k[:, keys], v[:, keys], [n], [n], 1, 1, scale, True)
        for a, w, b, what in zip((o[:, own], lse[:, h:h + 1]), T.attention(*one), T.attention_bounds(*one), ("o", "lse")):
            close(a, w, b, what)


def test_adamw_8_keeps_small_second_moments_above_zero(hip):
    """A second moment far below its block's largest is kept as the least code, also where its share of that underflows
    float32: 2^-110 beside 2^70."""
    n = 256
    g = np.full(n, 2.0 ** -50, np.float32)
    g[9], g[40:50] = 2.0 ** 40, 0
    zero = np.zeros(1, np.float32)
    t = [up(hip, np.zeros(n, np.float32)), up(hip, g), Bytes(hip, np.zeros(n, np.int8)), Bytes(hip, np.zeros(n, np.uint8)),
         up(hip, zero), up(hip, zero)]
    adamw_call(hip, 8, [(t, n)], [0.0], up(hip, np.zeros(2, np.int64)))
    want = np.where(g == 0, 0, np.where(g > 1, 255, 1))
    assert np.array_equal(t[3].numpy(), want)


@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-20])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_tiny_gradients_without_eps(hip, bits, eps):
    """The first step is lr g / (|g| + eps) whatever g's size: second moments of 1e-39, below float32's smallest normal.

    v rounds to a multiple of 2^-149, off by 7e-7 of 1e-39 at most; its root by half of that.  Ten roundings of the step
    besides, and two of p."""
    n, lr = 700, 0.01
    g = (1e-18 * (1 + np.arange(n) / n) * np.where(np.arange(n) % 3, 1, -1)).astype(np.float32)
    t = [up(hip, np.ones(n, np.float32)), up(hip, g)]
    if bits == 32:
        t += [up(hip, np.zeros(n, np.float32)) for _ in range(2)]
    else:
        t += [Bytes(hip, np.zeros(n, np.int8)), Bytes(hip, np.zeros(n, np.uint8))]
        t += [up(hip, np.zeros(3, np.float32)) for _ in range(2)]
    adamw_call(hip, bits, [(t, n)], [0.0], up(hip, np.zeros(2, np.int64)), hyper={**HYPER, "lr": lr, "eps": eps})
    want = 1 - lr * g.astype(np.float64) / (np.abs(g.astype(np.float64)) + eps)
    close(t[0].numpy(), want, lr * (3.5e-7 + 10 * T.U32) + 2 * T.U32, "p")


@pytest.mark.parametrize("n", [(1 << 21) + 5, (1 << 25) + 300])
def test_adamw_8_of_tiny_gradients_in_long_tensors(hip, n):
    """As above, with states of 8 bits and eps 0, past the sizes at which a lane takes four units and accesses stream."""
    lr = 0.01
    g = np.resize((1e-18 * np.where(np.arange(256) % 3, 1, -1)).astype(np.float32), n)
    t = [up(hip, np.ones(n, np.float32)), up(hip, g), Bytes(hip, np.zeros(n, np.int8)), Bytes(hip, np.zeros(n, np.uint8))]
    t += [up(hip, np.zeros(-(-n // 256), np.float32)) for _ in range(2)]
    adamw_call(hip, 8, [(t, n)], [0.0], up(hip, np.zeros(2, np.int64)), hyper={**HYPER, "lr": lr, "eps": 0.0})
    close(t[0].numpy(), 1 - lr * np.sign(g.astype(np.float64)), lr * (7e-7 + 10 * T.U32) + 2 * T.U32, "p")
