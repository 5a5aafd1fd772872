"""Rotary positions, dropout, gated linear layers and the vocabulary loss through the C ABI, against plain 64-bit forms
(tests/_decoder.py).  Tolerances count roundings (the bounds there); what dropout keeps has to be equal."""
import numpy as np
import pytest

import _decoder as D

pytestmark = pytest.mark.gpu


def up(hip, a):
    return hip.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


def padded(a, ld, fill=np.nan):
    """The rows of `a` in rows of ld values; what lies between them must not be read into results or written."""
    out = np.full((a.shape[0], ld), fill, a.dtype)
    out[:, :a.shape[1]] = a
    return out


def close(got, want, bound, what=""):
    err = np.abs(np.asarray(got, np.promote_types(got.dtype, np.float64)) - want)
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(err[bad].max()), float(np.broadcast_to(bound, err.shape)[bad].min()))


# ------------------------------------------------------------------ rotary

ROTARY = [  # rows, heads, dim, turned, columns after the heads
    (1, 1, 2, 2, 0), (1, 1, 128, 128, 0), (5, 3, 8, 6, 0), (7, 1, 9, 2, 3), (33, 4, 80, 20, 7), (32, 40, 128, 128, 1024),
    (3, 2, 5, 0, 4), (4, 0, 8, 8, 6), (17, 5, 30, 30, 1), (2, 3, 1000, 600, 0), (130, 48, 64, 32, 64), (1000, 2, 96, 96, 5),
    (3, 17, 256, 256, 0), (5001, 1, 16, 16, 0)]


def rotary(hip, x, positions, f, heads, dim, turned, interleaved, scale, inverse=0, shift=0, pad=0, in_place=False):
    rows, cols = x.shape
    ld = cols + pad
    flat = np.full(rows * ld + shift, np.nan, x.dtype)
    flat[shift:].reshape(rows, ld)[:, :cols] = x
    dx, dp, df = up(hip, flat), up(hip, positions.astype(np.int64)), up(hip, np.asarray(f, np.float64))
    y = dx if in_place else up(hip, np.full(rows * ld + shift, 7, x.dtype))
    at = shift * x.itemsize
    hip.check(hip.lib().lmp_k_rotary(hip.CODE_OF[x.dtype], rows, cols, heads, dim, turned, interleaved, dx.ptr + at, ld, dp.ptr,
                                     df.ptr, scale, inverse, y.ptr + at, ld))
    out = y.numpy()
    rest = out[shift:].reshape(rows, ld)[:, cols:]
    assert np.isnan(rest).all() if in_place else (rest == 7).all()
    return out[shift:].reshape(rows, ld)[:, :cols]


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("rows,heads,dim,turned,plain", ROTARY)
def test_rotary(hip, rows, heads, dim, turned, plain, interleaved, dtype):
    rng = np.random.default_rng(rows + 7 * dim)
    x = rng.standard_normal((rows, heads * dim + plain)).astype(dtype)
    positions = rng.integers(-5, 200000, rows)
    positions[0] = 0
    f = 10000.0 ** (-np.arange(turned // 2) / max(1, turned // 2))
    for scale, inverse, shift, pad in ((1.0, 0, 0, 0), (1.3, 1, 1, 3)):
        args = heads, dim, turned, bool(interleaved), positions, f, scale
        want = D.rotary(x, *args, inverse=bool(inverse))
        bound = D.rotary_bound(x, *args, unit=D.U32 if dtype == np.float32 else 2.0 ** -53)
        got = rotary(hip, x, positions, f, heads, dim, turned, interleaved, scale, inverse, shift, pad)
        close(got, want, bound)
        again = rotary(hip, x, positions, f, heads, dim, turned, interleaved, scale, inverse, shift, pad, in_place=True)
        assert np.array_equal(again, got)


def test_rotary_far_positions_and_special_values(hip):
    """Angles of far positions keep their digits; a value that is not finite stays in its pair."""
    f = np.array([1.0, 0.37, 1e-3, 1e-5])
    positions = np.array([1 << 20, 3_000_000_019, -(1 << 40), 7])
    x = np.random.default_rng(0).standard_normal((4, 16)).astype(np.float32)
    args = 2, 8, 8, False, positions, f, 1.0
    close(rotary(hip, x, positions, f, 2, 8, 8, 0, 1.0), D.rotary(x, *args), D.rotary_bound(x, *args))
    x[3, 1], x[3, 10] = np.inf, np.nan
    got = rotary(hip, x, positions, f, 2, 8, 8, 0, 1.0)
    assert [i for i in range(16) if not np.isfinite(got[3, i])] == [1, 5, 10, 14] and np.isfinite(got[:3]).all()


def test_rotary_beside_itself(hip):
    """Queries of one half of wider rows turned into the other half."""
    x = np.random.default_rng(1).standard_normal((6, 24)).astype(np.float32)
    positions, f = np.arange(6), np.array([1.0, 0.1])
    both = up(hip, x)
    p, df = up(hip, positions.astype(np.int64)), up(hip, f)
    hip.check(hip.lib().lmp_k_rotary(hip.FLOAT32, 6, 12, 3, 4, 4, 0, both.ptr, 24, p.ptr, df.ptr, 1.0, 0, both.ptr + 48, 24))
    out = both.numpy()
    assert np.array_equal(out[:, :12], x[:, :12])
    assert np.array_equal(out[:, 12:], rotary(hip, x[:, :12].copy(), positions, f, 3, 4, 4, 0, 1.0))


# ----------------------------------------------------------------- dropout

def dropout(hip, x, rate, seed, state, residual=None, used=None, over=None):
    dx, dr = up(hip, x), None if residual is None else up(hip, residual)
    y = dict(x=dx, residual=dr).get(over) or up(hip, np.full(x.shape, 7, x.dtype))
    hip.check(hip.lib().lmp_k_dropout(hip.CODE_OF[x.dtype], x.size, dx.ptr, dr and dr.ptr, rate, seed, state.ptr,
                                      used and used.ptr, y.ptr))
    return y.numpy()


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 255, 1024, 4095, 4097, 70001, 20_000_003])
def test_dropout(hip, n, dtype):
    rng = np.random.default_rng(n)
    # Roundings of a kept value: in float32 the factor's and the product's; in float64 1 - rate rounds too.  (The plain form
    # in long double: in 64 bits its own roundings would be as large as what is tested.)
    units = 2.01 * D.U32 if dtype == np.float32 else 3.01 * 2.0 ** -53
    wide, last = (lambda a: a.astype(np.longdouble)), D.U32 if dtype == np.float32 else 2.0 ** -53  # noqa: E731
    x, r, g = (rng.standard_normal(n).astype(dtype) for _ in range(3))
    state, used = up(hip, np.array([5, 0])), up(hip, np.array([-1]))
    seed, rate = 0xFEDCBA9876543210, 0.3
    for call, res in ((5, None), (6, r), (7, None)):
        y = dropout(hip, x, rate, seed, state, res, used)
        assert state.numpy().tolist() == [call + 1, 0] and used.numpy().tolist() == [call]
        keep = D.kept(n, rate, seed, call)
        base = np.zeros(n, np.longdouble) if res is None else wide(res)
        share = 1 - np.longdouble(rate)
        want = base + np.where(keep, wide(x) / share, 0)
        close(wide(y), want, units * np.abs(x) / (1 - rate) + last * np.abs(want))
        assert np.array_equal(y[~keep], base[~keep].astype(dtype))
        dg, dx = up(hip, g), up(hip, np.full(n, 7, dtype))
        for out in (dx, dg):
            hip.check(hip.lib().lmp_k_dropout_backward(hip.CODE_OF[np.dtype(dtype)], n, dg.ptr, rate, seed, used.ptr, out.ptr))
            d = out.numpy()
            assert (d[~keep] == 0).all()
            close(wide(d[keep]), wide(g[keep]) / share, units * np.abs(g[keep]) / (1 - rate))
    for over in ("x", "residual"):
        a, b = (up(hip, np.array([9, 0])) for _ in range(2))
        assert np.array_equal(dropout(hip, x, rate, seed, a, r), dropout(hip, x, rate, seed, b, r, over=over))


def test_dropout_rates_and_what_is_dropped(hip):
    x = np.full(40000, np.inf, np.float32)
    x[::3] = np.nan
    state = up(hip, np.array([0, 0]))
    assert np.array_equal(dropout(hip, x, 0.0, 1, state), x, equal_nan=True)
    assert (dropout(hip, x, 1.0, 1, state, used=up(hip, np.zeros(1, np.int64))) == 0).all()
    y = dropout(hip, x, 0.5, 1, state)
    keep = D.kept(40000, 0.5, 1, 2)
    assert (y[~keep] == 0).all() and not np.isfinite(y[keep]).any()
    # a call of nothing counts as one; calls past 2^32 have numbers of their own
    hip.check(hip.lib().lmp_k_dropout(hip.FLOAT32, 0, None, None, 0.5, 1, state.ptr, None, None))
    assert state.numpy().tolist() == [4, 0]
    ones, far = np.ones(5000, np.float32), (1 << 32) + 3
    a, b = dropout(hip, ones, 0.5, 1, up(hip, np.array([3, 0]))), dropout(hip, ones, 0.5, 1, up(hip, np.array([far, 0])))
    assert np.array_equal(a > 0, D.kept(5000, 0.5, 1, 3)) and np.array_equal(b > 0, D.kept(5000, 0.5, 1, far))
    assert 0.4 < (a > 0).mean() < 0.6 and (a != b).any()


# ------------------------------------------------------------ gated linear

GATED = [(1, 1, 1), (1, 7, 3), (3, 5, 4), (2, 64, 33), (32, 64, 64), (5, 300, 70), (33, 40, 129), (31, 1000, 96), (32, 1024, 515),
         (64, 32, 200), (70, 129, 65), (129, 128, 128), (300, 77, 260), (200, 512, 300), (1000, 64, 31), (513, 256, 640),
         (700, 400, 600), (1031, 257, 521), (32, 2048, 2100), (4000, 33, 1037), (6007, 300, 97), (130, 4097, 300),
         # products split into fp16 parts: forward, and both ways
         (9001, 33, 1037), (2100, 1031, 1100), (1031, 2050, 1001), (600, 2048, 2100), (5003, 600, 1201)]


def gated(hip, gate, x, w, b, g, pads=(0, 0, 0, 0), want=(True, True, True), keep=True):
    """h, dx, dw and db; rows of x, w, h and pre `pads` values apart."""
    rows, k = x.shape
    width = w.shape[1]
    n = width // 2
    px, pw, ph, pp = pads
    dx_, dw_, dg = up(hip, padded(x, k + px)), up(hip, padded(w, width + pw)), up(hip, padded(g, n + ph))
    db_ = None if b is None else up(hip, b)
    h = up(hip, np.full((rows, n + ph), 7, np.float32))
    pre = up(hip, np.full((rows, width + pp), 7, np.float32)) if keep else None
    code = hip.GATE[gate]
    hip.check(hip.lib().lmp_k_gated_linear_f32(code, rows, k, n, dx_.ptr, k + px, dw_.ptr, width + pw, db_ and db_.ptr, h.ptr,
                                               n + ph, pre and pre.ptr, width + pp))
    out = h.numpy()
    assert (out[:, n:] == 7).all()
    if not keep:
        return out[:, :n]
    assert (pre.numpy()[:, width:] == 7).all()
    outs = [up(hip, np.full(s, 7, np.float32)) for s in ((rows, k + px), (k, width + pw), (width,))]
    ptr = [o.ptr if t else None for o, t in zip(outs, want)]
    hip.check(hip.lib().lmp_k_gated_linear_backward_f32(code, rows, k, n, dg.ptr, n + ph, dx_.ptr, k + px, dw_.ptr, width + pw,
                                                        pre.ptr, width + pp, ptr[0], k + px, ptr[1], width + pw, ptr[2]))
    got = [o.numpy() for o in outs]
    assert (got[0][:, k:] == 7).all() and (got[1][:, width:] == 7).all()
    for o, t in zip(got, want):
        assert t or (o == 7).all()
    return out[:, :n], got[0][:, :k], got[1][:, :width], got[2]


@pytest.mark.parametrize("rows,k,n", GATED)
@pytest.mark.parametrize("gate", ["silu", "gelu", "gelu_tanh", "sigmoid"])
def test_gated_linear(hip, gate, rows, k, n):
    rng = np.random.default_rng(rows * 1009 + k * 31 + n)
    x, w = rng.standard_normal((rows, k)).astype(np.float32), (rng.standard_normal((k, 2 * n)) * k ** -0.5).astype(np.float32)
    b, g = rng.standard_normal(2 * n).astype(np.float32), rng.standard_normal((rows, n)).astype(np.float32)
    for bias, pads in ((b, (0, 0, 0, 0)), (None, (1, 3, 2, 5))):
        want, bound = D.gated(gate, x, w, bias, g), D.gated_bounds(gate, x, w, bias, g)
        got = gated(hip, gate, x, w, bias, g, pads)
        for a, v, e, what in zip(got, want, bound, ("h", "dx", "dw", "db")):
            close(a, v, e, (what, bias is None))
        assert np.array_equal(gated(hip, gate, x, w, bias, g, pads, keep=False), got[0])


def test_gated_linear_in_the_largest_tiles(hip):
    test_gated_linear(hip, "silu", 8200, 1024, 2080)


def test_gated_linear_relu_is_exact_on_integers(hip):
    """Small whole numbers: every product and sum is exact, so ReLU's two sides are too, at 0 as well."""
    rng = np.random.default_rng(4)
    for rows, k, n in ((3, 5, 4), (40, 33, 70), (300, 64, 129), (301, 700, 701), (1500, 1100, 1201)):
        x, w, g = (rng.integers(-3, 4, s).astype(np.float32) for s in ((rows, k), (k, 2 * n), (rows, n)))
        for got, want in zip(gated(hip, "relu", x, w, None, g), D.gated("relu", x, w, None, g)):
            assert np.array_equal(got, want)


def test_gated_linear_parts_of_the_backward(hip):
    rng = np.random.default_rng(6)
    for rows, k, n in ((5, 9, 6), (200, 70, 140), (300, 700, 701), (1500, 1100, 1201)):
        x, w, g = (rng.standard_normal(s).astype(np.float32) for s in ((rows, k), (k, 2 * n), (rows, n)))
        want, bound = D.gated("silu", x, w, None, g), D.gated_bounds("silu", x, w, None, g)
        for parts in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)):
            got = gated(hip, "silu", x, w, None, g, want=[bool(p) for p in parts])
            for i, p in enumerate(parts):
                if p:
                    close(got[1 + i], want[1 + i], bound[1 + i], parts)


def test_gated_linear_of_no_rows_clears_the_gradients(hip):
    dw, db, spare = (up(hip, np.full(s, 7, np.float32)) for s in ((5, 9), (8,), (4, 8)))
    hip.check(hip.lib().lmp_k_gated_linear_backward_f32(0, 0, 5, 4, None, 4, None, 5, None, 8, None, 8, spare.ptr, 5, dw.ptr, 9,
                                                        db.ptr))
    assert (dw.numpy()[:, :8] == 0).all() and (dw.numpy()[:, 8] == 7).all() and (db.numpy() == 0).all()
    assert (spare.numpy() == 7).all()


def test_gated_linear_special_values(hip):
    """Infinities and NaN in one row touch no other; gates far out are 0, a or 1; operands far apart and past the split's
    range come out as float32's products give them."""
    rng = np.random.default_rng(8)
    for rows, k, n in ((6, 40, 30), (150, 64, 130), (300, 700, 701), (1500, 1100, 1201)):
        x, w, g = (rng.standard_normal(s).astype(np.float32) for s in ((rows, k), (k, 2 * n), (rows, n)))
        clean = gated(hip, "silu", x, w, None, g)
        x[2, 3], x[4, 0] = np.nan, np.inf
        got = gated(hip, "silu", x, w, None, g)
        others = [r for r in range(rows) if r not in (2, 4)]
        assert np.isnan(got[0][2]).all() and not np.isfinite(got[0][4]).any()
        bound = D.gated_bounds("silu", x[others], w, None, g[others])[0]
        close(got[0][others], clean[0][others].astype(np.float64), 2 * bound)
    for gate in D.GATES:
        if gate == "relu":
            continue
        x = np.array([[-300.0], [300.0], [-1e30], [1e30], [0.0]], np.float32)
        w, g = np.array([[1.0, 1e-30]], np.float32), np.ones((5, 1), np.float32)
        h = gated(hip, gate, x, w, None, g, keep=False)[:, 0]
        u = (x * np.float32(1e-30))[:, 0]
        act = np.array([0, 1, 0, 1, 0.5]) if gate == "sigmoid" else np.maximum(x[:, 0].astype(np.float64), 0)
        close(h, act * u, 1e-5 * np.abs(act * u) + 1e-38, gate)
    # one row and one column far larger than the others, and far smaller
    for rows, k, n, scale in [(*size, scale) for size in ((70, 96, 70), (400, 600, 700), (1500, 1100, 1201)) for scale in (1e-20, 1e-12, 1e12)]:
        x, w, g = (rng.standard_normal(s).astype(np.float32) for s in ((rows, k), (k, 2 * n), (rows, n)))
        if k > 96:
            w *= np.float32(k ** -0.5)
        xs, gs = x.copy(), g.copy()
        xs[5] *= np.float32(scale)
        gs[9] *= np.float32(scale)
        want, bound = D.gated("sigmoid", xs, w, None, gs), D.gated_bounds("sigmoid", xs, w, None, gs)
        for a, v, e, what in zip(gated(hip, "sigmoid", xs, w, None, gs), want, bound, ("h", "dx", "dw", "db")):
            close(a, v, e + 1e-37, (what, scale))


# ----------------------------------------------------------- cross entropy

LOSS = [(1, 1, 1), (1, 3, 2), (3, 5, 7), (32, 64, 10), (7, 33, 1000), (64, 16, 129), (40, 130, 515), (130, 64, 1024),
        (33, 100, 4099), (300, 40, 333), (65, 7, 20001), (129, 256, 640),
        (1031, 257, 1021), (40, 1000, 7001), (3000, 33, 2801), (32, 600, 14100), (9000, 520, 64), (777, 1111, 513),
        # products split into fp16 parts
        (2300, 520, 10007), (9001, 97, 2801), (4099, 1031, 2001), (300, 1024, 30011), (5003, 600, 1009)]


def loss(hip, x, w, b, targets, weights=None, pads=(0, 0), grads=True, want=(True, True, True)):
    rows, k = x.shape
    vocab = w.shape[1]
    px, pw = pads
    dx_, dw_, dt = up(hip, padded(x, k + px)), up(hip, padded(w, vocab + pw)), up(hip, targets.astype(np.int64))
    db_, dwt = None if b is None else up(hip, b), None if weights is None else up(hip, weights)
    out = up(hip, np.full(rows, 7, np.float32))
    if not grads:
        hip.check(hip.lib().lmp_k_linear_cross_entropy_f32(rows, k, vocab, dx_.ptr, k + px, dw_.ptr, vocab + pw, db_ and db_.ptr,
                                                           dt.ptr, out.ptr))
        return out.numpy()
    outs = [up(hip, np.full(s, 7, np.float32)) for s in ((rows, k + px), (k, vocab + pw), (vocab,))]
    ptr = [o.ptr if t else None for o, t in zip(outs, want)]
    hip.check(hip.lib().lmp_k_linear_cross_entropy_grad_f32(
        rows, k, vocab, dx_.ptr, k + px, dw_.ptr, vocab + pw, db_ and db_.ptr, dt.ptr, dwt and dwt.ptr, out.ptr, ptr[0], k + px,
        ptr[1], vocab + pw, ptr[2]))
    got = [o.numpy() for o in outs]
    assert (got[0][:, k:] == 7).all() and (got[1][:, vocab:] == 7).all()
    for o, t in zip(got, want):
        assert t or (o == 7).all()
    return out.numpy(), got[0][:, :k], got[1][:, :vocab], got[2]


def check_loss(hip, x, w, b, targets, weights=None, pads=(0, 0)):
    want, bound = D.cross_entropy(x, w, b, targets, weights), D.cross_entropy_bounds(x, w, b, targets, weights)
    got = loss(hip, x, w, b, targets, weights, pads)
    for a, v, e, what in zip(got, want, bound, ("loss", "dx", "dw", "db")):
        close(a, v, e, what)
    close(loss(hip, x, w, b, targets, pads=pads, grads=False), want[0], bound[0], "loss alone")
    return got


@pytest.mark.parametrize("rows,k,vocab", LOSS)
def test_cross_entropy(hip, rows, k, vocab):
    rng = np.random.default_rng(rows * 1009 + k * 31 + vocab)
    x, w = rng.standard_normal((rows, k)).astype(np.float32), (2 * rng.standard_normal((k, vocab)) * k ** -0.5).astype(np.float32)
    b, weights = rng.standard_normal(vocab).astype(np.float32), rng.random(rows).astype(np.float32)
    targets = rng.integers(0, vocab, rows)
    check_loss(hip, x, w, b, targets, weights)
    targets[::3] = -1 - targets[::3]
    check_loss(hip, x, w, None, targets, None, (3, 1))


def test_cross_entropy_of_large_vocabularies(hip):
    rng = np.random.default_rng(1)
    for rows, k, vocab in ((2300, 12, 30011), (2300, 40, 30011), (1050, 64, 33000)):
        x, w = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((k, vocab)).astype(np.float32)
        targets = rng.integers(-vocab // 4, vocab, rows)
        check_loss(hip, x, w, rng.standard_normal(vocab).astype(np.float32), targets, rng.random(rows).astype(np.float32))


@pytest.mark.parametrize("k", [12, 64])  # as they are, and split into fp16 parts
def test_cross_entropy_in_several_pieces(hip, k):
    """More logits than one piece of the workspace holds.  The plain form by parts of the rows; a sum over all of them rounds
    as often as three such parts' bounds allow."""
    rng = np.random.default_rng(7)
    rows, vocab = 4500, 30011
    x, w = rng.standard_normal((rows, k)).astype(np.float32), (rng.standard_normal((k, vocab)) * k ** -0.5).astype(np.float32)
    b, weights, targets = rng.standard_normal(vocab).astype(np.float32), rng.random(rows).astype(np.float32), \
        rng.integers(-vocab // 4, vocab, rows)
    got = loss(hip, x, w, b, targets, weights)
    dw, db, ew, eb = 0, 0, 0, 0
    for at in range(0, rows, 1500):
        part = slice(at, at + 1500)
        args = x[part], w, b, targets[part], weights[part]
        want, bound = D.cross_entropy(*args), D.cross_entropy_bounds(*args)
        close(got[0][part], want[0], bound[0], "loss")
        close(got[1][part], want[1], bound[1], "dx")
        dw, db, ew, eb = dw + want[2], db + want[3], ew + 3 * bound[2], eb + 3 * bound[3]
    close(got[2], dw, ew, "dw")
    close(got[3], db, eb, "db")


def test_cross_entropy_rows_that_do_not_count_leave_no_trace(hip):
    rng = np.random.default_rng(2)
    for rows, k, vocab in ((9, 20, 50), (140, 64, 700), (700, 500, 1009), (2100, 900, 2003)):
        x, w = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((k, vocab)).astype(np.float32)
        targets, weights = rng.integers(0, vocab, rows), rng.random(rows).astype(np.float32)
        targets[[1, 4]] = -1, -(1 << 40)
        x[1], weights[1] = np.nan, np.nan
        x[4, ::2], x[4, 1::2], weights[4] = np.inf, -np.inf, np.inf
        got = check_loss(hip, x, w, None, targets, weights)
        assert (got[0][[1, 4]] == 0).all() and (got[1][[1, 4]] == 0).all()
        # no row counts
        got = loss(hip, x, w, None, np.full(rows, -1), weights)
        assert all((a == 0).all() for a in got)


def test_cross_entropy_targets_past_the_vocabulary(hip):
    rng = np.random.default_rng(3)
    for rows, k, vocab in ((6, 8, 33), (40, 130, 515), (700, 500, 1009), (2100, 900, 2003)):
        x, w = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((k, vocab)).astype(np.float32)
        targets = rng.integers(0, vocab, rows)
        targets[[1, 3, 4]] = vocab, 1 << 40, vocab - 1
        value, dx, dw, _ = loss(hip, x, w, None, targets)
        assert np.isnan(value[[1, 3]]).all() and np.isnan(dx[[1, 3]]).all() and np.isnan(dw).all()
        good = [r for r in range(rows) if r not in (1, 3)]
        want, bound = D.cross_entropy(x[good], w, None, targets[good]), D.cross_entropy_bounds(x[good], w, None, targets[good])
        close(value[good], want[0], bound[0])
        close(dx[good], want[1], bound[1])
        assert np.array_equal(np.isnan(loss(hip, x, w, None, targets, grads=False)), np.isnan(value))


def test_cross_entropy_of_barred_and_extreme_logits(hip):
    """A bias of -inf, or of the lowest float, bars a word; a target so barred has an infinite loss; logits of 1e30 give
    weights of 0 and 1; one NaN logit makes its row NaN."""
    rng = np.random.default_rng(4)
    for rows, k, vocab in ((5, 16, 300), (40, 130, 515), (9, 130, 2515), (500, 600, 1001), (2100, 900, 2003)):
        barred(hip, rng, rows, k, vocab)
    big = np.zeros((2, 1), np.float32) + 1e15
    wide = np.array([[1e15, -1e15, 0]], np.float32)
    value, dx, dw, _ = loss(hip, big, wide, None, np.array([0, 2]))
    assert value[0] == 0 and abs(value[1] / 1e30 - 1) < 1e-6
    assert np.array_equal(dw, [[1e15 * np.float32(1), 0, -1e15 * np.float32(1)]])


def barred(hip, rng, rows, k, vocab):
    x, w = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((k, vocab)).astype(np.float32)
    if k > 16:
        w *= np.float32(k ** -0.5)
    targets = rng.integers(0, vocab, rows)
    targets[[1, 2]] = 7, vocab - 1
    for low in (-np.inf, np.finfo(np.float32).min):
        b = np.where(np.arange(vocab) % 2 == 0, 0, low).astype(np.float32)
        b[targets] = 0
        open_ = b == 0
        want = D.cross_entropy(x, w[:, open_], None, np.cumsum(open_)[targets] - 1)
        bound = D.cross_entropy_bounds(x, w[:, open_], None, np.cumsum(open_)[targets] - 1)
        got = loss(hip, x, w, b, targets)
        close(got[0], want[0], bound[0])
        close(got[1], want[1], bound[1])
        close(got[2][:, open_], want[2], bound[2])
        assert (got[2][:, ~open_] == 0).all() and (got[3][~open_] == 0).all()
    targets[targets == 1] = 2
    targets[1] = 1
    b = np.where(np.arange(vocab) == 1, -np.inf, 0).astype(np.float32)
    value = loss(hip, x, w, b, targets, grads=False)
    assert value[1] == np.inf and np.isfinite(np.delete(value, 1)).all()
    assert np.isnan(loss(hip, x, w, np.full(vocab, -np.inf, np.float32), targets, grads=False)).all()
    b[:] = 0
    for bad in (np.nan, np.inf):
        b[9] = bad
        assert np.isnan(loss(hip, x, w, b, targets, grads=False)).all()
        assert np.isnan(loss(hip, x, w, b, targets)[0]).all()


def test_cross_entropy_without_parts(hip):
    rng = np.random.default_rng(5)
    for rows, k, vocab in ((3, 40, 90), (70, 40, 90), (600, 500, 1003), (2100, 900, 2003)):
        x, w = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((k, vocab)).astype(np.float32)
        targets = rng.integers(0, vocab, rows)
        full = loss(hip, x, w, None, targets)
        bound = D.cross_entropy_bounds(x, w, None, targets)
        for want in ((True, False, False), (False, True, False), (False, True, True), (False, False, False)):
            got = loss(hip, x, w, None, targets, want=want)
            for a, f, e, t in zip(got, full, bound, (True, *want)):
                if t:
                    close(a, f.astype(np.float64), 2 * e)
    dw, db, spare = (up(hip, np.full(s, 7, np.float32)) for s in ((4, 9), (8,), (3, 4)))
    hip.check(hip.lib().lmp_k_linear_cross_entropy_grad_f32(0, 4, 8, None, 4, None, 8, None, None, None, None, spare.ptr, 4, dw.ptr,
                                                            9, db.ptr))
    assert (dw.numpy()[:, :8] == 0).all() and (dw.numpy()[:, 8] == 7).all() and (db.numpy() == 0).all()
    assert (spare.numpy() == 7).all()


# ------------------------------------------------------------------ graphs

@pytest.mark.parametrize("rows,k,n,vocab", [(96, 64, 80, 500), (1500, 1100, 1201, 3001)])
def test_recorded_calls_equal_eager_ones(hip, rows, k, n, vocab):
    """Each operator recorded once and replayed, with eager calls and a second graph between the replays: every replay
    gives the eager bits, dropout those of the next call."""
    import ctypes as C
    rng = np.random.default_rng(11)
    lib = hip.lib()
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    x, w, b, g, wv = f32(rows, k), f32(k, 2 * n), f32(2 * n), f32(rows, n), f32(k, vocab)
    dev = {name: up(hip, a) for name, a in dict(x=x, w=w, b=b, g=g, wv=wv, pos=np.arange(rows), fr=np.array([1.0, 0.1]),
                                                t=rng.integers(-50, vocab, rows)).items()}

    def buffers():
        return {name: up(hip, np.zeros(s, np.float32)) for name, s in dict(
            y=(rows, k), z=(rows, k), d=(rows, k), h=(rows, n), pre=(rows, 2 * n), dx=(rows, k), dw=(k, 2 * n), db=(2 * n,),
            loss=(rows,), lx=(rows, k), lw=(k, vocab)).items()}

    def calls(o, state, used):
        p = lambda t: t.ptr  # noqa: E731
        hip.check(lib.lmp_k_rotary(4, rows, k, 3, 16, 4, 0, p(dev["x"]), k, p(dev["pos"]), p(dev["fr"]), 1.0, 0, p(o["y"]), k))
        hip.check(lib.lmp_k_dropout(4, rows * k, p(o["y"]), p(dev["x"]), 0.25, 9, p(state), p(used), p(o["z"])))
        hip.check(lib.lmp_k_dropout_backward(4, rows * k, p(dev["x"]), 0.25, 9, p(used), p(o["d"])))
        hip.check(lib.lmp_k_gated_linear_f32(0, rows, k, n, p(o["z"]), k, p(dev["w"]), 2 * n, p(dev["b"]), p(o["h"]), n,
                                             p(o["pre"]), 2 * n))
        hip.check(lib.lmp_k_gated_linear_backward_f32(0, rows, k, n, p(dev["g"]), n, p(o["z"]), k, p(dev["w"]), 2 * n, p(o["pre"]),
                                                      2 * n, p(o["dx"]), k, p(o["dw"]), 2 * n, p(o["db"])))
        hip.check(lib.lmp_k_linear_cross_entropy_grad_f32(rows, k, vocab, p(o["z"]), k, p(dev["wv"]), vocab, None, p(dev["t"]),
                                                          None, p(o["loss"]), p(o["lx"]), k, p(o["lw"]), vocab, None))

    sets = [(buffers(), up(hip, np.array([0, 0])), up(hip, np.array([0]))) for _ in range(3)]
    graphs = []
    for s in sets[:2]:
        hip.check(lib.lmp_rt_graph_begin())
        calls(*s)
        handle = C.c_void_p()
        hip.check(lib.lmp_rt_graph_end(C.byref(handle)))
        graphs.append(handle)
    for i in range(4):
        calls(*sets[2])
        for gr in graphs:
            hip.check(lib.lmp_rt_graph_launch(gr))
        for s in sets[:2]:
            assert s[1].numpy().tolist() == [i + 1, 0]
            for name, t in s[0].items():
                assert np.array_equal(t.numpy(), sets[2][0][name].numpy()), (i, name)
    for gr in graphs:
        hip.check(lib.lmp_rt_graph_destroy(gr))
