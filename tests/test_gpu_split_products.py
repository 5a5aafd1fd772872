"""Products of operands that spread widely along K, in the sizes whose products run on split operands: gated linear layers and
the vocabulary loss against 64-bit forms.

The bounds are four times those of tests/_decoder.py, which count a rounding a term: a sum of k products errs by 4 k + 64
units of its magnitudes, whatever else its operands hold."""
import numpy as np
import pytest

import _decoder as D
from test_gpu_decoder import close, gated, loss

pytestmark = pytest.mark.gpu


def gated_operands(rng, rows, k, n):
    return (rng.standard_normal((rows, k)).astype(np.float32), (rng.standard_normal((k, 2 * n)) * k ** -0.5).astype(np.float32),
            rng.standard_normal((rows, n)).astype(np.float32))


def check_gated(hip, gate, x, w, g, what=()):
    want, bound = D.gated(gate, x, w, None, g), D.gated_bounds(gate, x, w, None, g)
    for a, v, e, part in zip(gated(hip, gate, x, w, None, g), want, bound, ("h", "dx", "dw", "db")):
        # a product below float32's normal range, 2^-126, is off by up to itself
        close(a, v, 4 * e + 2.0 ** -126, (*what, part))


def check_loss(hip, x, w, b, targets, weights=None, what=()):
    want, bound = D.cross_entropy(x, w, b, targets, weights), D.cross_entropy_bounds(x, w, b, targets, weights)
    for a, v, e, part in zip(loss(hip, x, w, b, targets, weights), want, bound, ("loss", "dx", "dw", "db")):
        close(a, v, 4 * e, (*what, part))
    close(loss(hip, x, w, b, targets, grads=False), want[0], 4 * bound[0], (*what, "loss alone"))


# Rows, inputs and outputs that take several tiles, with K in one piece and in more (tests/native/half_plan_cases.cpp).
GATED = [(1500, 1100, 1201), (1031, 2050, 1001), (5003, 600, 1201)]
LOSS = [(2100, 900, 2003), (5003, 600, 1009)]


@pytest.mark.parametrize("rows,k,n", GATED)
def test_gated_an_input_column_far_above_the_others(hip, rows, k, n):
    """Its weights are zeros, or small enough to make up for it."""
    rng = np.random.default_rng(1)
    x, w, g = gated_operands(rng, rows, k, n)
    for c in (1e5, 1e7, 1e9, 1e11, 1e13, 1e25):
        for weight in (0.0, 1 / c):
            x[:, 5], w[5] = c, weight
            check_gated(hip, "sigmoid", x, w, g, (c, weight))


@pytest.mark.parametrize("rows,k,n", GATED)
def test_gated_rows_and_weights_that_meet_zeros(hip, rows, k, n):
    """A row of huge inputs without a gradient, and a huge weight of an output without one."""
    rng = np.random.default_rng(2)
    for c in (1e8, 1e10, 1e12):
        x, w, g = gated_operands(rng, rows, k, n)
        x[5] *= np.float32(c)
        g[5] = 0
        check_gated(hip, "sigmoid", x, w, g, (c, "row"))
        x, w, g = gated_operands(rng, rows, k, n)
        w[3, 7], w[4, n + 9] = c, -c
        x[:, 3:5] *= np.float32(1 / c)
        g[:, [7, 9]] = 0
        check_gated(hip, "sigmoid", x, w, g, (c, "weight"))


def test_gated_few_sums_far_below_their_operands(hip):
    """A column with one weight, met by a few inputs of almost nothing; rows and columns of zeros beside them."""
    rng = np.random.default_rng(3)
    for rows, k, n in GATED:
        x, w, g = gated_operands(rng, rows, k, n)
        for col in (17, n - 1, n + 17, 2 * n - 1):
            w[:, col] = 0
            w[70, col] = 0.7
        few = [0, 63, 64, 200, rows - 1]
        x[few, 70] = [1e-9, -3e-12, 1e-20, 2e-30, 5e-7]
        x[300:340] = 0
        x[:, 90], w[:, 40] = 0, 0
        check_gated(hip, "silu", x, w, g)
        # the same of both gradients: an output with a gradient in one row, whose inputs are almost nothing, and an input
        # with one weight, for an output with gradients of almost nothing
        x, w, g = gated_operands(rng, rows, k, n)
        g[:, 7], g[9, 7] = 0, 1
        x[9, [3, 40, k - 1]] = [1e-12, -1e-20, 1e-9]
        w[5], w[5, 20] = 0, 0.3
        g[[4, 70, rows - 1], 20] = [1e-11, -1e-18, 1e-25]
        check_gated(hip, "sigmoid", x, w, g)


def test_gated_infinities_and_weights_of_almost_nothing(hip):
    """An infinity times a value far below the largest it is held beside is an infinity, as in float32."""
    rng = np.random.default_rng(4)
    for rows, k, n in GATED:
        x, w, g = gated_operands(rng, rows, k, n)
        x[2, 3], w[3] = np.inf, 1e-30
        h = gated(hip, "sigmoid", x, w, None, g, keep=False)
        assert (h[2] == np.inf).all() and np.isfinite(np.delete(h, 2, 0)).all()
        x[2, 3] = 0
        clean = gated(hip, "sigmoid", x, w, None, g, keep=False)
        bound = D.gated_bounds("sigmoid", x, w, None, g)[0]
        close(np.delete(h, 2, 0), np.delete(clean, 2, 0).astype(np.float64), np.delete(8 * bound, 2, 0))
        # of the weights: one column of the second half
        x[:, 8] = np.abs(x[:, 8]) + 1e-30
        x[20:200, 8] = 1e-25
        w[8, n + 13] = np.inf
        h = gated(hip, "sigmoid", x, w, None, g, keep=False)
        assert (h[:, 13] == np.inf).all() and np.isfinite(np.delete(h, 13, 1)).all()


@pytest.mark.parametrize("rows,k,vocab", LOSS)
def test_loss_of_inputs_far_above_the_others(hip, rows, k, vocab):
    rng = np.random.default_rng(5)
    targets, weights = rng.integers(0, vocab, rows), rng.random(rows).astype(np.float32)
    w0 = (2 * rng.standard_normal((k, vocab)) * k ** -0.5).astype(np.float32)
    for c in (1e7, 1e10, 1e13):
        x, w = rng.standard_normal((rows, k)).astype(np.float32), w0.copy()
        x[:, 5], w[5] = c, 0
        check_loss(hip, x, w, None, targets, weights, (c, "column"))
    for c in (1e8, 1e12):
        # rows that count for nothing, and a word that a bias bars
        x, w, b = rng.standard_normal((rows, k)).astype(np.float32), w0.copy(), np.zeros(vocab, np.float32)
        x[5] *= np.float32(c)
        weights[5] = 0
        t = targets.copy()
        t[t == 11] = 12
        w[:, 11] *= np.float32(c)
        b[11] = -np.inf
        open_ = np.arange(vocab) != 11
        got = loss(hip, x, w, b, t, weights)
        args = x, w[:, open_], None, np.cumsum(open_)[t] - 1, weights
        for a, v, e, part in zip((got[0], got[1], got[2][:, open_]), D.cross_entropy(*args), D.cross_entropy_bounds(*args),
                                 ("loss", "dx", "dw")):
            keep = np.arange(len(a)) != 5 if part != "dw" else slice(None)
            close(a[keep], v[keep], 4 * e[keep], (c, part))


@pytest.mark.parametrize("rows,k,vocab", LOSS)
def test_loss_of_sparse_inputs_and_steep_logits(hip, rows, k, vocab):
    """Half of the inputs are zeros and the shares of a row span twenty orders of magnitude: where a word's own row has a zero,
    its gradient is what the small shares add up to."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    x[rng.random((rows, k)) < 0.5] = 0
    w = (9 * rng.standard_normal((k, vocab)) * k ** -0.5).astype(np.float32)
    targets, weights = rng.integers(-vocab // 4, vocab, rows), rng.random(rows).astype(np.float32)
    check_loss(hip, x, w, None, targets, weights)
    # rows that are sure of their target
    z = x.astype(np.float64) @ w
    check_loss(hip, x, w, None, np.where(targets < 0, -1, z.argmax(1)), weights, ("sure",))


@pytest.mark.parametrize("rows,k,n", [(423, 1000, 16001), (2300, 520, 5003), (1005, 2000, 1501), (8200, 1024, 2080)])
def test_gated_in_every_tile(hip, rows, k, n):
    """Forward in tiles of 256 x 256 and 128 x 128, the gradients in 256 x 256 with and without K in pieces: operands of one
    size, and a column, a row and a weight far above the others."""
    rng = np.random.default_rng(7)
    x, w, g = gated_operands(rng, rows, k, n)
    if rows < 8000:
        check_gated(hip, "silu", x, w, g)
    x[:, 5], w[5] = 1e9, 0
    x[rows - 2] *= np.float32(1e10)
    g[rows - 2] = 0
    w[3, 7], w[4, n + 9] = 1e10, -1e10
    x[:, 3:5] *= np.float32(1e-10)
    g[:, [7, 9]] = 0
    check_gated(hip, "sigmoid", x, w, g)


@pytest.mark.parametrize("rows,k,vocab", [(423, 1000, 32003), (2300, 520, 10007)])
def test_loss_in_every_tile(hip, rows, k, vocab):
    rng = np.random.default_rng(8)
    x, w = rng.standard_normal((rows, k)).astype(np.float32), (2 * rng.standard_normal((k, vocab)) * k ** -0.5).astype(np.float32)
    targets, weights = rng.integers(-vocab // 4, vocab, rows), rng.random(rows).astype(np.float32)
    check_loss(hip, x, w, rng.standard_normal(vocab).astype(np.float32), targets, weights)
    x[:, 5], w[5] = 1e9, 0
    x[:, 3], w[3, 7] = x[:, 3] * np.float32(1e-10), 1e10
    check_loss(hip, x, w, None, targets, weights, ("spread",))


def test_the_same_bits_from_call_to_call(hip):
    """In whatever order the sums that are formed again were found, one by one and tile by tile."""
    rng = np.random.default_rng(9)
    for rows, k, n in GATED:
        x, w, g = gated_operands(rng, rows, k, n)
        w[:, 17], w[70, 17] = 0, 0.7
        x[:rows // 2:40, 70] = 1e-9
        x[:, 5], w[5, n:] = 1e9, 0
        g[rows // 2:] = 0
        first = gated(hip, "silu", x, w, None, g)
        for _ in range(3):
            for a, b in zip(gated(hip, "silu", x, w, None, g), first):
                assert np.array_equal(a, b)
    for rows, k, vocab in LOSS:
        x, w = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((k, vocab)).astype(np.float32)
        x[rng.random((rows, k)) < 0.5] = 0
        targets = rng.integers(-5, vocab, rows)
        first = loss(hip, x, w, None, targets)
        for _ in range(3):
            for a, b in zip(loss(hip, x, w, None, targets), first):
                assert np.array_equal(a, b)


def test_a_recorded_call_looks_at_each_replays_operands(hip):
    """Recorded on operands of one size, replayed on others that spread, and again on the first."""
    import ctypes as C
    from test_gpu_decoder import up
    lib, rng = hip.lib(), np.random.default_rng(10)
    rows, k, n = GATED[0]
    plain = gated_operands(rng, rows, k, n)
    spread = [a.copy() for a in plain]
    spread[0][:, 5], spread[1][5] = 1e11, 0
    spread[0][7] *= np.float32(1e12)
    spread[2][7] = 0
    dev = [up(hip, a) for a in plain]
    outs = [up(hip, np.zeros(s, np.float32)) for s in ((rows, n), (rows, 2 * n), (rows, k), (k, 2 * n))]
    x, w, g, h, pre, dx, dw = (t.ptr for t in dev + outs)

    def calls():
        hip.check(lib.lmp_k_gated_linear_f32(4, rows, k, n, x, k, w, 2 * n, None, h, n, pre, 2 * n))
        hip.check(lib.lmp_k_gated_linear_backward_f32(4, rows, k, n, g, n, x, k, w, 2 * n, pre, 2 * n, dx, k, dw, 2 * n, None))

    hip.check(lib.lmp_rt_graph_begin())
    calls()
    graph = C.c_void_p()
    hip.check(lib.lmp_rt_graph_end(C.byref(graph)))
    for operands in (plain, spread, plain, spread):
        for t, a in zip(dev, operands):
            hip.check(lib.lmp_rt_memcpy_h2d(t.ptr, a.ctypes.data, a.nbytes))
        calls()
        want = [t.numpy() for t in outs]
        for t in outs:
            hip.check(lib.lmp_rt_memcpy_h2d(t.ptr, np.full(t.shape, 7, np.float32).ctypes.data, t.nbytes))
        hip.check(lib.lmp_rt_graph_launch(graph))
        for t, a in zip(outs, want):
            assert np.array_equal(t.numpy(), a)
    hip.check(lib.lmp_rt_graph_destroy(graph))
