"""The ways of the vocabulary loss and the gated layer that sizes or memory choose: few rows over large vocabularies, several
pieces with only some gradients wanted, and memory too short for the split operands."""
import ctypes as C

import numpy as np
import pytest

import _decoder as D
from test_gpu_decoder import close, gated, loss, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,k,vocab", [(1, 64, 33000), (5, 33, 40009), (31, 130, 65539), (40, 16, 70001), (2, 8, 131072)])
def test_loss_of_few_rows_over_a_large_vocabulary(hip, rows, k, vocab):
    rng = np.random.default_rng(vocab)
    x, w = rng.standard_normal((rows, k)).astype(np.float32), (2 * rng.standard_normal((k, vocab)) * k ** -0.5).astype(np.float32)
    b = rng.standard_normal(vocab).astype(np.float32)
    targets = rng.integers(0, vocab, rows)
    targets[0] = vocab - 1
    if rows > 2:
        targets[1], targets[2] = -7, 0
    want, bound = D.cross_entropy(x, w, b, targets), D.cross_entropy_bounds(x, w, b, targets)
    close(loss(hip, x, w, b, targets, grads=False), want[0], bound[0], "loss alone")
    for a, v, e, what in zip(loss(hip, x, w, b, targets), want, bound, ("loss", "dx", "dw", "db")):
        close(a, v, e, what)
    # a barred word, a row of nothing else, one NaN
    b[7] = -np.inf
    targets[targets == 7] = 8
    open_ = np.arange(vocab) != 7
    at = np.where(targets < 0, -1, np.cumsum(open_)[targets] - 1)
    close(loss(hip, x, w, b, targets, grads=False), D.cross_entropy(x, w[:, open_], b[open_], at)[0],
          D.cross_entropy_bounds(x, w[:, open_], b[open_], at)[0])
    assert np.isnan(loss(hip, x, w, np.full(vocab, -np.inf, np.float32), np.abs(targets) % vocab, grads=False)).all()
    b[vocab - 2] = np.nan
    assert np.isnan(loss(hip, x, w, b, np.abs(targets) % vocab, grads=False)).all()


@pytest.mark.parametrize("k", [12, 64])  # as they are, and split into fp16 parts
def test_loss_in_several_pieces_of_some_gradients(hip, k):
    """What each piece leaves does not depend on which other gradients are wanted but for the order of its sums."""
    rng = np.random.default_rng(9)
    rows, vocab = 4500, 30011
    x, w = rng.standard_normal((rows, k)).astype(np.float32), (rng.standard_normal((k, vocab)) * k ** -0.5).astype(np.float32)
    targets, weights = rng.integers(-vocab // 4, vocab, rows), rng.random(rows).astype(np.float32)
    full = loss(hip, x, w, None, targets, weights)
    # each of the two errs by the roundings of its sums, one for each term and 16 for the operands' parts
    z = x @ w
    d = np.exp(z - z.max(1, keepdims=True))
    d *= (weights * (targets >= 0) / d.sum(1))[:, None]
    rows_of, columns = d.sum(1) + weights, d.sum(0) + np.bincount(targets[targets >= 0], weights[targets >= 0], vocab)
    e_dx = 2 * (vocab + 16) * D.U32 * np.abs(w).max() * rows_of[:, None]
    e_dw = 2 * (rows + 16) * D.U32 * np.abs(x).max() * columns
    for want in ((True, False, False), (False, True, False), (False, True, True)):
        got = loss(hip, x, w, None, targets, weights, want=want)
        assert np.array_equal(got[0], full[0])
        if want[0]:
            close(got[1], full[1].astype(np.float64), e_dx, want)
        if want[1]:
            close(got[2], full[2].astype(np.float64), e_dw, want)
        if want[2]:
            close(got[3], full[3].astype(np.float64), 2 * (rows + 16) * D.U32 * columns, want)


def test_losses_alone_of_a_long_batch_keep_to_their_workspace(hip):
    """40000 rows over 131072 words: 655 MB of maxima and sums, in pieces of 512 MB."""
    lib = hip.lib()
    rng = np.random.default_rng(11)
    rows, k, vocab = 40000, 32, 131072
    x, w = rng.standard_normal((rows, k)).astype(np.float32), (rng.standard_normal((k, vocab)) * k ** -0.5).astype(np.float32)
    targets = rng.integers(-vocab // 4, vocab, rows)
    dx, dw, dt, out = up(hip, x), up(hip, w), up(hip, targets.astype(np.int64)), up(hip, np.full(rows, 7, np.float32))
    hip.check(lib.lmp_rt_empty_cache())
    stats = hip.PoolStats()
    hip.check(lib.lmp_rt_pool_stats_get(C.byref(stats)))
    before = stats.reserved_bytes
    hip.check(lib.lmp_k_linear_cross_entropy_f32(rows, k, vocab, dx.ptr, k, dw.ptr, vocab, None, dt.ptr, out.ptr))
    got = out.numpy()
    hip.check(lib.lmp_rt_pool_stats_get(C.byref(stats)))
    assert stats.reserved_bytes - before < 600 << 20
    some = np.r_[0:40, 32600:32900, rows - 40:rows]  # on both sides of where the second piece begins
    args = x[some], w, None, targets[some]
    close(got[some], D.cross_entropy(*args)[0], D.cross_entropy_bounds(*args)[0])
    parts = [loss(hip, x[at:at + 8000], w, None, targets[at:at + 8000], grads=False) for at in range(0, rows, 8000)]
    close(got, np.concatenate(parts).astype(np.float64), 2 * D.cross_entropy_bounds(*args)[0].max())


def fill(hip, leave):
    """Takes the device's memory until no more than `leave` bytes and 64 MB are to be had in one piece, `leave` still are;
    returns what to free."""
    lib = hip.lib()
    free, total, runtime = C.c_size_t(), C.c_size_t(), C.CDLL("libamdhip64.so")

    def take(size):
        p = C.c_void_p()
        return p if lib.lmp_rt_malloc(C.byref(p), size) == 0 else None

    hip.check(lib.lmp_rt_empty_cache())
    assert runtime.hipMemGetInfo(C.byref(free), C.byref(total)) == 0
    held = [take(free.value - leave - (1 << 30))]
    assert held[0]
    # the pool's own spans between other tests' buffers, and what the device holds back of what it reports
    while (p := take(leave + (64 << 20))) is not None:
        hip.check(lib.lmp_rt_free(p))
        hip.check(lib.lmp_rt_empty_cache())
        held.append(take(64 << 20))
        assert held[-1] and len(held) < 1000
    assert lib.lmp_rt_malloc(None, 1) != 0 and b"null" in lib.lmp_rt_last_error()  # another message than what short memory leaves
    return held


def release(hip, held):
    for p in held:
        hip.check(hip.lib().lmp_rt_free(p))


def test_short_memory_takes_the_products_that_need_less(hip):
    """Where the split operands of the gated gradients (2.0 GB) and of the loss (0.85 GB) are not to be had, the fp32 products
    run, which need 0.84 and 0.27; and the loss takes smaller pieces where its copy of x (1.2 GB) is not."""
    lib = hip.lib()
    rng = np.random.default_rng(10)
    short_of = lambda: "memory" in lib.lmp_rt_last_error().decode()  # noqa: E731  (what the call met and went round)

    # whole numbers: the products are exact, so both ways give the same bits; sums of the rows stay below 2^24
    rows, k, n = 150000, 512, 700
    x, w, g = (rng.integers(-2, 3, s).astype(np.float32) for s in ((rows, k), (k, 2 * n), (rows, n)))
    g[rows // 8:] = 0
    plenty = gated(hip, "relu", x, w, None, g)
    dev = {name: up(hip, a) for name, a in dict(x=x, w=w, g=g).items()}
    outs = {name: up(hip, np.zeros(s, np.float32)) for name, s in dict(h=(rows, n), pre=(rows, 2 * n), dx=(rows, k), dw=(k, 2 * n),
                                                                       db=(2 * n,)).items()}
    p = {name: t.ptr for name, t in {**dev, **outs}.items()}
    relu = hip.GATE["relu"]
    hip.check(lib.lmp_k_gated_linear_f32(relu, rows, k, n, p["x"], k, p["w"], 2 * n, None, p["h"], n, p["pre"], 2 * n))
    held = fill(hip, 1_500_000_000)
    try:
        hip.check(lib.lmp_k_gated_linear_backward_f32(relu, rows, k, n, p["g"], n, p["x"], k, p["w"], 2 * n, p["pre"], 2 * n, p["dx"], k,
                                                      p["dw"], 2 * n, p["db"]))
        assert short_of()
        got = [outs[name].numpy() for name in ("h", "dx", "dw", "db")]
    finally:
        release(hip, held)
    for a, b in zip(got, plenty):
        assert np.array_equal(a, b)
    del dev, outs, x, g, got, plenty

    for rows, k, vocab, leave in ((4500, 64, 30011, 350_000_000), (2000, 150001, 20, 650_000_000)):
        x, w = rng.standard_normal((rows, k)).astype(np.float32), (rng.standard_normal((k, vocab)) * k ** -0.5).astype(np.float32)
        targets = rng.integers(-vocab // 4, vocab, rows)
        plenty, bound = loss(hip, x, w, None, targets), D.cross_entropy_bounds(x, w, None, targets)
        # the call's own buffers: x, w and their gradients
        held = fill(hip, leave + 2 * (x.nbytes + w.nbytes))
        try:
            got = loss(hip, x, w, None, targets)
            assert short_of()
        finally:
            release(hip, held)
        for a, b, e in zip(got, plenty, bound):
            close(a, b.astype(np.float64), 2 * e)
    hip.check(lib.lmp_rt_empty_cache())
