"""Rotary positions, dropout, gated linear layers and the vocabulary loss through the Python API: values and gradients against
64-bit forms and differences, refusals, graphs, and the example that uses them together."""
import math
import sys
from pathlib import Path

import numpy as np
import pytest

import _decoder as D

ROOT = Path(__file__).resolve().parent.parent


def test_rotary_frequencies():
    from rushlite_amd.nets import layers
    f, scale = layers.rotary_frequencies(8, 100.0)
    assert np.allclose(f, [1, 100 ** -0.25, 0.1, 100 ** -0.75], rtol=1e-15) and scale == 1
    assert np.allclose(layers.rotary_frequencies(8, 100.0, dict(kind="linear", factor=4))[0], f / 4, rtol=1e-15)
    stretched, scale = layers.rotary_frequencies(8, 100.0, dict(kind="base", factor=4))
    assert scale == 1 and stretched[0] == 1 and abs(stretched[-1] * 4 / f[-1] - 1) < 1e-14
    parts, scale = layers.rotary_frequencies(64, 10000.0, dict(kind="by_parts", factor=8, original=4096))
    f, _ = layers.rotary_frequencies(64, 10000.0)
    turns = 4096 * f / (2 * math.pi)
    assert np.array_equal(parts[turns > 32], f[turns > 32]) and np.allclose(parts[turns < 1] * 8, f[turns < 1], rtol=1e-15)
    assert (np.diff(parts) < 0).all() and abs(scale - (0.1 * math.log(8) + 1)) < 1e-15
    assert len(layers.rotary_frequencies(0)[0]) == 0 and len(layers.rotary_frequencies(2)[0]) == 1
    for bad in (dict(rotary_dim=3), dict(rotary_dim=4, base=0), dict(rotary_dim=4, scaling=dict(kind="linear", factor=0)),
                dict(rotary_dim=4, scaling=dict(kind="other", factor=2)),
                dict(rotary_dim=4, scaling=dict(kind="by_parts", factor=2, original=64, slow=4, fast=4))):
        with pytest.raises(ValueError, match="rotary_frequencies"):
            layers.rotary_frequencies(**bad)
    with pytest.raises(ValueError, match="above head_dim"):
        layers.Rotary(8, 10)
    with pytest.raises(ValueError, match="another head_dim"):
        layers.SelfAttention(32, 4, rotary=layers.Rotary(16))


def test_cpu_tensors_and_bad_arguments_are_refused():
    import rushlite_amd as rsl
    from rushlite_amd.nets import layers
    cpu, i64, f64 = rsl.device.cpu, rsl.dtype.int64, rsl.dtype.float64

    def v(a, dtype=rsl.dtype.float32):
        return rsl.Variable(np.asarray(a), False, cpu, dtype)

    x, t = v(np.ones((2, 4))), v([0, 1], i64)
    f = rsl._C._Tensor(np.ones(2), [2], cpu, f64)
    turn = dict(heads=1, head_dim=4)
    for args, text in (((x, t, f), "not registered"), ((v(np.ones((2, 4)), i64), t, f), "float32 or float64"),
                       ((v(np.ones(4)), t, f), "two axes"), ((x, v([0, 1, 2], i64), f), "positions"),
                       ((x, v([0.0, 1.0]), f), "positions"), ((x, t, rsl._C._Tensor(np.ones(3), [3], cpu, f64)), "3 pairs"),
                       ((x, t, v(np.ones(2)).data), "frequencies")):
        with pytest.raises(RuntimeError, match=text):
            rsl.rotary(*args, **turn)
    with pytest.raises(ValueError, match="negative"):
        rsl.rotary(x, t, f, heads=-1, head_dim=4)
    with pytest.raises(ValueError, match="rate"):
        layers.RandomDropout(1.5, None)
    state = rsl._C._Tensor(np.zeros(2, np.int64), [2], cpu, i64)
    for args, text in (((x, None, 0.1, 1, state), "not registered"), ((x, v(np.ones((2, 3))), 0.1, 1, state), "residual"),
                       ((t, None, 0.1, 1, state), "float32 or float64"), ((x, None, 0.1, 1, t.data.reshape([2])), "not registered"),
                       ((x, None, 0.1, 1, v([1.0, 2.0]).data), "generator")):
        with pytest.raises(RuntimeError, match=text):
            rsl._C._dropout(*args)
    w = v(np.ones((4, 6)))
    for args, text in (((x, w), "not registered"), ((x, v(np.ones((3, 6)))), "do not multiply"),
                       ((x, v(np.ones((4, 5)))), "as many more"), ((x, w, v(np.ones(5))), "bias must have 6"),
                       ((x, v(np.ones((4, 6)), f64)), "float32 on one device"), ((v(np.ones(4)), w), "do not multiply")):
        with pytest.raises(RuntimeError, match=text):
            rsl.gated_linear(*args)
    with pytest.raises(ValueError, match="unknown gate 'tanh'"):
        rsl.gated_linear(x, w, None, "tanh")
    for args, text in (((x, w, None, t), "not registered"), ((x, w, None, v([0, 1, 2], i64)), "targets"),
                       ((x, w, None, v([0, 1])), "targets"), ((x, w, None, t, v([1.0])), "weights"),
                       ((x, w, v(np.ones(5)), t), "bias must have 6"), ((v(np.ones((0, 4))), w, None, v([], i64)), "no rows")):
        with pytest.raises(RuntimeError, match=text):
            rsl.linear_cross_entropy(*args)
    with pytest.raises(RuntimeError, match="targets"):
        rsl.linear_cross_entropy_rows(x, w, None, v([0], i64))


gpu = pytest.mark.gpu


@pytest.fixture
def rsl():
    import rushlite_amd
    if not rushlite_amd.hip.is_available():
        pytest.fail("no HIP device visible to a test marked gpu")
    return rushlite_amd


def close(got, want, bound, what=""):
    err = np.abs(np.asarray(got, np.float64) - want)
    assert (err <= bound).all(), (what, float(err.max()))


def ints(rsl, a):
    return rsl.Variable(np.asarray(a, np.int64), dtype=rsl.dtype.int64)


def total(v):
    return v.sum(1).sum(0)


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_and_its_gradient(rsl, interleaved):
    from rushlite_amd.nets import layers
    rng = np.random.default_rng(1)
    x, g = (rng.standard_normal((9, 70)).astype(np.float32) for _ in range(2))
    layer = layers.Rotary(16, 12, interleaved=interleaved, scaling=dict(kind="by_parts", factor=4, original=64))
    q, k = [3, 1, 2, 0], [3, 5, 2, 4]
    positions = layers.packed_positions([5, *q[1:], 1], [5, *k[1:], 1])
    want_positions = [0, 1, 2, 3, 4, 4, 0, 1, 0]
    assert positions.numpy().tolist() == want_positions
    xv = rsl.Variable(x, True)
    y = layer(xv, positions, 4)
    assert y.grad_fn == "RotaryBackward"
    total(y * rsl.Variable(g)).backward()
    args = 4, 16, 12, interleaved, np.array(want_positions), layer.frequencies, layer.scale
    close(y.numpy(), D.rotary(x, *args), D.rotary_bound(x, *args))
    close(xv.grad.numpy(), D.rotary(g, *args, inverse=True), D.rotary_bound(g, *args))
    assert list(layer.parameters()) == []
    with rsl.no_grad():
        assert not layer(xv, positions, 4).requires_grad


@gpu
def test_rotary_scores_depend_on_distances_alone(rsl):
    """Queries and keys moved by one offset together give the same attention."""
    from rushlite_amd.nets import layers
    rng = np.random.default_rng(2)
    rsl.manual_seed(3)
    layer = layers.SelfAttention(32, 4, 2, rotary=layers.Rotary(8))
    x = rsl.Variable(0.1 * rng.standard_normal((12, 32)).astype(np.float32))
    plan = layer.plan([7, 5])
    a = layer(x, plan, layers.packed_positions([7, 5])).numpy()
    b = layer(x, plan, ints(rsl, layers.packed_positions([7, 5]).numpy() + 1000)).numpy()
    c = layer(x, plan, ints(rsl, np.zeros(12))).numpy()
    assert np.abs(a - b).max() < 1e-4 * np.abs(a).max() < np.abs(a - c).max()
    with pytest.raises(ValueError, match="positions"):
        layer(x, plan)


@gpu
def test_dropout_and_its_gradients(rsl):
    from rushlite_amd.nets import layers
    rng = np.random.default_rng(3)
    x, r, g = (rng.standard_normal((33, 21)).astype(np.float32) for _ in range(3))
    generator = rsl.Generator(77, calls=4)
    xv, rv = rsl.Variable(x, True), rsl.Variable(r, True)
    y = rsl.dropout(xv, 0.4, generator, rv)
    rsl.dropout(xv, 0.4, generator)  # another call before the backward pass
    total(y * rsl.Variable(g)).backward()
    keep = D.kept(x.size, 0.4, 77, 4).reshape(x.shape)
    want = np.where(keep, x.astype(np.float64) / 0.6, 0)
    close(y.numpy(), r + want, 2.01 * D.U32 * np.abs(want) + D.U32 * np.abs(r + want))
    close(xv.grad.numpy(), np.where(keep, g / 0.6, 0), 2.01 * D.U32 * np.abs(g) / 0.6)
    assert np.array_equal(rv.grad.numpy(), g)
    assert generator.calls == 6
    # the same variable on both paths: 1 + kept / 0.6
    both = rsl.Variable(x, True)
    total(rsl.dropout(both, 0.4, generator, both)).backward()
    keep = D.kept(x.size, 0.4, 77, 6).reshape(x.shape)
    close(both.grad.numpy(), 1 + keep / 0.6, 4 * D.U32 * 2.7)
    # only the residual wants a gradient; none does; the layer switched off
    rv.zero_grad()
    total(rsl.dropout(rsl.Variable(x), 0.4, generator, rv)).backward()
    assert (rv.grad.numpy() == 1).all()
    assert not rsl.dropout(rsl.Variable(x), 0.4, generator).requires_grad
    layer = layers.RandomDropout(0.4, generator)
    layer.active = False
    assert layer(xv) is xv and np.array_equal(layer(xv, rv).numpy(), x + r)
    saved = generator.state_dict()
    a = rsl.dropout(xv, 0.4, generator).numpy()
    generator.load_state_dict(saved)
    assert np.array_equal(rsl.dropout(xv, 0.4, generator).numpy(), a)


@gpu
def test_gated_linear_and_its_gradients(rsl):
    from rushlite_amd.nets import layers
    rng = np.random.default_rng(4)
    x, w, b, g = (rng.standard_normal(s).astype(np.float32) for s in ((40, 24), (24, 36), (36,), (40, 18)))
    for gate in ("silu", "gelu", "gelu_tanh", "sigmoid"):
        for bias in (b, None):
            xv, wv, bv = rsl.Variable(x, True), rsl.Variable(w, True), None if bias is None else rsl.Variable(b, True)
            h = rsl.gated_linear(xv, wv, bv, gate)
            assert h.grad_fn == "GatedLinearBackward" and h.shape == [40, 18]
            total(h * rsl.Variable(g)).backward()
            grads = [t.grad.numpy() for t in (xv, wv, bv) if t is not None]
            for a, want, e in zip([h.numpy(), *grads], D.gated(gate, x, w, bias, g), D.gated_bounds(gate, x, w, bias, g)):
                close(a, want, e, gate)
    # frozen weights; a second pass adds
    xv = rsl.Variable(x, True)
    total(rsl.gated_linear(xv, rsl.Variable(w), None)).backward()
    once = xv.grad.numpy().copy()
    total(rsl.gated_linear(xv, rsl.Variable(w), None)).backward()
    assert np.array_equal(xv.grad.numpy(), 2 * once)
    with rsl.no_grad():
        assert not rsl.gated_linear(xv, wv).requires_grad
    rsl.manual_seed(1)
    net = layers.GatedFeedForward(24, 30, "gelu", bias=False)
    assert sorted(n for n, _ in net.named_parameters()) == ["down.weights", "up.weights"] and net(xv).shape == [40, 24]


@gpu
def test_cross_entropy_and_its_gradients(rsl):
    from rushlite_amd.nets import layers
    rng = np.random.default_rng(5)
    x, w, b = (rng.standard_normal(s).astype(np.float32) for s in ((50, 16), (16, 90), (90,)))
    targets, weights = rng.integers(-30, 90, 50), rng.random(50).astype(np.float32)
    counted = np.maximum((targets >= 0).sum(), 1)
    for bias, wt in ((b, weights), (None, None), (b, None)):
        share = wt if wt is not None else ((targets >= 0) / np.float32(counted)).astype(np.float32)
        xv, wv, bv = rsl.Variable(x, True), rsl.Variable(w, True), None if bias is None else rsl.Variable(b, True)
        loss = rsl.linear_cross_entropy(xv, wv, bv, ints(rsl, targets), None if wt is None else rsl.Variable(wt))
        assert loss.shape == [1] and loss.grad_fn == "LinearCrossEntropyBackward"
        (loss * 3.0).backward()
        want, e = D.cross_entropy(x, w, bias, targets, share), D.cross_entropy_bounds(x, w, bias, targets, share)
        sum_of = (want[0] * share).sum()
        close(loss.numpy(), sum_of, (e[0] * share).sum() + 60 * D.U32 * (np.abs(want[0]) * share).sum())
        for t, d, bound in zip((xv, wv, bv), want[1:], e[1:]):
            if t is not None:  # the share's rounding, the factor's product
                close(t.grad.numpy(), 3 * d, 3 * bound + 4 * D.U32 * np.abs(3 * d))
        close(rsl.linear_cross_entropy_rows(xv, wv, bv, ints(rsl, targets)).numpy(), want[0], e[0])
    # through the layer, twice: gradients add; only the bias wanted
    rsl.manual_seed(2)
    head = layers.VocabularyLoss(16, 90)
    for _ in range(2):
        head(rsl.Variable(x), ints(rsl, targets)).backward()
    grads = D.cross_entropy(x, head.head.weights.numpy(), head.head.bias.numpy(), targets, share)
    e = D.cross_entropy_bounds(x, head.head.weights.numpy(), head.head.bias.numpy(), targets, share)
    close(head.head.weights.grad.numpy(), 2 * grads[2], 2 * e[2] + 8 * D.U32 * np.abs(grads[2]))
    bv = rsl.Variable(b, True)
    rsl.linear_cross_entropy(rsl.Variable(x), rsl.Variable(w), bv, ints(rsl, targets)).backward()
    close(bv.grad.numpy(), D.cross_entropy(x, w, b, targets, share)[3],
          D.cross_entropy_bounds(x, w, b, targets, share)[3] + 4 * D.U32)
    assert head.logits(rsl.Variable(x)).shape == [50, 90] and not head.rows(rsl.Variable(x), ints(rsl, targets)).requires_grad
    with rsl.no_grad():
        assert not head(rsl.Variable(x), ints(rsl, targets)).requires_grad
    # no row counts: a loss of 0, gradients of 0
    xv = rsl.Variable(x, True)
    loss = rsl.linear_cross_entropy(xv, rsl.Variable(w), None, ints(rsl, np.full(50, -1)))
    loss.backward()
    assert loss.tolist() == [0.0] and (xv.grad.numpy() == 0).all()


@gpu
def test_the_decoder_gradients_against_differences(rsl):
    """All of them together, dropout included (the same calls of the generator each time)."""
    sys.path.insert(0, str(ROOT / "examples"))
    import decoder
    rsl.manual_seed(6)
    model = decoder.Decoder(40, "gelu")
    lengths = [9, 4, 1]
    rows, targets = decoder.variables(*decoder.batch(np.random.default_rng(0), 40, lengths))
    plan, positions = model.block0.attention.plan(lengths), decoder.layers.packed_positions(lengths)

    def loss():
        model.generator.load_state_dict({"seed": 5, "calls": 0})
        return model(rows, targets, plan, positions)

    model.zero_grad()
    loss().backward()
    rng = np.random.default_rng(1)
    for name in ("tokens", "block0.attention.qkv.weights", "block0.mlp.up.weights", "block1.mlp.up.bias", "loss.head.weights",
                 "block1.attention.out.bias", "norm.weights"):
        p = model.params[name]
        way = rng.standard_normal(p.shape).astype(np.float32)
        start, slope, h = p.numpy().copy(), float((p.grad.numpy().astype(np.float64) * way).sum()), 1e-2

        def difference(h):
            ends = []
            for sign in (1, -1):
                p.data.copy(rsl.Variable(start + np.float32(sign * h) * way).data)
                with rsl.no_grad():
                    ends.append(loss().tolist()[0])
            return (ends[0] - ends[1]) / (2 * h)

        # A central difference is s + a h^2 + b h^4 + ...: two of them leave s - b h^4 / 4, and a h^2 is 4 / 3 of their
        # distance.  With the fourth-order term no larger than the second-order one that is at most a third of the
        # distance.  The loss, some 4, is good to some 1e-6 in float32: 2e-6 / h in the half step's difference, 3e-4 in all.
        wide, near = difference(h), difference(h / 2)
        p.data.copy(rsl.Variable(start).data)
        assert abs((4 * near - wide) / 3 - slope) < abs(wide - near) / 3 + 1e-3, (name, slope, wide, near)


@gpu
def test_recorded_decoder_step_equals_the_eager_one(rsl):
    """Recorded while an eager graph of the same leaves is alive; replays, with eager work between them, equal eager steps
    bit for bit, each with a dropout of its own."""
    sys.path.insert(0, str(ROOT / "examples"))
    import decoder
    lengths = [20, 11, 1]
    host = decoder.batch(np.random.default_rng(3), 64, lengths)

    def build():
        rsl.manual_seed(7)
        model = decoder.Decoder(64)
        return model, rsl.optim.AdamW(model, lr=1e-3)

    inputs = decoder.variables(*host)
    eager, kept = build(), build()
    plan, positions = eager[0].block0.attention.plan(lengths), decoder.layers.packed_positions(lengths)

    def step(model, opt):
        opt.zero_grad()
        loss = model(*inputs, plan, positions)
        loss.backward()
        opt.step()
        return loss

    want = [step(*eager).tolist()[0]]
    alive = step(*kept)
    got = [alive.tolist()[0]]
    graph = rsl.hip.Graph()
    with graph.capture():
        loss = step(*kept)
    for _ in range(4):
        want.append(step(*eager).tolist()[0])
        graph.replay()
        got.append(loss.tolist()[0])
        assert np.isfinite(alive.tolist()[0])
        for a, b in zip(eager[0].parameters(), kept[0].parameters()):
            assert np.array_equal(a.numpy(), b.numpy())
    assert got == want and kept[0].generator.calls == eager[0].generator.calls == 5 * 4


@gpu
def test_rotary_first_called_in_a_recording(rsl):
    from rushlite_amd.nets import layers
    layer, positions = layers.Rotary(8), layers.packed_positions([5])
    x = rsl.Variable(np.random.default_rng(2).standard_normal((5, 16)).astype(np.float32))
    graph = rsl.hip.Graph()
    with graph.capture(), rsl.no_grad():
        y = layer(x, positions, 2)
    for _ in range(3):
        graph.replay()
        with rsl.no_grad():
            assert np.array_equal(y.numpy(), layer(x, positions, 2).numpy())


@gpu
def test_the_example_runs(rsl):
    sys.path.insert(0, str(ROOT / "examples"))
    import decoder
    model, losses = decoder.train(6, vocabulary=101, gate="sigmoid", report=lambda _: None)
    assert len(losses) == 6 and np.isfinite(losses).all() and model.generator.calls == 6 * 4
    scores = decoder.score(model, [40, 120])
    assert len(scores) == 2 and np.isfinite(scores).all()
    assert scores == decoder.score(model, [40, 120])
