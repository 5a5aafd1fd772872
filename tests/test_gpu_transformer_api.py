"""The transformer operators through the Python API: values and gradients against 64-bit forms, refusals, graphs, the
optimizer's states, and the example that uses them together."""
import sys
from pathlib import Path

import numpy as np
import pytest

import _transformer as T

ROOT = Path(__file__).resolve().parent.parent


def test_cpu_tensors_and_bad_arguments_are_refused():
    import rushlite_amd as rsl
    cpu = rsl.device.cpu
    x = rsl.Variable(np.ones((2, 3), np.float32), device=cpu)
    with pytest.raises(RuntimeError, match="not registered"):
        rsl.layer_norm(x)
    with pytest.raises(RuntimeError, match="weight and bias"):
        rsl.layer_norm(x, rsl.Variable(np.ones(2, np.float32), device=cpu))
    with pytest.raises(RuntimeError, match="weight and bias"):
        rsl.layer_norm(x, None, rsl.Variable(np.ones(3), device=cpu, dtype=rsl.dtype.float64))
    with pytest.raises(RuntimeError, match="float32 or float64"):
        rsl.layer_norm(rsl.Variable(np.ones((2, 3), np.int32), device=cpu, dtype=rsl.dtype.int32))
    with pytest.raises(RuntimeError, match="no values"):
        rsl.layer_norm(rsl.Variable(np.ones((2, 0), np.float32), device=cpu))
    with pytest.raises(ValueError, match="32 or 8"):
        rsl.optim.AdamW([], bits=16)
    with pytest.raises(ValueError, match="requires a gradient"):
        rsl.optim.AdamW([x])
    with pytest.raises(ValueError, match="HIP device"):
        rsl.optim.AdamW([rsl.Variable(np.ones(3, np.float32), True, cpu)])
    with pytest.raises(ValueError, match="negative"):
        rsl.AttentionPlan([1], heads=-1, head_dim=4)
    from rushlite_amd.nets import layers
    with pytest.raises(ValueError, match="multiple"):
        layers.SelfAttention(10, 3)


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


@gpu
@pytest.mark.parametrize("dtype", ["float32", "float64"])
def test_layer_norm_and_its_gradients(rsl, dtype):
    rng = np.random.default_rng(1)
    x, g = rng.standard_normal((3, 5, 24)).astype(dtype), rng.standard_normal((3, 5, 24)).astype(dtype)
    w, b = rng.standard_normal(24).astype(dtype), rng.standard_normal(24).astype(dtype)
    kw = dict(requires_grad=True, dtype=getattr(rsl.dtype, dtype))
    xv, wv, bv = rsl.Variable(x, **kw), rsl.Variable(w, **kw), rsl.Variable(b, **kw)
    y = rsl.layer_norm(xv, wv, bv, 1e-3)
    assert y.shape == [3, 5, 24] and y.grad_fn == "LayerNormBackward"
    loss = (y * rsl.Variable(g, dtype=getattr(rsl.dtype, dtype))).sum(2).sum(1).sum(0)
    loss.backward()
    x2, g2 = x.reshape(15, 24), g.reshape(15, 24)
    scale = 1 if dtype == "float32" else 2.0 ** -29
    bound = {k: v * scale for k, v in T.layer_norm_bounds(g2, x2, w, b, 1e-3).items()}
    slack = 0 if dtype == "float32" else 1e-15
    close(y.numpy().reshape(15, 24), T.layer_norm(x2, w, b, 1e-3)[0], bound["y"] + slack, "y")
    dx, dw, db = T.layer_norm_backward(g2, x2, w, 1e-3)
    close(xv.grad.numpy().reshape(15, 24), dx, bound["dx"] + slack, "dx")
    close(wv.grad.numpy(), dw, bound["dw"] + slack, "dw")
    close(bv.grad.numpy(), db, bound["db"] + slack, "db")
    # a second backward accumulates; parts without a gradient are not formed
    rsl.layer_norm(xv, wv, bv, 1e-3).sum(2).sum(1).sum(0).backward()
    ones = np.ones_like(g2)
    close(bv.grad.numpy(), db + 15, (bound["db"] + T.layer_norm_bounds(ones, x2, w, b, 1e-3)["db"] * scale
                                     + 2 * T.U32 * scale * np.abs(db + 15)), "db twice")
    y = rsl.layer_norm(rsl.Variable(x, dtype=getattr(rsl.dtype, dtype)))
    assert not y.requires_grad
    with rsl.no_grad():
        assert not rsl.layer_norm(xv, wv).requires_grad


@gpu
def test_layer_norm_of_a_pending_input_and_of_no_rows(rsl):
    x = rsl.Variable(np.random.default_rng(0).standard_normal((4, 8)).astype(np.float32), True)
    with rsl.capture_on():
        y = rsl.layer_norm(x * 2.0 + 1.0)
    want = T.layer_norm((x.numpy() * 2 + 1), None, None, 1e-5)[0]
    assert np.abs(y.numpy() - want).max() < 1e-5
    y.sum(1).sum(0).backward()
    assert np.isfinite(x.grad.numpy()).all()
    w = rsl.Variable(np.ones(8, np.float32), True)
    empty = rsl.layer_norm(rsl.zeros([0, 8], True), w)
    assert empty.shape == [0, 8]


@gpu
def test_attention_and_its_gradients(rsl):
    ql, heads, kv, d = [9, 30], 4, 2, 16
    rng = np.random.default_rng(2)
    q, k, v, g = (rng.standard_normal((39, n * d)).astype(np.float32) for n in (heads, kv, kv, heads))
    plan = rsl.AttentionPlan(ql, heads=heads, kv_heads=kv, head_dim=d)
    assert (plan.queries, plan.keys, plan.heads, plan.kv_heads, plan.head_dim, plan.causal) == (39, 39, 4, 2, 16, True)
    want = T.attention(q, k, v, ql, ql, heads, kv, 0.25, True, g)
    bound = T.attention_bounds(q, k, v, ql, ql, heads, kv, 0.25, True, g)
    qv, kv_, vv = (rsl.Variable(a, True) for a in (q, k, v))
    o = rsl.attention(qv, kv_, vv, plan)
    (o * rsl.Variable(g)).sum(1).sum(0).backward()
    for a, w, b, what in zip((o.numpy(), qv.grad.numpy(), kv_.grad.numpy(), vv.grad.numpy()), (want[0], *want[2:]),
                             (bound[0], *bound[2:]), ("o", "dq", "dk", "dv")):
        close(a, w, b, what)
    rows = rsl.Variable(np.concatenate([q, k, v], 1), True)
    o2 = rsl.attention_qkv(rows, plan)
    (o2 * rsl.Variable(g)).sum(1).sum(0).backward()
    assert np.array_equal(o2.numpy(), o.numpy())
    assert np.array_equal(rows.grad.numpy(), np.concatenate([x.grad.numpy() for x in (qv, kv_, vv)], 1))
    # one tensor as keys and values both: its gradients add up
    both = rsl.Variable(k, True)
    (rsl.attention(rsl.Variable(q), both, both, plan) * rsl.Variable(g)).sum(1).sum(0).backward()
    want = T.attention(q, k, k, ql, ql, heads, kv, 0.25, True, g)
    bound = T.attention_bounds(q, k, k, ql, ql, heads, kv, 0.25, True, g)
    close(both.grad.numpy(), want[3] + want[4], bound[3] + bound[4] + T.U32 * np.abs(want[3] + want[4]), "dk + dv")


@gpu
def test_attention_refusals(rsl):
    plan = rsl.AttentionPlan([3], [5], heads=4, kv_heads=2, head_dim=8)
    z = lambda *s, **k: rsl.zeros(list(s), **k)  # noqa: E731
    good = z(3, 32), z(5, 16), z(5, 16)
    assert rsl.attention(*good, plan).shape == [3, 32]
    for args, text in (((z(4, 32), *good[1:]), "q has shape"), ((good[0], z(5, 15), good[2]), "k has shape"),
                       ((*good[:2], z(3, 16)), "v has shape"), ((z(96), *good[1:]), "q has shape"),
                       ((z(3, 32, dtype=rsl.dtype.float64), *good[1:]), "q must be float32")):
        with pytest.raises(RuntimeError, match=text):
            rsl.attention(*args, plan)
    with pytest.raises(RuntimeError, match="3 queries and 5 keys"):
        rsl.attention_qkv(z(3, 64), plan)
    for scale in (float("nan"), float("inf"), 1e300):
        with pytest.raises(RuntimeError, match="scale is not finite"):
            rsl.attention(*good, plan, scale)
    with pytest.raises(RuntimeError, match="multiple of kv_heads"):
        rsl.AttentionPlan([3], heads=3, kv_heads=2, head_dim=8)
    with pytest.raises(RuntimeError, match="one query length"):
        rsl.AttentionPlan([3], [1, 2], heads=2, head_dim=8)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_follows_the_formula(rsl, bits):
    """Several steps against 64 bits.  With 8 bits the moments are those the codes stand for."""
    rng = np.random.default_rng(3)
    shapes = [(40, 30), (30,), (1,), (300,)]
    host = [(0.1 * rng.standard_normal(s)).astype(np.float32) for s in shapes]
    params = [rsl.Variable(a, True) for a in host]
    opt = rsl.optim.AdamW(params, lr=0.01, weight_decay=lambda p: 0.1 if len(p.shape) > 1 else 0.0, bits=bits, seed=5)
    p64 = [a.astype(np.float64) for a in host]
    m = [np.zeros(s) for s in shapes]
    v = [np.zeros(s) for s in shapes]
    buffers = [rsl._storage_ptr(p.data) for p in params]
    for t in range(1, 6):
        grads = [(rng.standard_normal(s) * 0.01).astype(np.float32) for s in shapes]
        opt.zero_grad()
        total = None
        for p, g in zip(params, grads):
            term = p * rsl.Variable(g)
            while len(term.shape) > 1:
                term = term.sum(len(term.shape) - 1).reshape(term.shape[:-1])
            term = term.sum(0)
            total = term if total is None else total + term
        total.backward()
        opt.step()
        assert opt.steps == t
        for i, g in enumerate(grads):
            p64[i], m[i], v[i] = T.adamw(p64[i], g, m[i], v[i], t, 0.01, 0.9, 0.999, 1e-8, 0.1 if len(shapes[i]) > 1 else 0.0)
            # an update is at most a few lr; 64 roundings of it a step
            assert np.abs(params[i].numpy() - p64[i]).max() < t * 64 * T.U32 * (0.1 + np.abs(p64[i]).max())
            gm, gv = opt.moments(i)
            if bits == 32:
                assert np.abs(gm - m[i]).max() <= 8 * t * T.U32 * 0.05 and np.abs(gv - v[i]).max() <= 8 * t * T.U32 * 0.0025
            else:
                # off by less than one code: (2 c + 1) / Q^2 of the block's scale, c / Q the value's root
                top = np.abs(gm).max() * 1.0001
                assert (np.abs(gm - m[i]) <= (2 * np.sqrt(np.abs(m[i]) / top) * 127 + 1) / 127 ** 2 * top).all()
                m[i], v[i] = gm.astype(np.float64), gv.astype(np.float64)
    assert [rsl._storage_ptr(p.data) for p in params] == buffers
    # a saved state goes on as the run itself does
    saved = opt.state_dict()
    twin_params = [rsl.Variable(p.numpy(), True) for p in params]
    twin = rsl.optim.AdamW(twin_params, lr=0.01, weight_decay=opt._decay[1], bits=bits, seed=1)
    twin._decay = list(opt._decay)
    twin.load_state_dict(saved)
    for o, ps in ((opt, params), (twin, twin_params)):
        o.zero_grad()
        (ps[0] * 0.5).sum(1).sum(0).backward()
        o.step()
    assert twin.steps == opt.steps == 6
    for a, b in zip(params, twin_params):
        assert np.array_equal(a.numpy(), b.numpy())
    with pytest.raises(ValueError, match="other parameters"):
        rsl.optim.AdamW(params[:2], bits=bits).load_state_dict(saved)
    with pytest.raises(ValueError, match="does not fit"):
        rsl.optim.AdamW([params[1], params[0], *params[2:]], bits=bits).load_state_dict(saved)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_training_step_equals_the_eager_one(rsl, bits):
    """Norm, attention, products and AdamW recorded while an eager graph of the same leaves is alive; replays, with eager
    work between them, equal eager steps bit for bit.  The plan and the optimizer's states live in the graph."""
    from rushlite_amd.nets import layers
    rng = np.random.default_rng(9)
    x_np, y_np = rng.standard_normal((40, 32)).astype(np.float32), rng.standard_normal((40, 32)).astype(np.float32)

    def build():
        rsl.manual_seed(4)
        norm, attention = layers.LayerNorm(32), layers.SelfAttention(32, 4, 2)
        params = list(norm.parameters()) + list(attention.parameters())
        return norm, attention, params, rsl.optim.AdamW(params, lr=1e-3, bits=bits, seed=2)

    def step(net, x, y, plan):
        norm, attention, _, opt = net
        opt.zero_grad()
        diff = attention(norm(x), plan) - y
        loss = (diff * diff).sum(1).sum(0)
        loss.backward()
        opt.step()
        return loss

    x, y = rsl.Variable(x_np), rsl.Variable(y_np)
    eager, kept = build(), build()
    plan = eager[1].plan([25, 15])
    want = [step(eager, x, y, plan).tolist()[0]]
    alive = step(kept, x, y, plan)  # its graph stays while the step is recorded
    got = [alive.tolist()[0]]
    graph = rsl.hip.Graph()
    with graph.capture():
        loss = step(kept, x, y, plan)
    for _ in range(5):
        want.append(step(eager, x, y, plan).tolist()[0])
        graph.replay()
        got.append(loss.tolist()[0])
        assert np.isfinite(alive.tolist()[0])
        for a, b in zip(eager[2], kept[2]):
            assert np.array_equal(a.numpy(), b.numpy())
    assert got == want
    assert kept[3].steps == eager[3].steps == 6
    # the plan's last Python holder goes; the graph still replays
    del plan
    step_again = eager[1].plan([25, 15])
    want = step(eager, x, y, step_again).tolist()[0]
    graph.replay()
    assert loss.tolist()[0] == want


@gpu
def test_example_trains_and_continues(rsl):
    sys.path.insert(0, str(ROOT / "examples"))
    import packed_transformer as example
    model, losses = example.train(steps=200, bits=8, report=lambda _: None)
    assert np.isfinite(losses).all()
    assert np.mean(losses[-20:]) < 0.35 * losses[0], (losses[0], np.mean(losses[-20:]))
    # token by token equals the whole prompt at once
    rng = np.random.default_rng(0)
    texts = [rng.integers(0, example.VOCAB, n) for n in (12, 5)]
    plan = model.block0.attention.plan([12, 5])
    with rsl.no_grad():
        probs = model(rsl.Variable(example.one_hot(np.concatenate(texts), example.VOCAB)),
                      rsl.Variable(example.one_hot(np.concatenate([np.arange(12), np.arange(5)]), model.positions)), plan).numpy()
    first = example.continue_prompts(model, texts, 1)
    for end, (token,) in zip((12, 17), first):
        top = np.sort(probs[end - 1])
        assert token == probs[end - 1].argmax() or top[-1] - top[-2] < 1e-4


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_takes_a_shared_parameter_once(rsl, bits):
    """A layer that hangs in a module twice: one state and one update for each of its parameters, bit for bit those of a
    list without repetitions."""
    from rushlite_amd.nets import layers
    x = np.random.default_rng(0).standard_normal((8, 300)).astype(np.float32)

    class Tied(rsl.Module):
        def __init__(self):
            super().__init__()
            rsl.manual_seed(3)
            self.first = layers.Linear(300, 300)
            self.again, self.norm, self.weights = self.first, layers.LayerNorm(300), self.first.weights

        def forward(self, x):
            return self.again(self.norm(self.first(x)))

    nets = [Tied(), Tied()]
    opts = [rsl.optim.AdamW(nets[0], lr=1e-2, bits=bits, seed=4),
            rsl.optim.AdamW([nets[1].first.weights, nets[1].first.bias, nets[1].norm.weights, nets[1].norm.bias], lr=1e-2,
                            bits=bits, seed=4)]
    assert len(list(nets[0].parameters())) == 7 and len(opts[0].params) == 4
    for _ in range(3):
        for net, opt in zip(nets, opts):
            opt.zero_grad()
            (net(rsl.Variable(x)) * 0.01).sum(1).sum(0).backward()
            opt.step()
        for a, b in zip(*(net.parameters() for net in nets)):
            assert np.array_equal(a.numpy(), b.numpy())


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_update_keeps_the_gradients_it_reads(rsl, bits):
    """Only the update is recorded, after an eager backward pass; the gradients go, their memory would be another tensor's.
    Every replay is the eager update by the same gradients."""
    rng = np.random.default_rng(6)
    p_np, g_np = rng.standard_normal((2, 300, 41)).astype(np.float32)

    def build():
        p = rsl.Variable(p_np, True)
        opt = rsl.optim.AdamW([p], lr=1e-2, bits=bits, seed=3)
        (p * rsl.Variable(g_np)).sum(1).sum(0).backward()
        return p, opt

    (eager, eager_opt), (kept, kept_opt) = build(), build()
    graph = rsl.hip.Graph()
    with graph.capture():
        kept_opt.step()
    assert kept_opt.steps == 0
    kept_opt.zero_grad()
    others = [rsl.Variable(np.full((300, 41), 1e6, np.float32)) for _ in range(8)]
    for i in range(4):
        graph.replay()
        eager_opt.step()
        assert np.array_equal(kept.numpy(), eager.numpy()), i
        others.append(rsl.Variable(np.full((300, 41), -1e6, np.float32)))
    assert kept_opt.steps == 4
    assert all((abs(o.numpy()) == 1e6).all() for o in others)


@gpu
def test_adamw_leaves_frozen_parameters_of_a_module(rsl):
    from rushlite_amd.nets import layers
    rsl.manual_seed(1)
    net = layers.SelfAttention(32, 2)
    net.qkv.weights = rsl.Variable(net.qkv.weights.data)
    frozen = net.qkv.weights.numpy().copy()
    opt = rsl.optim.AdamW(net, lr=0.1)
    assert len(opt.params) == 3 and all(p.requires_grad for p in opt.params)
    before = [p.numpy().copy() for p in opt.params]
    (net(rsl.Variable(np.random.default_rng(2).standard_normal((9, 32)).astype(np.float32)), net.plan([9])) * 0.1) \
        .sum(1).sum(0).backward()
    opt.step()
    opt.zero_grad()
    assert np.array_equal(net.qkv.weights.numpy(), frozen)
    assert all((p.numpy() != b).any() for p, b in zip(opt.params, before))
    with pytest.raises(ValueError, match="parameter 0 is not a Variable that requires a gradient"):
        rsl.optim.AdamW(list(net.parameters()))
