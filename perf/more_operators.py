"""The operators of a decoder's training step beside attention: what is timed, their plain forms, and the calls of the
framework's own kernels.

Operators
  rotary   pairs of each head's values turned by an angle, position times frequency; "train" also turns a gradient back
  dropout  y = residual + (kept ? x / (1 - rate) : 0), what is kept from a counter-based generator; "train" also dx
  gated    h = act(x Wg + bg) * (x Wu + bu); "train" also its gradients
  loss     softmax cross entropy of x W + b over a vocabulary; "train" also the gradients of the weighted sum of the losses

Where `own` is false, run() is the plain form in elementary torch operations; where it is true, run() calls the C ABI of
include/lmp_hip_transformer.h through rushlite_amd.abi, on the same tensors.  The library works on a stream of its own: the
inputs are complete when prepare() returns, and the library's calls are in order among themselves.

The random bits of dropout.  Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3",
2011): the seed's two halves are its key, and the counter is the place / 4 and the number of the call, low half first
each.  Value i takes word i % 4 and is kept if that is at least rate * 2^32.
"""
import functools
import math

import numpy as np
import torch

own = False

_DEV = "cuda"
_MASK32 = 0xFFFFFFFF
_CALLS0 = 70  # calls of the generator before the timed one
_GATES = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")
_TANH_SCALE, _TANH_CUBE = math.sqrt(2 / math.pi), 0.044715


def listed():
    return [
        # one new token for each of 32 requests, its queries and keys side by side: latency alone
        dict(name="rotary_token", op="rotary", pass_="forward", dtype="f32", rows=32, heads=40, plain_heads=8, dim=128,
             rotary_dim=128, interleaved=False, longest=8192, base=10000.0, factor=1.0),
        # a packed batch of documents, queries, keys and values three slices of one projection: a training step
        dict(name="rotary_packed", op="rotary", pass_="train", dtype="f32", rows=8192, heads=20, plain_heads=4, dim=64,
             rotary_dim=64, interleaved=False, longest=2048, base=10000.0, factor=1.0),
        # one long document in float64, neighbouring pairs, half of each head, frequencies scaled for a longer context
        dict(name="rotary_long_f64", op="rotary", pass_="train", dtype="f64", rows=16384, heads=16, plain_heads=0, dim=128,
             rotary_dim=64, interleaved=True, longest=16384, base=500000.0, factor=8.0),
        # the hidden activations of the README's net: latency alone
        dict(name="dropout_small", op="dropout", pass_="forward", dtype="f32", rows=32, cols=256, residual=False, rate=0.1),
        # a long batch of wide activations added to its residual stream, forward and backward: bound by memory
        dict(name="dropout_wide", op="dropout", pass_="train", dtype="f32", rows=8192, cols=8192, residual=True, rate=0.1),
        # one new token for each of 32 requests through a wide layer: bound by reading the weights
        dict(name="gated_token", op="gated", pass_="forward", gate="silu", rows=32, inp=4096, hidden=8192, bias=False),
        # 64 sequences of 197 positions of width 768, the hidden layer 8/3 as wide: a training step
        dict(name="gated_train", op="gated", pass_="train", gate="silu", rows=64 * 197, inp=768, hidden=2048, bias=False),
        # rows and columns of odd lengths, none of them aligned, biases, another gate
        dict(name="gated_ragged", op="gated", pass_="train", gate="gelu_tanh", rows=1000, inp=2047, hidden=1531, bias=True),
        # the README's net's last layer: latency alone
        dict(name="loss_small", op="loss", pass_="train", rows=32, inp=64, vocab=10, bias=True, ignored=0.0),
        # a packed batch over a large vocabulary: a training step
        dict(name="loss_train", op="loss", pass_="train", rows=4096, inp=1024, vocab=32768, bias=False, ignored=0.1),
        # odd sizes, a bias, a third of the positions not counted
        dict(name="loss_ragged", op="loss", pass_="train", rows=1013, inp=768, vocab=10001, bias=True, ignored=0.33),
        # scoring a long batch: the losses alone
        dict(name="loss_score", op="loss", pass_="forward", rows=8192, inp=1024, vocab=32768, bias=False, ignored=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, step=64):
    """Log-uniform in [lo, hi]; half of them multiples of `step`, the rest whatever comes."""
    v = _log(rng, lo, hi)
    if v >= step and rng.random() < 0.5:
        v = v // step * step
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "dropout", "gated", "gated", "loss", "loss"])
    if op == "rotary":
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        c = dict(op=op, pass_=rng.choice(["forward", "train"]), dtype=rng.choice(["f32", "f32", "f32", "f64"]),
                 heads=_size(rng, 1, 48), plain_heads=rng.choice([0, 0, 1, 4, 8]), dim=dim,
                 rotary_dim=rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.4,
                 base=rng.choice([10000.0, 500000.0]), factor=rng.choice([1.0, 1.0, 4.0, 8.0]))
        most = max(2, min(65536, (1 << 25) // ((c["heads"] + c["plain_heads"]) * dim)))
        c["rows"] = _size(rng, 1, most)
        c["longest"] = _size(rng, 1, 131072)
        return c
    if op == "dropout":
        cols = _size(rng, 16, 16384)
        return dict(op=op, pass_=rng.choice(["forward", "train"]), dtype=rng.choice(["f32", "f32", "f32", "f64"]),
                    rows=_size(rng, 1, max(2, min(65536, (1 << 25) // cols))), cols=cols, residual=rng.random() < 0.5,
                    rate=rng.choice([0.05, 0.1, 0.1, 0.2, 0.5]))
    if op == "gated":
        inp, hidden = _size(rng, 16, 4096), _size(rng, 16, 8192)
        most = max(2, min(16384, (1 << 36) // (inp * hidden)))
        return dict(op=op, pass_=rng.choice(["forward", "train", "train"]),
                    gate=rng.choice(["silu", "silu", "gelu", "gelu_tanh", "sigmoid"]), rows=_size(rng, 1, most), inp=inp,
                    hidden=hidden, bias=rng.random() < 0.4)
    inp, vocab = _size(rng, 16, 2048), _size(rng, 2, 65536)
    most = max(2, min(16384, (1 << 37) // (inp * vocab), (1 << 28) // vocab))
    return dict(op=op, pass_=rng.choice(["forward", "train", "train"]), rows=_size(rng, 1, most), inp=inp, vocab=vocab,
                bias=rng.random() < 0.4, ignored=rng.choice([0.0, 0.1, 0.5]))


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) * 7919 + 31)
    return g


def _randn(g, shape, scale=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=_DEV, dtype=dtype) * scale


def _frequencies(c):
    """(radians per position of each pair, the factor on the rotated values).  With `factor` above 1, pairs that turn less
    than once over 4096 positions are slowed down by it, those that turn over 32 times are not, others in between."""
    n = c["rotary_dim"]
    f = [c["base"] ** (-2.0 * j / n) for j in range(n // 2)]
    if c["factor"] == 1.0:
        return f, 1.0
    keep = [min(1.0, max(0.0, (4096 * x / (2 * math.pi) - 1) / 31)) for x in f]
    return [x * k + x / c["factor"] * (1 - k) for x, k in zip(f, keep)], 0.1 * math.log(c["factor"]) + 1


def prepare(case, seed):
    c, g, op = case, _gen(seed), case["op"]
    s = dict(op=op, case=c)
    t = torch.float64 if c.get("dtype") == "f64" else torch.float32
    train = c["pass_"] == "train"
    if op == "rotary":
        n = (c["heads"] + c["plain_heads"]) * c["dim"]
        f, scale = _frequencies(c)
        # documents one after another, from somewhere in the first to the end of the last
        first = int(seed) * 7919 % c["longest"]
        s.update(x=_randn(g, (c["rows"], n), 1.0, t), scale=scale,
                 frequencies=torch.tensor(f, dtype=torch.float64, device=_DEV),
                 positions=(torch.arange(c["rows"], device=_DEV) + first) % c["longest"])
        s.update(y=torch.empty_like(s["x"]))
        if train:
            s.update(g=_randn(g, (c["rows"], n), 0.1, t), dx=torch.empty_like(s["x"]))
    elif op == "dropout":
        shape = (c["rows"], c["cols"])
        s.update(x=_randn(g, shape, 1.0, t), residual=_randn(g, shape, 1.0, t) if c["residual"] else None,
                 y=torch.empty(shape, dtype=t, device=_DEV), seed=int(seed) * 0x9E3779B97F4A7C15 % (1 << 64),
                 calls=torch.tensor([_CALLS0, 0], dtype=torch.int64, device=_DEV),
                 used=torch.zeros(1, dtype=torch.int64, device=_DEV))
        if train:
            s.update(g=_randn(g, shape, 0.1, t), dx=torch.empty(shape, dtype=t, device=_DEV))
    elif op == "gated":
        n, d, h = c["rows"], c["inp"], c["hidden"]
        s.update(x=_randn(g, (n, d)), w=_randn(g, (d, 2 * h), d ** -0.5), b=_randn(g, (2 * h,), 0.1) if c["bias"] else None,
                 h=torch.empty(n, h, device=_DEV))
        if train:
            s.update(g=_randn(g, (n, h), 0.1), pre=torch.empty(n, 2 * h, device=_DEV), dx=torch.empty(n, d, device=_DEV),
                     dw=torch.empty(d, 2 * h, device=_DEV), db=torch.empty(2 * h, device=_DEV) if c["bias"] else None)
    else:
        n, d, v = c["rows"], c["inp"], c["vocab"]
        # logits of a deviation of 2; frequent tokens and rare ones
        u = torch.rand(n, generator=g, device=_DEV)
        targets = (v * u ** 3).to(torch.int64).clamp(max=v - 1)
        out = torch.rand(n, generator=g, device=_DEV) < c["ignored"]
        s.update(x=_randn(g, (n, d)), w=_randn(g, (d, v), 2 * d ** -0.5), b=_randn(g, (v,), 0.5) if c["bias"] else None,
                 targets=torch.where(out, torch.full_like(targets, -1), targets), loss=torch.empty(n, device=_DEV),
                 weights=(~out).to(torch.float32) / (~out).sum().clamp(min=1))
        if train:
            s.update(dx=torch.empty(n, d, device=_DEV), dw=torch.empty(d, v, device=_DEV),
                     db=torch.empty(v, device=_DEV) if c["bias"] else None)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------- plain forms

def _turned(s, x, sign):
    c = s["case"]
    n, r, rows = c["heads"] * c["dim"], c["rotary_dim"], c["rows"]
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos = (torch.cos(angle) * s["scale"]).to(x.dtype)[:, None, :]
    sin = (torch.sin(angle) * (s["scale"] * sign)).to(x.dtype)[:, None, :]
    v = x[:, :n].reshape(rows, c["heads"], c["dim"])
    u, w = (v[:, :, 0:r:2], v[:, :, 1:r:2]) if c["interleaved"] else (v[:, :, :r // 2], v[:, :, r // 2:r])
    a, b = u * cos - w * sin, w * cos + u * sin
    turned = torch.stack((a, b), 3).reshape(rows, c["heads"], r) if c["interleaved"] else torch.cat((a, b), 2)
    return torch.cat((torch.cat((turned, v[:, :, r:]), 2).reshape(rows, n), x[:, n:]), 1)


def _rotary_plain(s):
    y = _turned(s, s["x"], 1)
    return dict(y=y, dx=_turned(s, s["g"], -1)) if s["case"]["pass_"] == "train" else dict(y=y)


def _round(c, k):
    p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # bits past 63 are the sign's: the masks keep what is meant
    return ((q >> 32) & _MASK32) ^ c[1] ^ k[0], q & _MASK32, ((p >> 32) & _MASK32) ^ c[3] ^ k[1], p & _MASK32


def _kept(s, call):
    n, seed = s["x"].numel(), s["seed"]
    place = torch.arange(-(-n // 4), device=_DEV)
    each = lambda v: torch.zeros_like(place) + v  # noqa: E731
    c = (place & _MASK32, place >> 32, each(call & _MASK32), each(call >> 32))
    keys = [((seed + i * 0x9E3779B9) & _MASK32, ((seed >> 32) + i * 0xBB67AE85) & _MASK32) for i in range(10)]
    bits = torch.stack(functools.reduce(_round, keys, c), 1).reshape(-1)[:n]
    return (bits >= int(round(s["case"]["rate"] * 2 ** 32))).reshape(s["x"].shape)


def _dropout_plain(s):
    c, scale = s["case"], 1 / (1 - s["case"]["rate"])
    kept = _kept(s, s["calls"][0])
    y = torch.where(kept, s["x"] * scale, torch.zeros_like(s["x"]))
    if c["residual"]:
        y = s["residual"] + y
    s["calls"][0] += 1
    if c["pass_"] == "forward":
        return dict(y=y)
    return dict(y=y, dx=torch.where(kept, s["g"] * scale, torch.zeros_like(y)))


def _act_plain(gate, a):
    """(act(a), act'(a))"""
    if gate == "gelu":
        # through the complement, which keeps the digits of small values
        share = 0.5 * torch.special.erfc(a * -math.sqrt(0.5))
        return a * share, share + a * torch.exp(a * a * -0.5) * (1 / math.sqrt(2 * math.pi))
    v = a * (2 * _TANH_SCALE) * (1 + _TANH_CUBE * a * a) if gate == "gelu_tanh" else a
    share, rest = 1 / (1 + torch.exp(-v)), 1 / (1 + torch.exp(v))
    if gate == "sigmoid":
        return share, share * rest
    slope = 2 * _TANH_SCALE * (1 + 3 * _TANH_CUBE * a * a) if gate == "gelu_tanh" else 1
    return a * share, share + a * share * rest * slope


def _gated_plain(s):
    h = s["case"]["hidden"]
    pre = torch.matmul(s["x"], s["w"])
    if s["b"] is not None:
        pre = pre + s["b"]
    act, slope = _act_plain(s["case"]["gate"], pre[:, :h])
    out = dict(h=act * pre[:, h:])
    if s["case"]["pass_"] == "forward":
        return out
    d = torch.cat((s["g"] * pre[:, h:] * slope, s["g"] * act), 1)
    out.update(dx=torch.matmul(d, s["w"].t()), dw=torch.matmul(s["x"].t(), d))
    return dict(out, db=d.sum(0)) if s["b"] is not None else out


def _loss_plain(s):
    z = torch.matmul(s["x"], s["w"])
    if s["b"] is not None:
        z = z + s["b"]
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    counted, place = s["targets"] >= 0, s["targets"].clamp(min=0)[:, None]
    # the two differences apart: their sum keeps the digits of a small loss
    loss = torch.where(counted, (torch.log(total) - (z.gather(1, place) - top))[:, 0], torch.zeros_like(s["loss"]))
    if s["case"]["pass_"] == "forward":
        return dict(loss=loss)
    w = torch.where(counted, s["weights"], torch.zeros_like(loss))[:, None]
    d = e * (w / total)
    d.scatter_add_(1, place, -w)
    out = dict(loss=loss, dx=torch.matmul(d, s["w"].t()), dw=torch.matmul(s["x"].t(), d))
    return dict(out, db=d.sum(0)) if s["b"] is not None else out


# ------------------------------------------------- the framework's kernels

def _ptr(t):
    return None if t is None else t.data_ptr()


def _code(abi, s):
    return abi.FLOAT64 if s["case"]["dtype"] == "f64" else abi.FLOAT32


def _rotary_own(s):
    from rushlite_amd import abi
    lib, c, n = abi.lib(), s["case"], s["x"].shape[1]

    def turn(x, inverse, y):
        abi.check(lib.lmp_k_rotary(_code(abi, s), c["rows"], n, c["heads"], c["dim"], c["rotary_dim"],
                                   int(c["interleaved"]), x.data_ptr(), n, s["positions"].data_ptr(),
                                   s["frequencies"].data_ptr(), s["scale"], inverse, y.data_ptr(), n))

    turn(s["x"], 0, s["y"])
    if c["pass_"] == "forward":
        return dict(y=s["y"])
    turn(s["g"], 1, s["dx"])
    return dict(y=s["y"], dx=s["dx"])


def _dropout_own(s):
    from rushlite_amd import abi
    lib, c, n = abi.lib(), s["case"], s["x"].numel()
    abi.check(lib.lmp_k_dropout(_code(abi, s), n, s["x"].data_ptr(), _ptr(s["residual"]), c["rate"], s["seed"],
                                s["calls"].data_ptr(), s["used"].data_ptr(), s["y"].data_ptr()))
    if c["pass_"] == "forward":
        return dict(y=s["y"])
    abi.check(lib.lmp_k_dropout_backward(_code(abi, s), n, s["g"].data_ptr(), c["rate"], s["seed"], s["used"].data_ptr(),
                                         s["dx"].data_ptr()))
    return dict(y=s["y"], dx=s["dx"])


def _gated_own(s):
    from rushlite_amd import abi
    lib, c, gate = abi.lib(), s["case"], _GATES.index(s["case"]["gate"])
    n, d, h, train = c["rows"], c["inp"], c["hidden"], c["pass_"] == "train"
    x, w = s["x"].data_ptr(), s["w"].data_ptr()
    pre = s["pre"].data_ptr() if train else None
    abi.check(lib.lmp_k_gated_linear_f32(gate, n, d, h, x, d, w, 2 * h, _ptr(s["b"]), s["h"].data_ptr(), h, pre, 2 * h))
    if not train:
        return dict(h=s["h"])
    abi.check(lib.lmp_k_gated_linear_backward_f32(gate, n, d, h, s["g"].data_ptr(), h, x, d, w, 2 * h, pre, 2 * h,
                                                  s["dx"].data_ptr(), d, s["dw"].data_ptr(), 2 * h, _ptr(s["db"])))
    out = dict(h=s["h"], dx=s["dx"], dw=s["dw"])
    return dict(out, db=s["db"]) if s["b"] is not None else out


def _loss_own(s):
    from rushlite_amd import abi
    lib, c = abi.lib(), s["case"]
    n, d, v = c["rows"], c["inp"], c["vocab"]
    x, w, b, t, loss = s["x"].data_ptr(), s["w"].data_ptr(), _ptr(s["b"]), s["targets"].data_ptr(), s["loss"].data_ptr()
    if c["pass_"] == "forward":
        abi.check(lib.lmp_k_linear_cross_entropy_f32(n, d, v, x, d, w, v, b, t, loss))
        return dict(loss=s["loss"])
    abi.check(lib.lmp_k_linear_cross_entropy_grad_f32(n, d, v, x, d, w, v, b, t, s["weights"].data_ptr(), loss,
                                                      s["dx"].data_ptr(), d, s["dw"].data_ptr(), v, _ptr(s["db"])))
    out = dict(loss=s["loss"], dx=s["dx"], dw=s["dw"])
    return dict(out, db=s["db"]) if s["b"] is not None else out


def run(state):
    op = state["op"]
    if own:
        return dict(rotary=_rotary_own, dropout=_dropout_own, gated=_gated_own, loss=_loss_own)[op](state)
    return dict(rotary=_rotary_plain, dropout=_dropout_plain, gated=_gated_plain, loss=_loss_plain)[op](state)


# ------------------------------------------------------------ work and truth

def work(case):
    c = case
    train = c["pass_"] == "train"
    size = 8 if c.get("dtype") == "f64" else 4
    if c["op"] == "rotary":
        n, turned = c["rows"] * (c["heads"] + c["plain_heads"]) * c["dim"], c["rows"] * c["heads"] * c["rotary_dim"]
        return dict(bytes=(2 * size * n + 8 * c["rows"]) * (1 + train) + 4 * c["rotary_dim"], flops=3 * turned * (1 + train))
    if c["op"] == "dropout":
        n = c["rows"] * c["cols"]
        return dict(bytes=size * n * (2 + c["residual"] + 2 * train), flops=n * (1 + c["residual"] + train))
    if c["op"] == "gated":
        n, d, h = c["rows"], c["inp"], c["hidden"]
        forward = n * d + 2 * d * h + n * h + 2 * h * c["bias"]
        return dict(bytes=4 * (forward + train * (n * h + n * d + 2 * d * h + 2 * h * c["bias"])),
                    flops=4 * n * d * h * (3 if train else 1) + 10 * n * h)
    n, d, v = c["rows"], c["inp"], c["vocab"]
    forward = n * d + d * v + v * c["bias"] + 3 * n
    return dict(bytes=4 * (forward + train * (n * d + d * v + v * c["bias"] + n)),
                flops=2 * n * d * v * (3 if train else 1) + 5 * n * v)


def _rotary_exact(s):
    c = s["case"]
    rows, heads, d, r = c["rows"], c["heads"], c["dim"], c["rotary_dim"]
    # each pair a complex number, times scale e^(i angle)
    turn = torch.polar(torch.full((rows, r // 2), float(s["scale"]), dtype=torch.float64, device=_DEV),
                       s["positions"][:, None].double() * s["frequencies"][None])[:, None]

    def by(x, factor):
        out = x.double().clone()
        part = out[:, :heads * d].view(rows, heads, d)[:, :, :r]
        if c["interleaved"]:
            pairs = torch.view_as_complex(part.reshape(rows, heads, r // 2, 2).contiguous()) * factor
            part.copy_(torch.view_as_real(pairs).reshape(rows, heads, r))
        else:
            pairs = torch.complex(part[:, :, :r // 2].contiguous(), part[:, :, r // 2:].contiguous()) * factor
            part[:, :, :r // 2], part[:, :, r // 2:] = pairs.real, pairs.imag
        return out

    if c["pass_"] == "forward":
        return dict(y=by(s["x"], turn))
    return dict(y=by(s["x"], turn), dx=by(s["g"], turn.conj()))


def _dropout_exact(s):
    c, n, seed = s["case"], s["x"].numel(), s["seed"]
    low = np.uint64(_MASK32)
    ctr = np.zeros((4, -(-n // 4)), np.uint64)
    place = np.arange(ctr.shape[1], dtype=np.uint64)
    ctr[0], ctr[1], ctr[2] = place & low, place >> np.uint64(32), _CALLS0
    k0, k1 = seed & _MASK32, seed >> 32
    for _ in range(10):
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr[0], ctr[2] = (b >> np.uint64(32)) ^ ctr[1] ^ np.uint64(k0), (a >> np.uint64(32)) ^ ctr[3] ^ np.uint64(k1)
        ctr[1], ctr[3] = b & low, a & low
        k0, k1 = (k0 + 0x9E3779B9) & _MASK32, (k1 + 0xBB67AE85) & _MASK32
    words = ctr.T.reshape(-1)[:n].astype(np.int64)
    factor = torch.from_numpy(words >= round(c["rate"] * 4294967296.0)).to(_DEV).double().view(s["x"].shape) / (1 - c["rate"])
    y = s["x"].double() * factor
    if c["residual"]:
        y = y + s["residual"].double()
    return dict(y=y) if c["pass_"] == "forward" else dict(y=y, dx=s["g"].double() * factor)


def _gated_exact(s):
    c = s["case"]
    x, w = s["x"].double(), s["w"].double()
    b = torch.zeros(w.shape[1], dtype=torch.float64, device=_DEV) if s["b"] is None else s["b"].double()
    a, u = torch.addmm(b, x, w).chunk(2, 1)
    if c["gate"] == "gelu":
        cdf = torch.special.ndtr(a)
        act, slope = a * cdf, cdf + a * torch.exp(-a ** 2 / 2) / math.sqrt(2 * math.pi)
    elif c["gate"] == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3))
        act = a / 2 * (1 + t)
        slope = (1 + t) / 2 + a / 2 * (1 - t ** 2) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * a ** 2)
    else:
        sig = torch.sigmoid(a)
        act, slope = (sig, sig - sig ** 2) if c["gate"] == "sigmoid" else (a * sig, sig + a * sig * (1 - sig))
    out = dict(h=act * u)
    if c["pass_"] == "forward":
        return out
    g = s["g"].double()
    da, du = g * u * slope, g * act
    out["dx"] = da @ w[:, :c["hidden"]].t() + du @ w[:, c["hidden"]:].t()
    out["dw"] = torch.cat((x.t() @ da, x.t() @ du), 1)
    if s["b"] is not None:
        out["db"] = torch.cat((da.sum(0), du.sum(0)))
    return out


def _loss_exact(s):
    c = s["case"]
    x, w = s["x"].double(), s["w"].double()
    logits = x @ w if s["b"] is None else torch.addmm(s["b"].double(), x, w)
    logp = logits - torch.logsumexp(logits, 1, keepdim=True)
    del logits
    rows = torch.nonzero(s["targets"] >= 0)[:, 0]
    loss = torch.zeros(c["rows"], dtype=torch.float64, device=_DEV)
    loss[rows] = -logp[rows, s["targets"][rows]]
    if c["pass_"] == "forward":
        return dict(loss=loss)
    d = logp.exp_()
    d[rows, s["targets"][rows]] -= 1
    weight = torch.zeros_like(loss)
    weight[rows] = s["weights"][rows].double()
    d *= weight[:, None]
    out = dict(loss=loss, dx=d @ w.t(), dw=x.t() @ d)
    return dict(out, db=d.sum(0)) if s["b"] is not None else out


def exact(case, seed):
    s = prepare(case, seed)
    return dict(rotary=_rotary_exact, dropout=_dropout_exact, gated=_gated_exact, loss=_loss_exact)[s["op"]](s)
