"""The transformer-training operators: what is timed, their plain forms, and the calls of the framework's own kernels.

Operators
  layer_norm   y = (x - mean) / sqrt(var + eps) * w + b over the last axis; "train" also its three gradients
  adamw        one AdamW step over every parameter of a model, its states in 32 or in 8 bits
  attention    softmax(scale q k^T + causal mask) v over packed sequences, grouped heads; "train" also dq, dk and dv

Where `own` is false, run() is the plain form in elementary torch operations; where it is true, run() calls the C ABI
of include/lmp_hip.h through rushlite_amd.abi, on the same tensors.  The library works on a stream of its own: the
inputs are complete when prepare() returns, and the library's calls are in order among themselves.

The AdamW states in 8 bits.  Per block of 256 values of one tensor: the largest magnitude M in float32, and a code c of
one byte per value that stands for sign(c) (|c| / Q)^2 M, with Q = 127 for the first moment and 255 for the second.
Codes are rounded up or down at random so that their expectation is the value; the 16 random bits of each come from
MurmurHash3's 32-bit finalizer over (seed, step, tensor, place).  A second moment above zero never rounds to zero.
Codes returned by run() are returned as the values they stand for.
"""
import math

import torch

own = False

_DEV = "cuda"
_BLOCK = 256
_EPS = 1e-5
_HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, decay=1e-2)
_STEP0 = 100  # steps done before the timed one
_MASK32 = 0xFFFFFFFF


def listed():
    return [
        # the hidden activations of the README's net, normalised: latency alone
        dict(name="norm_small", op="layer_norm", pass_="forward", dtype="f32", rows=32, cols=256),
        # a long batch of wide activations, as an inference pass normalises it: bound by memory
        dict(name="norm_wide", op="layer_norm", pass_="forward", dtype="f32", rows=8192, cols=8192),
        # 64 sequences of 197 positions of width 768: forward and backward of a training step
        dict(name="norm_train", op="layer_norm", pass_="train", dtype="f32", rows=64 * 197, cols=768),
        # rows of an odd length, none of them aligned
        dict(name="norm_train_ragged", op="layer_norm", pass_="train", dtype="f32", rows=4095, cols=3001),
        # float64, numpy's own type
        dict(name="norm_train_f64", op="layer_norm", pass_="train", dtype="f64", rows=4096, cols=1024),
        # the README's net: four tensors, 17 thousand parameters, latency alone
        dict(name="adamw_readme", op="adamw", bits=32, layers=1, inp=256, hidden=64, out=10, norms=False),
        # the wide net of bench.py, 37.7 million parameters: bound by memory
        dict(name="adamw_wide", op="adamw", bits=32, layers=2, inp=4096, hidden=4096, out=1000, norms=False),
        # the same net with its states in 8 bits
        dict(name="adamw_wide_8bit", op="adamw", bits=8, layers=2, inp=4096, hidden=4096, out=1000, norms=False),
        # one short prompt of few heads: latency alone
        dict(name="attention_small", op="attention", pass_="forward", kind="prompt", sequences=1, longest=32, keys=32,
             heads=4, kv_heads=4, dim=64, causal=True, fused=False),
        # a packed batch of ragged documents, grouped heads, q, k and v three slices of one projection: a training step
        dict(name="attention_packed", op="attention", pass_="train", kind="prompt", sequences=8, longest=2048, keys=2048,
             heads=16, kv_heads=4, dim=64, causal=True, fused=True),
        # one long document: forward and backward, bound by the matrix cores
        dict(name="attention_long", op="attention", pass_="train", kind="prompt", sequences=1, longest=8192, keys=8192,
             heads=16, kv_heads=4, dim=128, causal=True, fused=False),
        # one new token for each of 32 requests against keys of up to 8192 positions: bound by reading the keys
        dict(name="attention_token", op="attention", pass_="forward", kind="token", sequences=32, longest=1, keys=8192,
             heads=32, kv_heads=8, dim=128, causal=True, fused=False),
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
    op = rng.choice(["layer_norm", "layer_norm", "adamw", "adamw", "attention", "attention", "attention"])
    if op == "layer_norm":
        cols = _size(rng, 16, 16384)
        return dict(op=op, pass_=rng.choice(["forward", "train"]), dtype=rng.choice(["f32", "f32", "f32", "f64"]),
                    rows=_size(rng, 1, max(2, min(65536, (1 << 25) // cols))), cols=cols)
    if op == "adamw":
        return dict(op=op, bits=rng.choice([8, 32]), layers=rng.choice([1, 2, 3, 4, 6]), inp=_size(rng, 16, 2048),
                    hidden=_size(rng, 16, 2048), out=_size(rng, 2, 1000), norms=rng.random() < 0.5)
    kind = rng.choice(["prompt", "prompt", "prompt", "chunk", "token"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    c = dict(op=op, pass_=rng.choice(["forward", "train"]) if kind == "prompt" else "forward", kind=kind,
             sequences=_size(rng, 1, 16 if kind != "token" else 64, 8), longest=1, keys=1, heads=heads, kv_heads=kv_heads,
             dim=rng.choice([32, 64, 64, 80, 96, 128, 128]), causal=rng.random() < 0.85, fused=False)
    if kind == "prompt":
        c["longest"] = c["keys"] = _size(rng, 1, 4096)
        c["fused"] = rng.random() < 0.5
    else:
        c["keys"] = _size(rng, 2, 16384)
        if kind == "chunk":
            c["longest"] = _size(rng, 2, min(512, c["keys"]))
    while c["sequences"] > 1 and c["sequences"] * c["heads"] * c["longest"] * c["keys"] > 1 << 29:
        c["sequences"] //= 2
    return c


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _randn(g, shape, scale=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=_DEV, dtype=dtype) * scale


def _shapes(c):
    """The parameters of a net: weights, biases and, with `norms`, a layer norm's pair behind each hidden layer."""
    dims = [c["inp"]] + [c["hidden"]] * c["layers"] + [c["out"]]
    got = []
    for i, (a, b) in enumerate(zip(dims, dims[1:])):
        got += [(a, b), (b,)]
        if c["norms"] and i < c["layers"]:
            got += [(b,), (b,)]
    return got


def _lengths(c):
    """(query lengths, key lengths) of the case's sequences: spread over [1, longest], the first of them the longest."""
    golden = 0.6180339887498949
    part = [1.0] + [(i * golden) % 1.0 for i in range(1, c["sequences"])]
    if c["kind"] == "prompt":
        q = [max(1, int(c["longest"] * f)) for f in part]
        return q, q
    k = [max(1, int(c["keys"] * f)) for f in part]
    return [min(c["longest"], n) for n in k], k


def prepare(case, seed):
    c, g, op = case, _gen(seed), case["op"]
    s = dict(op=op, case=c)
    if op == "layer_norm":
        t = torch.float64 if c["dtype"] == "f64" else torch.float32
        n = c["cols"]
        # activations with an offset, as a residual stream has
        s.update(x=_randn(g, (c["rows"], n), 1.0, t) + 0.5, w=1 + _randn(g, (n,), 0.1, t), b=_randn(g, (n,), 0.1, t),
                 g=_randn(g, (c["rows"], n), 0.1, t))
        s.update(y=torch.empty_like(s["x"]), mean=torch.empty(c["rows"], dtype=t, device=_DEV),
                 rstd=torch.empty(c["rows"], dtype=t, device=_DEV))
        if c["pass_"] == "train":
            s.update(dx=torch.empty_like(s["x"]), dw=torch.empty_like(s["w"]), db=torch.empty_like(s["b"]))
    elif op == "adamw":
        # one arena for all parameters, each tensor at a multiple of a block
        at, spans = 0, []
        for shape in _shapes(c):
            n = math.prod(shape)
            spans.append((at, n))
            at += -(-n // _BLOCK) * _BLOCK
        keep = torch.zeros(at, device=_DEV)
        for a, n in spans:
            keep[a:a + n] = 1
        m = _randn(g, (at,), 1e-3) * keep
        v = (_randn(g, (at,), 1e-3).square() + 1e-8) * keep
        s.update(spans=spans, seed=int(seed), p=_randn(g, (at,), 0.02) * keep, g=_randn(g, (at,), 2e-3) * keep,
                 step=torch.tensor([_STEP0, 0], dtype=torch.int64, device=_DEV))
        if c["bits"] == 32:
            s.update(m=m, v=v)
        else:
            ms, vs = m.reshape(-1, _BLOCK).abs().amax(1), v.reshape(-1, _BLOCK).amax(1)
            mc = (m.reshape(-1, _BLOCK).abs() / ms[:, None]).sqrt() * 127
            vc = (v.reshape(-1, _BLOCK) / vs[:, None]).sqrt() * 255
            s.update(mc=(mc.round() * m.reshape(-1, _BLOCK).sign()).to(torch.int8).reshape(-1), ms=ms,
                     vc=vc.round().to(torch.uint8).reshape(-1), vs=vs, m=torch.empty_like(m), v=torch.empty_like(v))
    else:
        ql, kl = _lengths(c)
        h, kv, d = c["heads"], c["kv_heads"], c["dim"]
        tq, tk = sum(ql), sum(kl)
        if c["fused"]:
            rows = _randn(g, (tq, (h + 2 * kv) * d))
            s.update(q=rows[:, :h * d], k=rows[:, h * d:(h + kv) * d], v=rows[:, (h + kv) * d:])
        else:
            s.update(q=_randn(g, (tq, h * d)), k=_randn(g, (tk, kv * d)), v=_randn(g, (tk, kv * d)))
        s.update(scale=d ** -0.5, o=torch.empty(tq, h * d, device=_DEV), lse=torch.empty(tq, h, device=_DEV))
        if c["pass_"] == "train":
            s.update(g=_randn(g, (tq, h * d), 0.1), dq=torch.empty(tq, h * d, device=_DEV),
                     dk=torch.empty(tk, kv * d, device=_DEV), dv=torch.empty(tk, kv * d, device=_DEV))
        # what a data loader hands over with a packed batch: each token's sequence and place
        lens = lambda v: torch.tensor(v, device=_DEV)  # noqa: E731
        seq = lambda v: torch.repeat_interleave(torch.arange(len(v), device=_DEV), lens(v))  # noqa: E731
        s.update(ql=lens(ql), kl=lens(kl), qseq=seq(ql), kseq=seq(kl), most=(max(ql), max(kl)))
        s.update(qpos=torch.arange(tq, device=_DEV) - (lens(ql).cumsum(0) - lens(ql))[s["qseq"]],
                 kpos=torch.arange(tk, device=_DEV) - (lens(kl).cumsum(0) - lens(kl))[s["kseq"]])
        if own:
            from rushlite_amd import abi
            s["plan"] = abi.AttentionPlan(ql, kl, heads=h, kv_heads=kv, head_dim=d, causal=c["causal"])
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------- plain forms

def _norm_plain(s):
    x, n = s["x"], s["x"].shape[1]
    mean = x.sum(1, keepdim=True) / n
    xc = x - mean
    rstd = 1 / torch.sqrt((xc * xc).sum(1, keepdim=True) / n + _EPS)
    xh = xc * rstd
    y = xh * s["w"] + s["b"]
    if s["case"]["pass_"] == "forward":
        return dict(y=y, mean=mean[:, 0], rstd=rstd[:, 0])
    g = s["g"]
    gw = g * s["w"]
    dx = rstd * (gw - gw.sum(1, keepdim=True) / n - xh * ((gw * xh).sum(1, keepdim=True) / n))
    return dict(y=y, dx=dx, dw=(g * xh).sum(0), db=g.sum(0))


def _fmix32(x):
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & _MASK32
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & _MASK32
    return x ^ (x >> 16)


def _random_bits(n, tensor, step, seed):
    """32 random bits per place, of which the first moment takes the low 16 and the second the high 16."""
    key = _fmix32((step ^ (seed & _MASK32)) & _MASK32)
    key = _fmix32((key + 0x9E3779B9 * (tensor + 1)) & _MASK32)
    place = torch.arange(n, device=_DEV)
    return _fmix32((place & _MASK32) ^ key ^ ((place >> 32) * 0x85EBCA6B & _MASK32))


def _encode(x, q, bits):
    """(codes, scales) of blocks [k, 256] of float32 values; q 127 with signs or 255 without."""
    top = x.abs().amax(1)
    live = (top >= 1e-30) & (top < math.inf)
    scale = torch.where(live, top, torch.where(top < 1e-30, torch.zeros_like(top), torch.full_like(top, math.nan)))
    inv = torch.where(live, float(q * q) / torch.where(live, top, torch.ones_like(top)), torch.zeros_like(top))
    t = torch.where(live[:, None], x.abs() * inv[:, None], torch.zeros_like(x)).clamp(max=float(q * q))
    c = t.sqrt().floor()
    c = torch.where(c * c > t, c - 1, c)
    c = torch.where((c + 1) * (c + 1) <= t, c + 1, c)
    u = bits.reshape(x.shape).to(torch.float32) * (1.0 / 65536)
    c = torch.where(u * (2 * c + 1) < t - c * c, c + 1, c)
    if q == 255:
        c = torch.where((c == 0) & (t > 0), torch.ones_like(c), c)
    return torch.where(x < 0, -c, c).clamp(-q, q), scale


def _decode(codes, scales, q):
    c = codes.reshape(-1, _BLOCK).to(torch.float32)
    return (c * c.abs()) * (scales * (1.0 / (q * q)))[:, None]


def _adamw_plain(s):
    h, bits = _HYPER, s["case"]["bits"]
    t = s["step"][0] + 1
    t64 = t.double()
    size = (h["lr"] / (1 - torch.pow(torch.tensor(h["beta1"], dtype=torch.float64, device=_DEV), t64))).float()
    root = (1 / torch.sqrt(1 - torch.pow(torch.tensor(h["beta2"], dtype=torch.float64, device=_DEV), t64))).float()
    keep = 1 - h["lr"] * h["decay"]

    def one(i, at, n):
        end = at + -(-n // _BLOCK) * _BLOCK
        p, g = s["p"][at:end], s["g"][at:end]
        if bits == 32:
            m, v = s["m"][at:end], s["v"][at:end]
        else:
            blocks = slice(at // _BLOCK, end // _BLOCK)
            m = _decode(s["mc"][at:end], s["ms"][blocks], 127).reshape(-1)
            v = _decode(s["vc"][at:end], s["vs"][blocks], 255).reshape(-1)
        m2 = m * h["beta1"] + g * (1 - h["beta1"])
        v2 = v * h["beta2"] + (g * g) * (1 - h["beta2"])
        p.copy_(p * keep - size * (m2 / (torch.sqrt(v2) * root + h["eps"])))
        if bits == 32:
            m.copy_(m2)
            v.copy_(v2)
            return
        r = _random_bits(end - at, i, t, s["seed"])
        mc, ms = _encode(m2.reshape(-1, _BLOCK), 127, r & 0xFFFF)
        vc, vs = _encode(v2.reshape(-1, _BLOCK), 255, r >> 16)
        s["mc"][at:end] = mc.reshape(-1).to(torch.int8)
        s["vc"][at:end] = vc.reshape(-1).to(torch.uint8)
        s["ms"][blocks], s["vs"][blocks] = ms, vs
        s["m"][at:end] = _decode(s["mc"][at:end], ms, 127).reshape(-1)
        s["v"][at:end] = _decode(s["vc"][at:end], vs, 255).reshape(-1)

    [one(i, at, n) for i, (at, n) in enumerate(s["spans"])]
    s["step"][0] += 1
    return dict(p=s["p"], m=s["m"], v=s["v"])


def _padded(rows, seq, pos, shape):
    out = torch.zeros(shape, device=_DEV)
    out[seq, :, pos] = rows.reshape(rows.shape[0], shape[1], shape[3])
    return out


def _attention_plain(s):
    c, (lq, lk), scale = s["case"], s["most"], s["scale"]
    n, h, kv, d = c["sequences"], c["heads"], c["kv_heads"], c["dim"]
    spread = lambda t: t.repeat_interleave(h // kv, dim=1)  # noqa: E731  (a group's heads share one key head)
    q = _padded(s["q"], s["qseq"], s["qpos"], (n, h, lq, d))
    k = _padded(s["k"], s["kseq"], s["kpos"], (n, kv, lk, d))
    v = _padded(s["v"], s["kseq"], s["kpos"], (n, kv, lk, d))
    i, j = torch.arange(lq, device=_DEV)[:, None], torch.arange(lk, device=_DEV)[None, :]
    seen = (i[None] < s["ql"][:, None, None]) & (j[None] < s["kl"][:, None, None])
    if c["causal"]:
        seen = seen & (j[None] <= i[None] + (s["kl"] - s["ql"])[:, None, None])
    sc = torch.matmul(q, spread(k).transpose(2, 3).contiguous()) * scale
    sc = sc.masked_fill_(~seen[:, None], -math.inf)
    top = sc.amax(3, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = sc.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    lse = top + torch.log(total)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    o = torch.matmul(p, spread(v))
    rows = lambda t, seq, pos: t[seq, :, pos].reshape(seq.shape[0], -1)  # noqa: E731
    out = dict(o=rows(o, s["qseq"], s["qpos"]))
    if c["pass_"] == "forward":
        return dict(out, lse=lse[s["qseq"], :, s["qpos"], 0])
    g = _padded(s["g"], s["qseq"], s["qpos"], (n, h, lq, d))
    joined = lambda t: t.reshape(n, kv, h // kv, lk, d).sum(2)  # noqa: E731
    dv = joined(torch.matmul(p.transpose(2, 3).contiguous(), g))
    ds = torch.matmul(g, spread(v).transpose(2, 3).contiguous())
    ds = ds.sub_((g * o).sum(3, keepdim=True)).mul_(p)
    del p, sc
    dq = torch.matmul(ds, spread(k)) * scale
    dk = joined(torch.matmul(ds.transpose(2, 3).contiguous(), q)) * scale
    return dict(out, dq=rows(dq, s["qseq"], s["qpos"]), dk=rows(dk, s["kseq"], s["kpos"]),
                dv=rows(dv, s["kseq"], s["kpos"]))


# ------------------------------------------------- the framework's kernels

def _norm_own(s):
    from rushlite_amd import abi
    lib, c = abi.lib(), s["case"]
    rows, n = s["x"].shape
    dt = abi.FLOAT64 if c["dtype"] == "f64" else abi.FLOAT32
    abi.check(lib.lmp_k_layer_norm(dt, rows, n, s["x"].data_ptr(), n, s["w"].data_ptr(), s["b"].data_ptr(), _EPS,
                                   s["y"].data_ptr(), n, s["mean"].data_ptr(), s["rstd"].data_ptr()))
    if c["pass_"] == "forward":
        return dict(y=s["y"], mean=s["mean"], rstd=s["rstd"])
    abi.check(lib.lmp_k_layer_norm_backward(
        dt, rows, n, s["g"].data_ptr(), n, s["x"].data_ptr(), n, s["w"].data_ptr(), s["mean"].data_ptr(),
        s["rstd"].data_ptr(), s["dx"].data_ptr(), n, s["dw"].data_ptr(), s["db"].data_ptr()))
    return dict(y=s["y"], dx=s["dx"], dw=s["dw"], db=s["db"])


def _adamw_own(s):
    from rushlite_amd import abi
    lib, h, bits = abi.lib(), _HYPER, s["case"]["bits"]
    if "list" not in s:  # the list of tensors, which an optimizer makes once
        ptr = lambda t, at: t.data_ptr() + at * t.element_size()  # noqa: E731
        wide = bits == 32
        s["list"] = (abi.AdamWTensor * len(s["spans"]))(*[
            abi.AdamWTensor(ptr(s["p"], at), ptr(s["g"], at), ptr(s["m"] if wide else s["mc"], at),
                            ptr(s["v"] if wide else s["vc"], at), None if wide else ptr(s["ms"], at // _BLOCK),
                            None if wide else ptr(s["vs"], at // _BLOCK), n, h["decay"]) for at, n in s["spans"]])
    abi.check(lib.lmp_k_adamw_f32(bits, len(s["spans"]), s["list"], h["lr"], h["beta1"], h["beta2"], h["eps"], s["seed"],
                                  s["step"].data_ptr()))
    if bits == 8:
        # the arena is whole blocks: one call reads every tensor's states
        n = s["p"].numel()
        abi.check(lib.lmp_k_adamw_decode(1, s["mc"].data_ptr(), s["ms"].data_ptr(), n, s["m"].data_ptr()))
        abi.check(lib.lmp_k_adamw_decode(0, s["vc"].data_ptr(), s["vs"].data_ptr(), n, s["v"].data_ptr()))
    return dict(p=s["p"], m=s["m"], v=s["v"])


def _attention_own(s):
    from rushlite_amd import abi
    lib, plan = abi.lib(), s["plan"].handle
    q, k, v, o = s["q"], s["k"], s["v"], s["o"]
    abi.check(lib.lmp_k_attention_f32(plan, q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(),
                                      v.stride(0), s["scale"], o.data_ptr(), o.stride(0), s["lse"].data_ptr()))
    if s["case"]["pass_"] == "forward":
        return dict(o=o, lse=s["lse"])
    g, dq, dk, dv = s["g"], s["dq"], s["dk"], s["dv"]
    abi.check(lib.lmp_k_attention_backward_f32(
        plan, q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), s["scale"], o.data_ptr(),
        o.stride(0), s["lse"].data_ptr(), g.data_ptr(), g.stride(0), dq.data_ptr(), dq.stride(0), dk.data_ptr(),
        dk.stride(0), dv.data_ptr(), dv.stride(0)))
    return dict(o=o, dq=dq, dk=dk, dv=dv)


def run(state):
    op = state["op"]
    if own:
        return (_norm_own if op == "layer_norm" else _adamw_own if op == "adamw" else _attention_own)(state)
    return (_norm_plain if op == "layer_norm" else _adamw_plain if op == "adamw" else _attention_plain)(state)


# ------------------------------------------------------------ work and truth

def _pairs(c):
    """How many (query, key) pairs the mask leaves."""
    total = 0
    for q, k in zip(*_lengths(c)):
        if not c["causal"]:
            total += q * k
        else:
            first = k - q + 1  # keys that the first query sees; each later one sees one more
            total += sum(range(max(0, first), k + 1)) if first <= 0 else q * (first + k) // 2
    return total


def work(case):
    c = case
    if c["op"] == "layer_norm":
        size, n = (8 if c["dtype"] == "f64" else 4), c["rows"] * c["cols"]
        train = c["pass_"] == "train"
        return dict(bytes=size * (n * (4 if train else 2) + c["cols"] * (4 if train else 2) + 2 * c["rows"] * (not train)),
                    flops=n * (20 if train else 8))
    if c["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(c))
        # p, g, m, v read and p, m, v written; in 8 bits the states are read out as float32 besides
        return dict(bytes=n * 28 if c["bits"] == 32 else int(n * (16 + 8 + 16 / _BLOCK)), flops=n * 14)
    ql, kl = _lengths(c)
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    rows, keys, train = sum(ql) * h * d, sum(kl) * kv * d, c["pass_"] == "train"
    return dict(bytes=4 * (rows * (4 if train else 2) + keys * (4 if train else 2) + sum(ql) * h * (not train)),
                flops=_pairs(c) * h * d * (14 if train else 4))


def _norm_exact(s):
    x, w, b = (s[n].double() for n in ("x", "w", "b"))
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sd = torch.sqrt(var + _EPS)
    y = (x - mean) / sd * w + b
    if s["case"]["pass_"] == "forward":
        return dict(y=y, mean=mean[:, 0], rstd=1 / sd[:, 0])
    # dx is the gradient projected off the ones vector and off the normalised row
    z = (x - mean) / sd
    u = s["g"].double() * w
    dx = (u - u.mean(1, keepdim=True) - z * (u * z).mean(1, keepdim=True)) / sd
    return dict(y=y, dx=dx, dw=torch.mul(s["g"].double(), z).sum(0), db=s["g"].double().sum(0))


def _adamw_exact(s):
    h, c = _HYPER, s["case"]
    t = _STEP0 + 1
    p, g = s["p"].double(), s["g"].double()
    if c["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        each = lambda t: t.double().repeat_interleave(_BLOCK)  # noqa: E731
        m = s["mc"].double().abs().pow(2) * s["mc"].double().sign() / 127 ** 2 * each(s["ms"])
        v = s["vc"].double().pow(2) / 255 ** 2 * each(s["vs"])
    m = m + (1 - h["beta1"]) * (g - m)
    v = v + (1 - h["beta2"]) * (g ** 2 - v)
    mh, vh = m / (1 - h["beta1"] ** t), v / (1 - h["beta2"] ** t)
    p = p - h["lr"] * h["decay"] * p - h["lr"] * mh / (vh.sqrt() + h["eps"])
    # what the codes come to hangs on which side of a random threshold a value falls: no 64-bit value of its own
    return dict(p=p, m=m, v=v) if c["bits"] == 32 else dict(p=p, m=None, v=None)


def _attention_exact(s):
    c, scale = s["case"], s["scale"]
    ql, kl = _lengths(c)
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    group, train = h // kv, c["pass_"] == "train"
    like = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=_DEV)  # noqa: E731
    out = dict(o=like(s["o"]))
    out.update(dq=like(s["dq"]), dk=like(s["dk"]), dv=like(s["dv"])) if train else out.update(lse=like(s["lse"]))
    q0 = k0 = 0
    for lq, lk in zip(ql, kl):
        rq, rk = slice(q0, q0 + lq), slice(k0, k0 + lk)
        bar = None
        if c["causal"]:
            bar = torch.ones(lq, lk, dtype=torch.bool, device=_DEV).triu(lk - lq + 1)
        for a in range(h):
            ca, cb = slice(a * d, (a + 1) * d), slice(a // group * d, (a // group + 1) * d)
            q, k, v = s["q"][rq, ca].double(), s["k"][rk, cb].double(), s["v"][rk, cb].double()
            logit = q @ k.t() * scale
            if bar is not None:
                logit = logit.masked_fill(bar, -math.inf)
            z = torch.logsumexp(logit, 1, keepdim=True)
            p = torch.exp(logit - torch.where(z == -math.inf, torch.zeros_like(z), z))
            out["o"][rq, ca] = p @ v
            if not train:
                out["lse"][rq, a] = z[:, 0]
                continue
            g = s["g"][rq, ca].double()
            dp = g @ v.t()
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
            out["dq"][rq, ca] = ds @ k
            out["dk"][rk, cb] += ds.t() @ q
            out["dv"][rk, cb] += p.t() @ g
        q0, k0 = q0 + lq, k0 + lk
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return (_norm_exact if s["op"] == "layer_norm" else _adamw_exact if s["op"] == "adamw" else _attention_exact)(s)
