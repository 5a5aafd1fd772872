"""CPU checks of the transformer operators' boundary: the header and its ctypes mirror, the refusals (made before anything
touches the device), and the work lists of packed attention against a count of what they have to cover."""
import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "lmp_hip_transformer.h"
HIP_SRC = ROOT / "rushlite_amd" / "csrc" / "hip"
P = 4096  # a non-null placeholder address, which nothing reads


def declared():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return sorted(set(re.findall(r"\b(lmp_k_\w+)\s*\(", text)))


def test_header_library_and_binding_agree():
    from rushlite_amd import abi
    lib = ctypes.CDLL(str(abi.LIB_PATH))
    assert set(declared()) == set(abi.TRANSFORMER_SIGNATURES)
    assert not [n for n in declared() if not hasattr(lib, n)]
    abi.lib()
    assert ctypes.sizeof(abi.AdamWTensor) == 64


@pytest.fixture
def L():
    """The library on a host without a GPU: every call below has to be refused by its checks alone."""
    from conftest import gpu_available
    if gpu_available():
        pytest.skip("placeholder pointers: the checks are tested on a host without a GPU")
    from rushlite_amd import abi
    return abi.lib()


def refused(abi, status, code, text):
    message = abi.lib().lmp_rt_last_error().decode()
    assert status == code and text in message, (status, message)


NORM = dict(dtype=4, rows=3, cols=8, x=P, ldx=8, w=P, b=P, eps=1e-5, y=P, ldy=8, mean=P, rstd=P)
NORM_BACK = dict(dtype=4, rows=3, cols=8, g=P, ldg=8, x=P, ldx=8, w=P, mean=P, rstd=P, dx=P, lddx=8, dw=P, db=P)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "neither Float32 nor Float64"), (dict(cols=0), "no values"), (dict(x=None), "null buffer"),
    (dict(y=None), "null buffer"), (dict(ldx=7), "leading dimension"), (dict(ldy=7), "leading dimension"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps")], ids=str)
def test_layer_norm_refusals(L, change, text):
    from rushlite_amd import abi
    refused(abi, L.lmp_k_layer_norm(*{**NORM, **change}.values()), abi.ERR_INVALID, text)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=0), "neither"), (dict(cols=0), "no values"), (dict(g=None), "null buffer"), (dict(x=None), "null buffer"),
    (dict(mean=None), "null buffer"), (dict(rstd=None), "null buffer"), (dict(ldg=7), "leading dimension"),
    (dict(ldx=7), "leading dimension"), (dict(lddx=7), "leading dimension")], ids=str)
def test_layer_norm_backward_refusals(L, change, text):
    from rushlite_amd import abi
    refused(abi, L.lmp_k_layer_norm_backward(*{**NORM_BACK, **change}.values()), abi.ERR_INVALID, text)


def test_layer_norm_of_nothing(L):
    from rushlite_amd import abi
    assert L.lmp_k_layer_norm(*{**NORM, "rows": 0, "x": None, "y": None}.values()) == abi.OK
    assert L.lmp_k_layer_norm_backward(*{**NORM_BACK, "dx": None, "dw": None, "db": None}.values()) == abi.OK
    assert L.lmp_k_layer_norm(*{**NORM, "cols": 1 << 31, "ldx": 1 << 31, "ldy": 1 << 31}.values()) == abi.ERR_UNSUPPORTED


@pytest.mark.parametrize("change,text", [
    (dict(bits=16), "32 or 8 bits"), (dict(step=None), "null step"), (dict(lr=float("nan")), "lr"),
    (dict(beta1=1.0), "beta1"), (dict(beta2=-0.1), "beta2"), (dict(beta2=float("nan")), "beta2"), (dict(eps=-1e-8), "eps"),
    (dict(p=None), "tensor 1: null buffer"), (dict(g=None), "tensor 1: null buffer"), (dict(v=None), "tensor 1: null buffer"),
    (dict(bits=8, m_scale=None), "tensor 1: states of 8 bits"), (dict(decay=float("inf")), "tensor 1: decay"),
    (dict(list=None), "null list")], ids=str)
def test_adamw_refusals(L, change, text):
    from rushlite_amd import abi
    call = dict(bits=32, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=P, p=P, g=P, m=P, v=P, m_scale=P, v_scale=P, n=5,
                decay=0.0, **{k: v for k, v in change.items() if k == "list"})
    call.update(change)
    good = abi.AdamWTensor(P, P, P, P, P, P, 5, 0.0)
    bad = abi.AdamWTensor(*[call[k] for k in ("p", "g", "m", "v", "m_scale", "v_scale", "n", "decay")])
    tensors = None if "list" in change else ctypes.cast((abi.AdamWTensor * 2)(good, bad), ctypes.c_void_p)
    refused(abi, L.lmp_k_adamw_f32(call["bits"], 2, tensors, call["lr"], call["beta1"], call["beta2"], call["eps"], 1,
                                   call["step"]), abi.ERR_INVALID, text)


def test_adamw_decode_refusals(L):
    from rushlite_amd import abi
    for args in ((None, P, 3, P), (P, None, 3, P), (P, P, 3, None)):
        refused(abi, L.lmp_k_adamw_decode(1, *args), abi.ERR_INVALID, "null buffer")
    assert L.lmp_k_adamw_decode(1, None, None, 0, None) == abi.OK


@pytest.mark.parametrize("ql,kl,heads,kv_heads,dim,code,text", [
    ([1], [1], 6, 4, 8, 1, "multiple of kv_heads"), ([1], [1], 0, 0, 8, 1, "multiple of kv_heads"),
    ([1], [1], 4, 0, 8, 1, "multiple of kv_heads"), ([1], [1], 4, 4, 0, 1, "head_dim is 0"),
    ([1], [1], 4, 4, 257, 4, "above 256"), ([1, -1], [1, 1], 4, 4, 8, 1, "sequence 1: negative"),
    ([1, 1], [1, -2], 4, 4, 8, 1, "sequence 1: negative"), ([1 << 30], [1], 4, 4, 8, 4, "too many rows"),
    ([1], [1 << 31], 4, 4, 8, 4, "too many rows"), ([1], [1], 1 << 17, 1, 8, 4, "65536 heads")])
def test_attention_plan_refusals(L, ql, kl, heads, kv_heads, dim, code, text):
    from rushlite_amd import abi
    with pytest.raises(abi.LmpError, match=text) as e:
        abi.AttentionPlan(ql, kl, heads=heads, kv_heads=kv_heads, head_dim=dim)
    assert e.value.status == code


def test_attention_plan_arguments():
    from rushlite_amd import abi
    with pytest.raises(ValueError, match="per sequence"):
        abi.AttentionPlan([1, 2], [1], heads=1, head_dim=8)
    assert abi.lib().lmp_k_attention_plan_destroy(None) == abi.OK


def test_attention_without_a_plan(L):
    from rushlite_amd import abi
    refused(abi, L.lmp_k_attention_f32(None, P, 8, P, 8, P, 8, 1.0, P, 8, P), abi.ERR_INVALID, "null plan")
    refused(abi, L.lmp_k_attention_backward_f32(None, P, 8, P, 8, P, 8, 1.0, P, 8, P, P, 8, P, 8, P, 8, P, 8),
            abi.ERR_INVALID, "null plan")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_attention_work_lists(tmp_path):
    """Every (row, key) pair of a batch is covered once by the lists, parts are joined once, and indices stay inside."""
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-O2", "-std=c++20", "-fsanitize=address,undefined", f"-I{HIP_SRC}",
                    str(ROOT / "tests" / "native" / "attention_plan_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "attention lists ok" in out.stdout


def test_plain_forms_against_differences():
    """The 64-bit gradients the GPU tests compare with, against central differences of the 64-bit forward forms."""
    import _transformer as T
    rng = np.random.default_rng(3)
    x, g, w, b = rng.standard_normal((3, 7)), rng.standard_normal((3, 7)), rng.standard_normal(7), rng.standard_normal(7)
    dx, dw, db = T.layer_norm_backward(g, x, w, 1e-5)
    f = lambda: (T.layer_norm(x, w, b, 1e-5)[0] * g).sum()  # noqa: E731
    ql, kl, heads, kv, d = [3, 0, 2], [4, 2, 1], 4, 2, 3
    q, go = rng.standard_normal((5, heads * d)), rng.standard_normal((5, heads * d))
    k, v = rng.standard_normal((7, kv * d)), rng.standard_normal((7, kv * d))
    _, _, dq, dk, dv = T.attention(q, k, v, ql, kl, heads, kv, 0.6, True, go)
    h = lambda: (T.attention(q, k, v, ql, kl, heads, kv, 0.6, True)[0] * go).sum()  # noqa: E731
    for fn, pairs in ((f, ((x, dx), (w, dw), (b, db))), (h, ((q, dq), (k, dk), (v, dv)))):
        for a, grad in pairs:
            for i in np.ndindex(a.shape):
                old = a[i]
                a[i] = old + 1e-5
                up = fn()
                a[i] = old - 1e-5
                down = fn()
                a[i] = old
                assert abs((up - down) / 2e-5 - grad[i]) < 1e-7


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("field,text", [
    ("p", "tensors 0 and 1"), ("m", "tensors 0 and 1"), ("v", "tensors 0 and 1"), ("m_scale", "tensors 0 and 1"),
    ("v_scale", "tensors 0 and 1"), ("own", "tensors 1 and 1")])
def test_adamw_refuses_buffers_that_overlap(L, bits, field, text):
    """One buffer in two entries, or in one entry twice, from its start or from within it; neighbours do not overlap.  600
    values: states of 2400 or 600 bytes, three scales."""
    from rushlite_amd import abi
    if bits == 32 and "scale" in field:
        pytest.skip("states of 32 bits have no scales")

    def call(*tensors):
        args = ctypes.cast((abi.AdamWTensor * len(tensors))(*tensors), ctypes.c_void_p)
        return L.lmp_k_adamw_f32(bits, len(tensors), args, 1e-3, 0.9, 0.999, 1e-8, 1, P)

    names = [n for n, _ in abi.AdamWTensor._fields_]
    size = dict(p=2400, g=2400, m=2400 if bits == 32 else 600, v=2400 if bits == 32 else 600, m_scale=12, v_scale=12)
    # one after another without room between them
    at, both = 1 << 20, []
    for _ in range(2):
        t = {}
        for name, n in size.items():
            t[name] = at
            at += n
        both.append(t)
    make = lambda t: abi.AdamWTensor(*[t[n] for n in names[:6]], 600, 0.0)  # noqa: E731
    status = call(*map(make, both))
    assert status != abi.OK and "overlap" not in L.lmp_rt_last_error().decode()  # there is no device
    for shift in (0, size["p" if field == "own" else field] - 4):
        bad = dict(both[1])
        if field == "own":
            bad["m"] = bad["p"] + shift
        else:
            bad[field] = both[0][field] + shift
        refused(abi, call(make(both[0]), make(bad)), abi.ERR_INVALID, text)
    # what has no values holds no memory
    empty = abi.AdamWTensor(*[both[0][n] for n in names[:6]], 0, 0.0)
    assert call(make(both[0]), empty) != abi.OK and "overlap" not in L.lmp_rt_last_error().decode()


def test_adamw_refuses_two_variables_over_one_buffer():
    import rushlite_amd as rsl
    x = rsl.Variable(np.ones(3, np.float32), True, rsl.device.cpu)
    with pytest.raises(ValueError, match="same memory"):
        rsl.optim.AdamW([x, rsl.Variable(x.data, True)])


def test_adamw_of_a_module_passes_over_frozen_parameters():
    """What is refused here is the trained parameter's device."""
    import rushlite_amd as rsl

    class Half(rsl.Module):
        def __init__(self):
            super().__init__()
            self.frozen = rsl.Variable(np.ones(3, np.float32), False, rsl.device.cpu)
            self.trained = rsl.Variable(np.ones(3, np.float32), True, rsl.device.cpu)

        def forward(self):
            return self.frozen

    with pytest.raises(ValueError, match="parameter 0 is not float32 on the HIP device"):
        rsl.optim.AdamW(Half())
