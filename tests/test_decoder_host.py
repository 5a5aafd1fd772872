"""CPU checks of rotary positions, dropout, gated linear layers and the vocabulary loss: their refusals, which come before
anything touches the device, the generator's known answers, and the 64-bit gradients against differences."""
import numpy as np
import pytest

import _decoder as D

P = 1 << 20  # a non-null placeholder address, which nothing reads


@pytest.fixture
def L():
    """The library on a host without a GPU: every call below has to be refused by its checks alone."""
    from conftest import gpu_available
    if gpu_available():
        pytest.skip("placeholder pointers: the checks are tested on a host without a GPU")
    from rushlite_amd import abi
    return abi.lib()


def refused(status, text, code=1):
    from rushlite_amd import abi
    message = abi.lib().lmp_rt_last_error().decode()
    assert status == code and text in message, (status, message)


def no_device(status):
    """The checks let the call pass; then there is no device."""
    from rushlite_amd import abi
    assert status == abi.ERR_RUNTIME, abi.lib().lmp_rt_last_error().decode()


ROTARY = dict(dtype=4, rows=3, cols=40, heads=4, dim=8, turned=8, interleaved=0, x=P, ldx=40, positions=P, frequencies=P,
              scale=1.0, inverse=0, y=2 * P, ldy=40)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "neither Float32 nor Float64"), (dict(turned=7), "rotary_dim"), (dict(turned=10), "rotary_dim"),
    (dict(cols=31), "fewer than heads"), (dict(scale=float("nan")), "scale"), (dict(scale=1e300), "scale"),
    (dict(x=None), "null buffer"), (dict(y=None), "null buffer"), (dict(positions=None), "null buffer"),
    (dict(frequencies=None), "null buffer"), (dict(ldx=39), "leading dimension"), (dict(ldy=39), "leading dimension"),
    (dict(y=P, ldy=41), "in place"), (dict(y=P + 4), "overlap"), (dict(y=P + 160), "overlap"), (dict(y=P - 4), "overlap"),
    (dict(ldx=100, ldy=100, y=P + 4 * 39), "overlap"), (dict(ldx=100, ldy=100, y=P + 4 * 61), "overlap")], ids=str)
def test_rotary_refusals(L, change, text):
    refused(L.lmp_k_rotary(*{**ROTARY, **change}.values()), text)


def test_rotary_takes_rows_in_place_and_beside_each_other(L):
    for change in (dict(), dict(y=P), dict(y=P + 480), dict(ldx=100, ldy=100, y=P + 4 * 40), dict(ldx=100, ldy=100, y=P + 4 * 60),
                   dict(x=P + 160, y=P, ldx=80, ldy=80), dict(turned=0, frequencies=None), dict(dtype=5)):
        no_device(L.lmp_k_rotary(*{**ROTARY, **change}.values()))
    assert L.lmp_k_rotary(*{**ROTARY, "rows": 0, "x": None}.values()) == 0
    assert L.lmp_k_rotary(*{**ROTARY, "turned": 0, "y": P}.values()) == 0
    refused(L.lmp_k_rotary(*{**ROTARY, "cols": 1 << 31}.values()), "too many", 4)


DROP = dict(dtype=4, n=10, x=P, residual=None, rate=0.1, seed=3, state=P, used=2 * P, y=3 * P)
DROP_BACK = dict(dtype=4, n=10, g=P, rate=0.1, seed=3, used=P, dx=P)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), "neither Float32 nor Float64"), (dict(rate=-0.1), "rate"), (dict(rate=1.1), "rate"),
    (dict(rate=float("nan")), "rate"), (dict(x=None), "null buffer"), (dict(y=None), "null buffer"),
    (dict(state=None), "null buffer"), (dict(used=P), "used"), (dict(used=P + 8), "used")], ids=str)
def test_dropout_refusals(L, change, text):
    refused(L.lmp_k_dropout(*{**DROP, **change}.values()), text)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=0), "neither"), (dict(rate=2.0), "rate"), (dict(g=None), "null buffer"), (dict(used=None), "null buffer"),
    (dict(dx=None), "null buffer")], ids=str)
def test_dropout_backward_refusals(L, change, text):
    refused(L.lmp_k_dropout_backward(*{**DROP_BACK, **change}.values()), text)


@pytest.mark.parametrize("change", [dict(y=P + 4), dict(y=P + 36), dict(x=P + 36, y=P), dict(residual=3 * P + 8),
                                    dict(dtype=5, y=P + 76)], ids=str)
def test_dropout_refuses_an_output_beside_itself(L, change):
    refused(L.lmp_k_dropout(*{**DROP, **change}.values()), "overlaps")
    if "residual" not in change:
        y = change["y"]
        refused(L.lmp_k_dropout_backward(*{**DROP_BACK, "dtype": change.get("dtype", 4), "g": change.get("x", P), "dx": y}.values()),
                "overlaps")


def test_dropout_takes_outputs_that_touch_an_operand(L):
    for change in (dict(y=P + 40), dict(x=P + 40, y=P), dict(dtype=5, y=P + 80), dict(residual=3 * P)):
        no_device(L.lmp_k_dropout(*{**DROP, **change}.values()))


def test_dropout_edges(L):
    assert L.lmp_k_dropout_backward(*{**DROP_BACK, "n": 0, "g": None}.values()) == 0
    refused(L.lmp_k_dropout(*{**DROP, "n": 1 << 41}.values()), "too many", 4)
    for change in (dict(rate=0.0), dict(rate=1.0), dict(used=None), dict(residual=P), dict(y=P)):
        no_device(L.lmp_k_dropout(*{**DROP, **change}.values()))


GATED = dict(gate=0, rows=3, inp=5, hidden=4, x=P, ldx=5, w=P, ldw=8, b=P, h=P, ldh=4, pre=P, ldpre=8)
GATED_BACK = dict(gate=0, rows=3, inp=5, hidden=4, g=P, ldg=4, x=P, ldx=5, w=P, ldw=8, pre=P, ldpre=8, dx=P, lddx=5, dw=P,
                  lddw=8, db=P)


@pytest.mark.parametrize("change,text", [
    (dict(gate=5), "unknown gate 5"), (dict(gate=-1), "unknown gate"), (dict(inp=0), "no inputs"), (dict(hidden=0), "no inputs"),
    (dict(x=None), "null buffer"), (dict(w=None), "null buffer"), (dict(h=None), "null buffer"),
    (dict(ldx=4), "leading dimension"), (dict(ldw=7), "leading dimension"), (dict(ldh=3), "leading dimension"),
    (dict(ldpre=7), "leading dimension")], ids=str)
def test_gated_refusals(L, change, text):
    refused(L.lmp_k_gated_linear_f32(*{**GATED, **change}.values()), text)


@pytest.mark.parametrize("change,text", [
    (dict(gate=5), "unknown gate 5"), (dict(inp=0), "no inputs"), (dict(g=None), "null buffer"), (dict(x=None), "null buffer"),
    (dict(w=None), "null buffer"), (dict(pre=None), "null buffer"), (dict(ldg=3), "leading dimension"),
    (dict(ldx=4), "leading dimension"), (dict(ldw=7), "leading dimension"), (dict(ldpre=7), "leading dimension"),
    (dict(lddx=4), "leading dimension"), (dict(lddw=7), "leading dimension"), (dict(rows=0, lddw=7), "leading dimension")],
    ids=str)
def test_gated_backward_refusals(L, change, text):
    refused(L.lmp_k_gated_linear_backward_f32(*{**GATED_BACK, **change}.values()), text)


def test_gated_of_nothing(L):
    assert L.lmp_k_gated_linear_f32(*{**GATED, "rows": 0, "x": None}.values()) == 0
    assert L.lmp_k_gated_linear_backward_f32(*{**GATED_BACK, "dx": None, "dw": None, "db": None}.values()) == 0
    refused(L.lmp_k_gated_linear_f32(*{**GATED, "hidden": 1 << 30, "ldw": 1 << 31}.values()), "2^31", 4)
    refused(L.lmp_k_gated_linear_f32(*{**GATED, "ldx": 1 << 31}.values()), "2^31", 4)
    refused(L.lmp_k_gated_linear_backward_f32(*{**GATED_BACK, "ldg": 1 << 31}.values()), "2^31", 4)
    # what is not wanted needs no operands
    no_device(L.lmp_k_gated_linear_backward_f32(*{**GATED_BACK, "dx": None, "w": None, "ldw": 0, "lddx": 0}.values()))
    no_device(L.lmp_k_gated_linear_backward_f32(*{**GATED_BACK, "dw": None, "x": None, "ldx": 0, "lddw": 0}.values()))


LOSS = dict(rows=3, inp=5, vocab=7, x=P, ldx=5, w=P, ldw=7, b=P, targets=P, loss=P)
LOSS_GRAD = dict(rows=3, inp=5, vocab=7, x=P, ldx=5, w=P, ldw=7, b=P, targets=P, weights=P, loss=P, dx=P, lddx=5, dw=P, lddw=7,
                 db=P)


@pytest.mark.parametrize("change,text", [
    (dict(inp=0), "no inputs"), (dict(vocab=0), "no inputs"), (dict(x=None), "null buffer"), (dict(w=None), "null buffer"),
    (dict(targets=None), "null buffer"), (dict(loss=None), "null buffer"), (dict(ldx=4), "leading dimension"),
    (dict(ldw=6), "leading dimension")], ids=str)
def test_loss_refusals(L, change, text):
    refused(L.lmp_k_linear_cross_entropy_f32(*{**LOSS, **change}.values()), text)
    refused(L.lmp_k_linear_cross_entropy_grad_f32(*{**LOSS_GRAD, **change}.values()), text)


@pytest.mark.parametrize("change,text", [
    (dict(lddx=4), "leading dimension"), (dict(lddw=6), "leading dimension"), (dict(dw=None), "db without dw"),
    (dict(rows=0, lddw=6), "leading dimension")], ids=str)
def test_loss_gradient_refusals(L, change, text):
    refused(L.lmp_k_linear_cross_entropy_grad_f32(*{**LOSS_GRAD, **change}.values()), text)


def test_loss_of_nothing(L):
    assert L.lmp_k_linear_cross_entropy_f32(*{**LOSS, "rows": 0, "x": None}.values()) == 0
    refused(L.lmp_k_linear_cross_entropy_f32(*{**LOSS, "vocab": 1 << 31, "ldw": 1 << 31}.values()), "2^31", 4)
    refused(L.lmp_k_linear_cross_entropy_grad_f32(*{**LOSS_GRAD, "lddx": 1 << 31}.values()), "2^31", 4)
    no_device(L.lmp_k_linear_cross_entropy_grad_f32(*{**LOSS_GRAD, "b": None, "db": None, "weights": None}.values()))


def test_philox_known_answers():
    """The published test vectors of Philox4x32-10."""
    ones = 0xFFFFFFFF
    for counter, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
            ((ones,) * 4, (ones,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
            ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
             (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))):
        assert tuple(int(w) for w in D.philox(counter, key)) == want


def test_plain_forms_against_differences():
    """The 64-bit gradients the GPU tests compare with, against central differences of the 64-bit forward forms."""
    rng = np.random.default_rng(5)
    cases = []
    positions, f = np.array([0, 3, -7]), np.array([1.0, 0.3, 0.02])
    for interleaved in (False, True):
        x, g = rng.standard_normal((3, 19)), rng.standard_normal((3, 19))
        args = 2, 8, 6, interleaved, positions, f, 1.3
        cases.append((lambda x=x, g=g, args=args: (D.rotary(x, *args) * g).sum(), [(x, D.rotary(g, *args, inverse=True))]))
    for name in D.GATES:
        x, w, b, g = (rng.standard_normal(s) for s in ((4, 5), (5, 6), (6,), (4, 3)))
        _, *grads = D.gated(name, x, w, b, g)
        cases.append((lambda name=name, x=x, w=w, b=b, g=g: (D.gated(name, x, w, b) * g).sum(), list(zip((x, w, b), grads))))
    x, w, b, weights = (rng.standard_normal(s) for s in ((4, 5), (5, 7), (7,), (4,)))
    targets = np.array([3, -1, 0, 6])
    _, *grads = D.cross_entropy(x, w, b, targets, weights)
    cases.append((lambda: (D.cross_entropy(x, w, b, targets)[0] * weights).sum(), list(zip((x, w, b), grads))))
    for fn, pairs in cases:
        for a, grad in pairs:
            for i in np.ndindex(a.shape):
                old = a[i]
                a[i] = old + 1e-5
                up = fn()
                a[i] = old - 1e-5
                down = fn()
                a[i] = old
                assert abs((up - down) / 2e-5 - grad[i]) < 1e-7
