"""Gates far out: values and slopes against their limits, through the C ABI."""
import numpy as np
import pytest

import _decoder as D
from test_gpu_decoder import gated

pytestmark = pytest.mark.gpu

MOST = float(np.finfo(np.float32).max)
FAR = [64.0, 300.0, 1e10, 1e19, 2e19, 1e25, 1e30, 3e38]


@pytest.mark.parametrize("gate", D.GATES)
def test_gate_and_slope_far_out(hip, gate):
    """For finite a of any size act is 0, 1 or a and the slope 0 or 1 (h and dx are exact to the roundings of two products)."""
    a = np.array(FAR + [-v for v in FAR], np.float32)[:, None]
    tiny = np.float32(2.0 ** -100)
    w = np.array([[1, tiny]], np.float32)
    h, dx, _, _ = gated(hip, gate, a, w, None, np.full_like(a, 0.5))
    a64, u = a.astype(np.float64), a.astype(np.float64) * float(tiny)
    up = a64 > 0
    act = up * 1.0 if gate == "sigmoid" else np.where(up, a64, 0)
    slope = 0 * a64 if gate == "sigmoid" else up * 1.0
    # a logistic of 64 is 1 - 2^-92, and of -64 2^-92 with what it is multiplied by
    slack = 2.0 ** -80 * np.maximum(1, np.abs(u)) * np.maximum(np.abs(a64), 1) * (np.abs(a64) < 300)
    past = np.abs(act * u) > MOST  # float32 has no such number: act(3e38) times 3e38 / 2^100
    assert (h[past] == np.inf).all()
    assert (np.abs(h - act * u) <= 4 * D.U32 * np.abs(act * u) + slack + 2.0 ** -126)[~past].all()
    want = 0.5 * u * slope + 0.5 * act * float(tiny)
    assert (np.abs(dx - want) <= 8 * D.U32 * np.abs(want) + slack + 2.0 ** -126).all()
