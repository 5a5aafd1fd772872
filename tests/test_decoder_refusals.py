"""CPU checks of what the vocabulary loss refuses beside shapes and types."""
import numpy as np
import pytest


def test_weights_that_want_a_gradient_are_refused():
    """None would be formed for them."""
    import rushlite_amd as rsl
    cpu, i64 = rsl.device.cpu, rsl.dtype.int64

    def v(a, grad=False, dtype=rsl.dtype.float32):
        return rsl.Variable(np.asarray(a), grad, cpu, dtype)

    args = v(np.ones((2, 4))), v(np.ones((4, 6))), None, v([0, 1], dtype=i64)
    with pytest.raises(ValueError, match="weights take no gradient"):
        rsl.linear_cross_entropy(*args, v([1.0, 2.0], True))
    with rsl.no_grad(), pytest.raises(RuntimeError, match="not registered"):  # the CPU has no such operator
        rsl.linear_cross_entropy(*args, v([1.0, 2.0], True))
    with pytest.raises(RuntimeError, match="not registered"):
        rsl.linear_cross_entropy(*args, v([1.0, 2.0]))
