"""Runtime.sample's numbers on their way into C's types, without a device."""
import ctypes
import math

import pytest

import plamo_hip


class Library:
    """Takes plamo_sample's arguments as the library does, by the types it declares."""

    def plamo_sample(self, handle, slot, temperature, top_k, top_p, min_p, uniform, token, prob, err, size):
        self.top_k, self.uniform = ctypes.c_int32(top_k).value, ctypes.c_float(uniform).value
        return 0 if 0 <= self.uniform < 1 else 1


@pytest.fixture
def runtime():
    rt = plamo_hip.Runtime.__new__(plamo_hip.Runtime)
    rt._lib, rt._h = Library(), None
    yield rt
    rt._h = None


@pytest.mark.parametrize("uniform", [1 - 2.0 ** -53, 1 - 2.0 ** -25, 1 - 2.0 ** -24, 0.0, 5e-324, 2.0 ** -30, 0.7])
def test_numbers_below_one(runtime, uniform):
    runtime.sample(uniform)
    # the nearest FP32 number below 1
    assert runtime._lib.uniform == min(ctypes.c_float(uniform).value, 1 - 2.0 ** -24)


@pytest.mark.parametrize("uniform", [1.0, 1 + 2.0 ** -52, -5e-324, -2.0 ** -60, -0.5, math.nan, math.inf])
def test_numbers_outside(runtime, uniform):
    with pytest.raises(plamo_hip.PlamoError):
        runtime.sample(uniform)


@pytest.mark.parametrize("top_k,want", [(0, 0), (-1, -1), (5, 5), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1),
                                        (2 ** 32 + 1, 2 ** 31 - 1), (2 ** 63 - 1, 2 ** 31 - 1), (-2 ** 32 + 5, -2 ** 31)])
def test_top_k_past_32_bits(runtime, top_k, want):
    """More tokens than there are is all of them, not what is left in the low bits."""
    runtime.sample(0.5, top_k=top_k)
    assert runtime._lib.top_k == want
