"""Scales of cross attention that its exponents of two cannot hold: host work, no device is touched."""
import ctypes

import pytest

import krea2_hrx_b200 as k


def status_of(scale, out):
    buffer = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buffer) + 15) & ~15
    return k.lib().krea2_cross_attention(None, 1, 5, 7, at, at, at, None, None, at + out, 4, 2, 64, 1280, 256, 896, 128, 896, 128, 1280, 256, 0, scale, 1)


# the output is off a 16-byte boundary, which is refused after the scale: no call reaches the device
@pytest.mark.parametrize("scale,needle", [(3.0e38, "scale"), (2.0 ** 127.7, "scale"), (float("inf"), "scale"), (2.0 ** 126, "aligned"), (2.0 ** -140, "aligned")])
def test_scales_whose_power_of_two_overflows_are_refused(scale, needle):
    assert status_of(scale, 8) == 1
    assert needle in k.lib().krea2_last_error().decode()
