"""Whose bits a status read takes, against a fake of the library's status word: no device is touched."""
import ctypes
import os
import re

import pytest

import krea2_hrx_b200 as k
from krea2_hrx_b200 import _lib, parallel

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class FakeLibrary:
    """A status word that a read clears, all of it or the bits asked for."""

    def __init__(self, word):
        self.word = word

    def krea2_device_status_of(self, mask, out):
        ctypes.cast(out, ctypes.POINTER(ctypes.c_int))[0] = self.word & mask
        self.word &= ~mask
        return 0

    def krea2_device_status(self, out):
        return self.krea2_device_status_of(~0, out)


@pytest.mark.parametrize("word", [0, 64, 128, 192])
def test_a_sharded_chain_leaves_the_bits_of_other_kernels(monkeypatch, word):
    """An e4m3 product or a cross attention that gave up is not the chain's failure, and its caller still reads it."""
    fake = FakeLibrary(word)
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    parallel.require_clean_status()
    assert k.device_status() == word
    assert k.device_status() == 0


@pytest.mark.parametrize("bit", [1, 2, 4, 8, 16, 32])
def test_a_sharded_chain_reports_its_own_bits(monkeypatch, bit):
    fake = FakeLibrary(bit | 64)
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    with pytest.raises(k.Runtime, match=f"device status {bit}:"):
        parallel.require_clean_status()
    assert fake.word == 64


def test_the_mask_is_the_header_s():
    with open(os.path.join(ROOT, "include", "krea2_b200.h")) as f:
        header = dict(re.findall(r"(KREA2_STATUS_\w+) = (\d+)", f.read()))
    with open(os.path.join(ROOT, "krea2-b200-sys", "src", "lib.rs")) as f:
        crate = dict(re.findall(r"pub const (KREA2_STATUS_\w+): c_int = (\d+);", f.read()))
    assert header == crate and len(header) == 6
    assert int(header["KREA2_STATUS_CHAIN"]) == _lib.STATUS_CHAIN


def test_a_null_output_is_refused():
    assert k.lib().krea2_device_status_of(63, None) == 1
