"""The 8-bit operators without a GPU: addresses, empty batches and libraries that nobody asked for."""

import pytest

from libmir_b200 import kernels
from test_eight_bit import AT, BAD_ARGUMENT, native_decode, native_prefill


@pytest.mark.parametrize("off", [4, 8, 12])
def test_scratch_off_its_16_bytes_is_refused(off):
    """The kernels store and read it 8 and 16 bytes at a time."""
    assert native_decode(scratch=AT + off) == BAD_ARGUMENT                               # shared out over CTAs
    assert native_decode(dim=64, partition=128, parts=2, scratch=AT + off, floats=3 * 32 * 2 * 66) == BAD_ARGUMENT
    assert native_prefill(parts=2, scratch=AT + off, floats=1 << 24) == BAD_ARGUMENT
    assert native_prefill(dim=64, parts=2, scratch=AT + off, floats=1 << 24) == BAD_ARGUMENT
    message = kernels.library("eight_bit").mir_last_error().decode()
    assert "scratch" in message and "16-byte" in message
