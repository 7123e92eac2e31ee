"""The 8-bit operators without a GPU: addresses, empty batches and libraries that nobody asked for."""

import pathlib
import subprocess
import sys

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


def test_a_launch_mode_is_told_to_the_8bit_library_when_it_is_loaded():
    """set_programmatic_launch neither compiles nor loads the library for callers that never use it; those who do get the mode that was
    set last, before or after."""
    program = """
from libmir_b200 import kernels
kernels.set_programmatic_launch(2)
assert sorted(kernels.loaded_libraries()) == ["bf16", "core"], kernels.loaded_libraries()
assert kernels.library("eight_bit").mir_get_pdl() == kernels.library("core").mir_get_pdl() == 2
kernels.set_programmatic_launch(False)
assert [kernels.library(name).mir_get_pdl() for name in ("core", "bf16", "eight_bit")] == [0, 0, 0]
"""
    done = subprocess.run([sys.executable, "-c", program], cwd=pathlib.Path(__file__).parents[1], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr


def test_an_empty_batch_has_an_empty_table():
    """No rows, and a table of no columns, as a step without requests has them: nothing to do, nothing to refuse.  With rows it is refused."""
    assert native_decode(rows=0, table=None, width=0) == 0 and native_decode(dim=64, rows=0, table=None, width=0) == 0
    assert native_prefill(rows=0, tokens=0, table=None, width=0) == 0
    for call in (native_decode, native_prefill):
        assert call(width=0) == call(width=-1) == call(rows=0, width=-1) == BAD_ARGUMENT
