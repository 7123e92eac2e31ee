"""The 8-bit operators without a GPU: addresses, empty batches and libraries that nobody asked for."""

import ctypes
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


def prefill_plan(tokens, heads, kv_heads, dim, context):
    keys, count, floats = ctypes.c_int(), ctypes.c_int(), ctypes.c_longlong()
    assert kernels.library("eight_bit").mir_prefill_attention_8bit_plan(1, tokens, heads, kv_heads, dim, 16, context, ctypes.byref(keys),
                                                                        ctypes.byref(count), ctypes.byref(floats)) == 0
    return keys.value, count.value, floats.value


@pytest.mark.parametrize("dim, rows, at_once, start", [(128, 128, 148, 4), (64, 64, 296, 1)])
@pytest.mark.parametrize("tokens, heads, kv_heads", [(1, 32, 8), (4, 32, 8), (16, 32, 8), (100, 28, 4), (300, 32, 8), (400, 32, 8), (512, 32, 8),
                                                     (2048, 32, 8), (3, 1, 1), (5000, 64, 8)])
@pytest.mark.parametrize("context", [1, 500, 5000, 16513, 131072, 2147483391])
def test_portions_are_cut_over_the_keys_only_where_that_takes_less_time(dim, rows, at_once, start, tokens, heads, kv_heads, context):
    """Partitions cover the context in whole tiles of 128 keys, and their items, each some tiles' time longer than its keys, take a sixth
    less time on the CTAs that run at once than uncut ones."""
    keys, count, floats = prefill_plan(tokens, heads, kv_heads, dim, context)
    tiles, items = -(-context // 128), -(-tokens * heads // kv_heads // rows) * kv_heads
    assert keys % 128 == 0 and keys * count >= context and (count == 1 or keys * (count - 1) < context) and count <= 65535
    assert floats == (0 if count == 1 else tokens * heads * count * (dim + 2))
    time = -(-items * count // at_once) * (keys // 128 + start)
    assert count == 1 or time < -(-items // at_once) * (tiles + start) * 5 / 6 + 1
    if tiles >= 16 and items * 4 <= at_once:
        assert count >= 2


def test_a_portion_whose_items_fill_the_machine_is_not_cut():
    """512 tokens behind 16,001 keys, 32 heads over 8: 128 items on 148 SMs."""
    assert prefill_plan(512, 32, 8, 128, 16513)[1] == 1
