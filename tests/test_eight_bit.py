"""The 8-bit operators without a GPU: the oracle's number format against torch's, and what the native entry points refuse."""

import ctypes
import math

import pytest
import torch

import plain_eight_bit as plain
from libmir_b200 import kernels
from libmir_b200.errors import KernelError

BAD_ARGUMENT = 1


def test_the_oracles_rounding_is_e4m3s():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    every = every[~every.isnan()]
    assert torch.equal(plain.e4m3(every).float(), every)
    middles = (every.sort().values[:-1] + every.sort().values[1:]) / 2              # ties: to the even neighbour
    random = torch.randn(20000, generator=torch.Generator().manual_seed(0)) * torch.exp2(torch.randint(-12, 8, (20000,)).float())
    beyond = torch.tensor([math.inf, -math.inf, 449.0, 1e30, -470.0])
    for x in (middles, middles * (1 + 2.0 ** -20), random, beyond):
        assert torch.equal(plain.e4m3(x).float(), x.clamp(-448, 448).to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("largest", [0.0, 1e-44, 2.0 ** -110, 447.9, 448.0, 448.1, 1.0, 1.75, 1.7500001, 3.3e38])
def test_the_oracles_scale_is_the_least_that_holds_the_largest(largest):
    e = plain.exponent(largest)
    assert largest <= math.ldexp(448.0, e) and (e == plain.LEAST or largest > math.ldexp(448.0, e - 1))


def test_python_refuses_tensors_of_the_cpu():
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    weight = torch.zeros(128, 128).to(torch.float8_e4m3fn)
    with pytest.raises(KernelError, match="CUDA tensors"):
        kernels.linear_8bit(x, weight, torch.ones(1, 1), torch.zeros(2, 128))
    with pytest.raises(KernelError, match="CUDA tensors"):
        kernels.quantize_weight_8bit(torch.zeros(128, 128))
    pages, scales = torch.zeros(16, 1, 64).to(torch.float8_e4m3fn), torch.ones(1, 1)
    with pytest.raises(KernelError, match="CUDA tensors"):
        kernels.store_kv_8bit(torch.zeros(1, 192, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), pages, pages, scales,
                              scales, 16, 1, 1, 64)


# The native entry points check sizes, strides and addresses before anything is launched: made-up addresses never get further.
AT = 1 << 20


def native_store(**change):
    a = dict(qkv=AT, stride=(32 + 16) * 128, slots=AT, k=AT, v=AT, ks=AT, vs=AT, tokens=4, page=16, pages=10, heads=32, kv_heads=8,
             dim=128, stream=None)
    a.update(change)
    return kernels.library("eight_bit").mir_store_8bit(*a.values())


@pytest.mark.parametrize("change", [dict(dim=96), dict(dim=0), dict(page=0), dict(pages=0), dict(kv_heads=0), dict(tokens=-1),
                                    dict(stride=47 * 128), dict(stride=(32 + 16) * 128 + 2), dict(qkv=AT + 2), dict(k=AT + 1),
                                    dict(pages=1 << 28, page=16)])
def test_store_refuses(change):
    assert native_store(**change) == BAD_ARGUMENT


def native_decode(**change):
    a = dict(q=AT, stride=48 * 128, out=AT, k=AT, v=AT, ks=AT, vs=AT, pages=100, table=AT, width=10, positions=AT, rows=3, page=16,
             heads=32, kv_heads=8, dim=128, scale=0.1, window=0, partition=256, parts=1, scratch=None, floats=0, sinks=None, stream=None)
    if "partition" not in change and change.get("dim", 128) != 64:
        a.update(partition=0, parts=8, scratch=AT, floats=1 << 20)               # (what the plan says for these sizes)
    a.update(change)
    return kernels.library("eight_bit").mir_decode_attention_8bit(*a.values())


def native_prefill(**change):
    a = dict(q=AT, stride=48 * 128, out=AT, k=AT, v=AT, ks=AT, vs=AT, pages=100, table=AT, width=10, starts=AT, contexts=AT, rows=3,
             tokens=70, page=16, heads=32, kv_heads=8, dim=128, scale=0.1, window=0, partition=256, parts=1, scratch=None, floats=0,
             sinks=None, stream=None)
    a.update(change)
    return kernels.library("eight_bit").mir_prefill_attention_8bit(*a.values())


BAD_ATTENTION = [dict(dim=96), dict(dim=256), dict(heads=33), dict(heads=0), dict(kv_heads=0), dict(page=0), dict(pages=0),
                 dict(pages=1 << 28), dict(width=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(window=-1),
                 dict(stride=48 * 128 + 4), dict(stride=31 * 128), dict(q=AT + 8), dict(out=AT + 8), dict(k=AT + 8), dict(v=AT + 4),
                 dict(partition=0), dict(partition=100), dict(parts=0), dict(parts=70000), dict(parts=2), dict(rows=-1),
                 dict(parts=2, scratch=AT, floats=3 * 32 * 2 * 130 - 1)]


@pytest.mark.parametrize("change", [c for c in BAD_ATTENTION if c.get("parts") != 2]
                         + [dict(scratch=None), dict(floats=8 * 2 * 4 * 130 - 1), dict(parts=9), dict(partition=128), dict(dim=64, partition=0), dict(page=24, partition=0),
                            dict(parts=2, dim=64, scratch=None), dict(parts=2, dim=64, scratch=AT, floats=3 * 32 * 2 * 66 - 1)])
def test_decode_attention_refuses(change):
    assert native_decode(**change) == BAD_ARGUMENT


@pytest.mark.parametrize("change", BAD_ATTENTION + [dict(tokens=-1)])
def test_prefill_attention_refuses(change):
    assert native_prefill(**change) == BAD_ARGUMENT


@pytest.mark.parametrize("change", [dict(k=72), dict(k=0), dict(x_stride=100), dict(x_stride=130), dict(x=AT + 2), dict(weight=AT + 8),
                                    dict(out_stride=255), dict(accumulate=1), dict(bytes=100), dict(workspace=None),
                                    dict(workspace=AT + 4), dict(m=-1), dict(n=-1)])
def test_linear_refuses(change):
    a = dict(x=AT, x_stride=128, weight=AT, scales=AT, bias=None, out=AT, out_stride=256, out_float=0, accumulate=0, m=20, n=256, k=128,
             workspace=AT, bytes=1 << 20, stream=None)
    a.update(change)
    assert kernels.library("eight_bit").mir_linear_8bit(*a.values()) == BAD_ARGUMENT


def test_quantize_weight_refuses():
    for rows, columns in ((0, 128), (128, 0), (65536 * 128, 16)):
        assert kernels.library("eight_bit").mir_quantize_weight_8bit(1, AT, AT, AT, rows, columns, None) == BAD_ARGUMENT


@pytest.mark.parametrize("rows, heads, kv_heads, context", [(1, 32, 8, 1), (1, 32, 8, 40000), (64, 32, 8, 2048), (3, 28, 4, 0), (500, 8, 8, 129),
                                                            (1, 8, 8, 2147483647)])
def test_a_plan_covers_the_context_with_whole_tiles(rows, heads, kv_heads, context):
    keys, count, floats = kernels.decode_attention_8bit_plan(rows, heads, kv_heads, 64, 16, context)
    assert keys % 128 == 0 and keys * count >= context and (count == 1 or keys * (count - 1) < context) and count <= 65535
    assert floats == (0 if count == 1 else rows * heads * count * 66)
    keys, count, floats = kernels.decode_attention_8bit_plan(rows, heads, kv_heads, 128, 16, context)      # shared out
    units = kv_heads * -(-(heads // kv_heads) // 16)
    assert keys == 0 and count % units == 0 and 1 <= count // units <= max(1, min(2 * 148 // units, rows * max(1, -(-context // 128))))
    assert floats == 2 * count * min(heads // kv_heads, 16) * 130
    with pytest.raises(KernelError):
        kernels.decode_attention_8bit_plan(rows, heads, kv_heads + heads, 128, 16, context)
