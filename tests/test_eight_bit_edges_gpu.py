"""The 8-bit operators on the GPU at the edges of what they take (against plain_eight_bit.py where there is a result)."""

import pytest
import torch

import plain_eight_bit as plain
from test_eight_bit_gpu import E4M3, Batch, close, product_bound, seeded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
def test_scratch_cut_from_an_arena_at_an_odd_element_is_refused(dim):
    from libmir_b200 import kernels
    from libmir_b200.errors import KernelError
    heads, kv_heads, page, context = 8, 2, 16, 3000
    batch = Batch(1, [context], heads, kv_heads, dim, page)
    cache, table, out = batch.on_gpu(), batch.table.cuda(), torch.full((1, heads * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    partition, count, floats = kernels.decode_attention_8bit_plan(1, heads, kv_heads, dim, page, context)
    arena = torch.empty(floats + 16, device="cuda")
    positions = torch.tensor([context - 1], dtype=torch.int32).cuda()

    def decode(first):
        kernels.decode_attention_8bit(batch.qkv[:1].cuda(), out, *cache, table, positions, page, heads, kv_heads, dim, 0.1, None, partition,
                                      count, arena[first:first + floats])

    def prefill(first):
        starts = torch.tensor([0, 1], dtype=torch.int32).cuda()
        kernels.prefill_attention_8bit(batch.qkv[:1].cuda(), out, *cache, table, starts, positions + 1, page, heads, kv_heads, dim, 0.1, None,
                                       alloc=lambda shape, dtype: torch.empty(shape[0] + 16, dtype=dtype, device="cuda")[first:first + shape[0]])
    for call in (decode, prefill):
        for first in (1, 2, 3):
            with pytest.raises(KernelError, match="16-byte"):
                call(first)
        assert (out == 7.0).all()
        call(4)
        assert not (out == 7.0).any()
        out.fill_(7.0)


def test_the_error_is_read_when_every_stream_is_done():
    """A kernel on a stream of its own, which a copy on the default stream does not wait for, might still give up."""
    from libmir_b200 import kernels
    assert kernels.eight_bit_error() == 0                              # (loads the library)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(200_000_000)                                 # a tenth of a second
    assert kernels.eight_bit_error() == 0
    assert stream.query()


def test_a_kernel_that_gave_up_stores_nothing_until_it_is_reset():
    """The flag that a wait which runs out sets, set by the reader here (no wait runs out): every call leaves its result as it is, what
    it adds to among them, and joins nothing; afterwards all is as before."""
    from libmir_b200 import kernels
    from libmir_b200.kernels import eight_bit
    lib = kernels.library("eight_bit")
    heads, kv_heads, page = 8, 2, 16
    batch = Batch(2, [3000, 40], heads, kv_heads, 128, page)
    cache, table = batch.on_gpu(), batch.table.cuda()
    positions = torch.tensor([2999, 39], dtype=torch.int32).cuda()
    plan = kernels.decode_attention_8bit_plan(2, heads, kv_heads, 128, page, 3000)
    scratch = torch.zeros(plan[2], device="cuda")
    codes = torch.ones(1000, 1024, device="cuda").to(eight_bit.E4M3)
    scales = torch.ones(8, 8, device="cuda")

    def decode(out):
        kernels.decode_attention_8bit(batch.qkv[:2].cuda(), out, *cache, table, positions, page, heads, kv_heads, 128, 0.1, None, plan[0],
                                      plan[1], scratch)

    def prefill(counts):
        def call(out):
            starts = torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32).cuda()
            kernels.prefill_attention_8bit(batch.qkv[:sum(counts)].cuda(), out, *cache, table, starts, positions + 1, page, heads, kv_heads,
                                           128, 0.1, None)
        return call

    def linear(out):
        kernels.linear_8bit(torch.ones(out.shape[0], 1024, dtype=torch.bfloat16, device="cuda"), codes, scales, out,
                            accumulate=out.dtype == torch.float32)
    calls = [(decode, 2, heads * 128, torch.bfloat16), (prefill([2, 1]), 3, heads * 128, torch.bfloat16),
             (prefill([2900, 40]), 2940, heads * 128, torch.bfloat16)]
    calls += [(linear, m, 1000, dtype) for m in (1, 16, 40, 128, 129, 300) for dtype in (torch.bfloat16, torch.float32)]
    try:
        for name in eight_bit._ERRORS:
            assert getattr(lib, name)(3) == 0
        assert kernels.eight_bit_error() == 3
        for call, rows, width, dtype in calls:
            out = torch.full((rows, width), 7.0, dtype=dtype, device="cuda")
            call(out)
            assert (out == 7.0).all()
        assert kernels.eight_bit_error(reset=True) == 3 and kernels.eight_bit_error() == 0
    finally:
        kernels.eight_bit_error(reset=True)
    for call, rows, width, dtype in calls:
        out = torch.full((rows, width), 7.0, dtype=dtype, device="cuda")
        call(out)
        assert not (out == 7.0).any() if call is linear else (out != 7.0).any(dim=1).all()
        if call is linear:
            assert (out == 1024.0 + (7.0 if dtype == torch.float32 else 0.0)).all()
    assert kernels.eight_bit_error() == 0


@pytest.mark.parametrize("size", [1e35, 1e-35])
@pytest.mark.parametrize("n", [200, 19000])
@pytest.mark.parametrize("m", [1, 16, 17, 128, 129])
def test_products_of_very_large_and_very_small_rows(m, n, size):
    """Rows near both ends of the 32-bit numbers whose results are ordinary ones: what is on the way there is, too, with few rows and with
    many.  (Blocks' scales that multiply to less than the normal numbers, 2^-126, are held to 2^-150: 2^25 times that at most for 128
    products of two numbers of 448, for each block.)"""
    from libmir_b200 import kernels
    g = seeded(m)
    k = 272
    x = (torch.randn(m, k, generator=g) * size).bfloat16()
    codes = (torch.randn(n, k, generator=g) * 100).clamp(-448, 448).to(E4M3)
    scales = torch.rand(-(-n // 128), -(-k // 128), generator=g) * 1e-3 + 1e-4
    weight = plain.weight_values(codes, scales)
    out = torch.full((m, n), 7.0, device="cuda")
    kernels.linear_8bit(x.cuda(), codes.cuda(), scales.cuda(), out)
    want = plain.rounded_rows(x) @ weight.t()
    bound = product_bound(x, weight, torch.float32, torch.zeros(1, dtype=torch.float64))(want)
    close(out, want, bound - 1e-35 + 3 * 2.0 ** -125)


@pytest.mark.parametrize("dim", [64, 128])
def test_a_step_without_requests(dim):
    from libmir_b200 import kernels
    batch = Batch(3, [40], 8, 2, dim, 16)
    cache, empty = batch.on_gpu(), torch.zeros(0, dtype=torch.int32, device="cuda")
    qkv, out = batch.qkv[:0].cuda(), torch.zeros(0, 8 * dim, dtype=torch.bfloat16, device="cuda")
    plan = kernels.decode_attention_8bit_plan(0, 8, 2, dim, 16, 0)
    for width in (0, 5):
        table = torch.zeros(0, width, dtype=torch.int32, device="cuda")
        kernels.decode_attention_8bit(qkv, out, *cache, table, empty, 16, 8, 2, dim, 0.1, None, plan[0], plan[1],
                                      torch.empty(plan[2], device="cuda"))
        kernels.prefill_attention_8bit(qkv, out, *cache, table, torch.zeros(1, dtype=torch.int32, device="cuda"), empty, 16, 8, 2, dim, 0.1, None)
        kernels.store_kv_8bit(qkv, empty, *cache, 16, 8, 2, dim)


def test_a_workspace_that_is_too_small_or_off_its_16_bytes_is_refused():
    from libmir_b200 import kernels
    from libmir_b200.errors import KernelError
    x = torch.ones(20, 256, dtype=torch.bfloat16, device="cuda")
    codes, scales = torch.ones(130, 256, device="cuda").to(E4M3), torch.ones(2, 2, device="cuda")
    out = torch.full((20, 130), 7.0, device="cuda")
    for take in (lambda n: slice(0, n - 1), lambda n: slice(8, n + 8), lambda n: slice(0, 0)):
        with pytest.raises(KernelError, match="workspace"):
            kernels.linear_8bit(x, codes, scales, out, alloc=lambda shape, dtype: torch.empty(shape[0] + 64, dtype=dtype, device="cuda")[take(shape[0])])
    assert (out == 7.0).all()
    kernels.linear_8bit(x, codes, scales, out, alloc=lambda shape, dtype: torch.empty(shape[0] + 64, dtype=dtype, device="cuda")[16:])
    assert (out == 256.0).all()
