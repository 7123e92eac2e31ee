"""The 8-bit operators on the GPU at the edges of what they take (against plain_eight_bit.py where there is a result)."""

import pytest
import torch

from test_eight_bit_gpu import Batch

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
