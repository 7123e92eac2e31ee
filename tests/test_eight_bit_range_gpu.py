"""Attention of single tokens over the 8-bit cache where the softmax's weights span many powers of two, against the plain 64-bit
implementation: one key far ahead of the others, scores spread widely within a tile of keys, pages that are loud in one channel alone.

A weight counts for the result in proportion to itself, however small it is beside the largest: where the keys ahead hold small values
or none, the others are all there is.  The kernels round a weight to bfloat16 or to two 8-bit numbers, off by at most 2^-8 of it, and the
bound is test_eight_bit_gpu.py's as it is, 2^-7 of the same average of |v|.  With two 8-bit numbers that holds down to 2^-56 of the
largest weight, times its page's scale, of the key's tile.  Below that a weight is off by at most half the least e5m2 number, 2^-17,
in the units of the last band, 2^-42, of a largest one of 2^8: 2^-67 of the largest, and a value is at most 448 times its scale.  So
`floor` is the keys' number times 448 times 2^-67 times the largest scale: a weight is at most the denominator."""

import math

import pytest
import torch

import plain_eight_bit as plain
from test_eight_bit_gpu import Batch, attention_bound, close, run_decode, run_prefill, seeded

pytestmark = pytest.mark.gpu

# (heads, kv_heads, head_dim, page): one to 16 heads of a unit on tcgen05, and sizes that the other kernel takes
FORMS = [(4, 1, 128, 16), (2, 2, 128, 128), (8, 1, 128, 64), (16, 1, 128, 8), (24, 1, 128, 32), (4, 1, 64, 16), (4, 1, 128, 24)]


def one_ahead(seed, form, keys, ahead, gap, spread, value):
    """A request whose key `ahead` lies `gap` nats in front of the others, which are spread by `spread` nats (0: equal).  Its values are
    `value`, the others' about 1.  The softmax's scale goes with it."""
    heads, kv_heads, dim, page = form
    batch = Batch(seed, [keys], heads, kv_heads, dim, page)
    scale = gap / 256.0                                                # a query element of 1 against a key element of 256 (the scales are 1)
    batch.qkv[:, :heads * dim] = 1.0
    batch.k.scales[:] = 1.0
    batch.v.scales[:] = 2.0 ** -7
    batch.k.codes[:] = plain.e4m3(torch.randn(batch.k.codes.shape, generator=batch.g) * (spread / (scale * math.sqrt(dim - 1))))
    batch.k.codes[..., 0] = 0.0
    batch.v.codes[:] = plain.e4m3(128.0 + 12.0 * torch.randn(batch.v.codes.shape, generator=batch.g))
    at = int(batch.table[0, ahead // page]), ahead % page
    batch.k.codes[at] = 0.0
    batch.k.codes[at][..., 0] = 256.0
    batch.v.codes[at] = plain.e4m3(torch.tensor(value * 128.0))
    return batch, scale


def floor(batch, keys):
    return keys * 448.0 * 2.0 ** -67 * float(batch.v.scales.max())


def against_the_plain_result(batch, scale, keys, whole, window=None):
    """`whole`: one team of CTAs for all keys, as in a batch that fills the machine (sizes whose plan shares all keys out: its CTAs
    are what a plan for a short context has); else the keys are cut over many."""
    from libmir_b200 import kernels
    shared_out = kernels.decode_attention_8bit_plan(1, batch.heads, batch.kv_heads, batch.dim, batch.page, keys)[0] == 0
    out = run_decode(batch, batch.on_gpu(), [keys - 1], scale, window, plan_context=1 if whole and shared_out else keys)
    want, size = batch.decode([keys - 1], scale, window)
    close(out, want, attention_bound(want, size) + (floor(batch, keys) if shared_out else 0.0))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("gap", [9.0, 12.0, 14.7, 17.0, 24.0, 40.0])
@pytest.mark.parametrize("keys, ahead, spread, value", [(100, 40, 0.0, 0.0), (2048, 0, 0.3, 0.0), (2048, 1000, 0.0, 0.05)])
def test_one_key_ahead_of_many(form, gap, keys, ahead, spread, value):
    batch, scale = one_ahead(7, form, keys, ahead, gap, spread, value)
    against_the_plain_result(batch, scale, keys, whole=True)


@pytest.mark.parametrize("keys", [8192, 16384])
@pytest.mark.parametrize("gap", [9.0, 12.0, 14.0, 15.0, 17.0])
@pytest.mark.parametrize("spread, value", [(0.0, 0.0), (0.3, 0.05), (0.0, 0.05)])
def test_one_key_ahead_of_a_long_context(keys, gap, spread, value):
    batch, scale = one_ahead(8, (2, 1, 128, 16), keys, 3, gap, spread, value)
    against_the_plain_result(batch, scale, keys, whole=True)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("deviation", [3.0, 12.0, 30.0])
@pytest.mark.parametrize("whole", [True, False])
def test_scores_spread_widely_within_a_tile(form, deviation, whole):
    """Scores of some 100 nats of range in every tile, other ones for each head; the keys that are ahead of all hold zeros, so that the
    result comes from the others."""
    heads, kv_heads, dim, page = form
    keys = 700
    batch = Batch(9, [keys], heads, kv_heads, dim, page)
    batch.k.scales[:] = 1.0
    scale = deviation / (0.7 * 120.0 * math.sqrt(dim))
    s = torch.einsum("bpgd,ghd->bpgh", batch.k.codes, batch.qkv[0, :heads * dim].double().view(kv_heads, heads // kv_heads, dim)) * scale
    loudest = s.amax(dim=(0, 1))                                       # per head
    batch.v.codes[(s > loudest - 2.0 * deviation).any(dim=-1)] = 0.0
    for window in (None, 300):
        against_the_plain_result(batch, scale, keys, whole, window)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("louder", [10, 17, 22, 45, 80])
@pytest.mark.parametrize("whole", [True, False])
def test_pages_that_are_loud_in_one_channel(form, louder, whole):
    """A page whose scale is 2^louder times the others', for one channel's sake: its other channels are zeros, and the quiet pages'
    values are all there is."""
    heads, kv_heads, dim, page = form
    keys = 600
    batch = Batch(10, [keys], heads, kv_heads, dim, page)
    batch.v.scales[:] = torch.exp2(torch.randint(-3, 3, batch.v.scales.shape, generator=batch.g).double())
    for block in (0, (keys // page) // 2):
        at = int(batch.table[0, block])
        batch.v.scales[at] = 2.0 ** louder
        batch.v.codes[at] = 0.0
        batch.v.codes[at, :, :, 5] = 208.0
    against_the_plain_result(batch, dim ** -0.5, keys, whole)


@pytest.mark.parametrize("heads, kv_heads", [(8, 2), (16, 2), (32, 2)])
def test_many_requests_some_of_them_with_a_key_ahead(heads, kv_heads):
    """Whole rows and cut ones, wide and narrow tiles side by side, twice with the same result bit for bit."""
    dim, page, g = 128, 16, seeded(11)
    lengths = torch.randint(100, 900, (40,), generator=g).tolist()
    batch = Batch(12, lengths, heads, kv_heads, dim, page)
    scale = dim ** -0.5
    for r in range(0, 40, 3):                                          # queries that hold to one of their keys
        at = int(batch.table[r, 2]), 5
        for h in range(heads):
            key = batch.k.codes[at][h // (heads // kv_heads)]
            batch.qkv[r, h * dim:(h + 1) * dim] = (key / key.norm() * float(8 + r + h)).bfloat16()
        batch.v.codes[at] = 0.0
    cache = batch.on_gpu()
    positions = [n - 1 if i % 11 else -1 for i, n in enumerate(lengths)]
    first = run_decode(batch, cache, positions, scale)
    assert torch.equal(first, run_decode(batch, cache, positions, scale))
    picked = [i for i in range(0, 40, 3) if positions[i] >= 0] + [1, 20]
    want, size = batch.decode([p if i in picked else -1 for i, p in enumerate(positions)], scale)
    close(first[picked], want[picked], attention_bound(want, size)[picked] + floor(batch, 900))


def hidden_by_their_scores(form, block):
    """Keys whose scores are -inf in 32 bits, alone in their tile; the others' scores are 0."""
    heads, kv_heads, dim, page = form
    keys = 384 + page
    batch = Batch(13, [keys], heads, kv_heads, dim, page)
    batch.qkv[:, :heads * dim] = 1e30
    batch.k.codes[:] = 0.0
    for at in range(0, 128 // page * page) if block == "first" else range(-(-384 // page) * page, keys):
        where = int(batch.table[0, at // page]), at % page
        batch.k.codes[where] = -448.0
        batch.k.scales[where[0]] = 2.0 ** 60
    return batch, keys


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("block", ["first", "last"])
def test_single_tokens_with_scores_below_the_32_bit_numbers(form, block):
    """They weigh nothing, the others all the same."""
    batch, keys = hidden_by_their_scores(form, block)
    out = run_decode(batch, batch.on_gpu(), [keys - 1], 0.1)
    want, size = batch.decode([keys - 1], 0.1)
    close(out, want, attention_bound(want, size))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("block", ["first", "last"])
def test_portions_with_scores_below_the_32_bit_numbers(form, block):
    batch, keys = hidden_by_their_scores(form, block)
    for new in (5, 150):
        out = run_prefill(batch, batch.on_gpu(), [new], 0.1)
        want, size = batch.prefill([new], 0.1)
        close(out, want, attention_bound(want, size))
