"""The 8-bit operators on the GPU against the plain 64-bit implementation (plain_eight_bit.py).

Tolerances count roundings.  The stored cache is compared bit for bit.  Attention: the result is rounded to bf16 (half a
step: 2^-8 of it), a weight of the softmax is rounded on its way into the product with the values, to bf16 (2^-8) or to
an e4m3 number and an e5m2 number that holds what the first left (2^-4 * 2^-3 = 2^-7), which moves the result by at most
that share of the same average of |v|; scores, exponentials and sums are 32-bit (2^-12 leaves room for scores up to 100 and
a query's 2^-25 of its largest element).  Products: 32-bit sums of exact products, at most 128 terms and then one per block
of 128 columns, the scale, the bias and what is added to: 2^-24 each of the sum of magnitudes, and the result's rounding."""

import math

import numpy as np
import pytest
import torch

import plain_eight_bit as plain

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def seeded(seed):
    return torch.Generator().manual_seed(seed)


def attention_bound(want, size):
    return want.abs() * 2.0 ** -8 + size * (2.0 ** -7 + 2.0 ** -12) + 1e-30


def close(got, want, bound, what=""):
    got = got.double().cpu()
    off = (got - want).abs() - bound
    assert not torch.isnan(got).any() and off.max() <= 0, f"{what}: {off.max()} over the bound at {int(off.argmax())}"


class Batch:
    """Requests with a filled 8-bit cache: `lengths` cached tokens each, pages anywhere in the pool."""

    def __init__(self, seed, lengths, heads, kv_heads, dim, page, loud=1.0, width=None):
        g = seeded(seed)
        self.g, self.lengths, self.heads, self.kv_heads, self.dim, self.page = g, lengths, heads, kv_heads, dim, page
        blocks = [-(-n // page) for n in lengths]
        self.pool = sum(blocks) + 2
        order = torch.randperm(self.pool, generator=g)
        self.table = torch.full((len(lengths), max(max(blocks), 1) if width is None else width), -1, dtype=torch.int32)
        at = 0
        for r, count in enumerate(blocks):
            self.table[r, :count] = order[at:at + count].int()
            at += count
        self.k, self.v = plain.Cache(self.pool, page, kv_heads, dim), plain.Cache(self.pool, page, kv_heads, dim)
        for cache in (self.k, self.v):
            cache.codes = plain.e4m3(torch.randn(cache.codes.shape, generator=g) * 120.0)
            cache.scales = torch.exp2(torch.randint(-9, -4, cache.scales.shape, generator=g).double()) * loud
        self.qkv = (torch.randn(max(1, sum(lengths)), (heads + 2 * kv_heads) * dim, generator=g) * 0.7).bfloat16()

    def on_gpu(self):
        return tuple(t.contiguous().cuda() for t in (self.k.rows().float().to(E4M3), self.v.rows().float().to(E4M3),
                                                     self.k.scales.float(), self.v.scales.float()))

    def decode(self, positions, scale, window=None, sinks=None, qkv=None):
        """The 64-bit results [rows, heads * dim] (zeros for padding rows) and sizes."""
        qkv = self.qkv if qkv is None else qkv
        kv, vv = self.k.values(), self.v.values()
        out = torch.zeros(len(positions), self.heads * self.dim, dtype=torch.float64)
        size = torch.zeros_like(out)
        for r, position in enumerate(positions):
            if position >= 0:
                q = qkv[r:r + 1, :self.heads * self.dim].view(1, self.heads, self.dim)
                o, s = plain.attention(q, kv, vv, self.page, self.table[r].tolist(), [position], scale, window, sinks)
                out[r], size[r] = o.flatten(), s.flatten()
        return out, size

    def prefill(self, new, scale, window=None, sinks=None):
        kv, vv = self.k.values(), self.v.values()
        outs, sizes, first = [], [], 0
        for r, (count, context) in enumerate(zip(new, self.lengths)):
            q = self.qkv[first:first + count, :self.heads * self.dim].view(count, self.heads, self.dim)
            o, s = plain.attention(q, kv, vv, self.page, self.table[r].tolist(), range(context - count, context), scale, window, sinks)
            outs.append(o.flatten(1))
            sizes.append(s.flatten(1))
            first += count
        return torch.cat(outs), torch.cat(sizes)


def run_decode(batch, cache, positions, scale, window=None, sinks=None, table=None, plan_context=None, qkv=None, out=None):
    from libmir_b200 import kernels
    rows = len(positions)
    table = batch.table.cuda() if table is None else table
    longest = max(max(positions) + 1, 1) if plan_context is None else plan_context
    partition, count, floats = kernels.decode_attention_8bit_plan(rows, batch.heads, batch.kv_heads, batch.dim, batch.page, longest)
    scratch = torch.full((floats,), math.nan, device="cuda") if floats else None
    out = torch.full((rows, batch.heads * batch.dim), 7.0, dtype=torch.bfloat16, device="cuda") if out is None else out
    qkv = batch.qkv[:rows].cuda() if qkv is None else qkv
    kernels.decode_attention_8bit(qkv, out, *cache, table, torch.tensor(positions, dtype=torch.int32).cuda(), batch.page, batch.heads,
                                  batch.kv_heads, batch.dim, scale, window, partition, count, scratch,
                                  None if sinks is None else sinks.cuda())
    return out


def run_prefill(batch, cache, new, scale, window=None, sinks=None, extra=0, **more):
    from libmir_b200 import kernels
    tokens = sum(new)
    out = torch.full((tokens + extra, batch.heads * batch.dim), 7.0, dtype=torch.bfloat16, device="cuda")
    qkv = torch.cat([batch.qkv[:tokens], batch.qkv[:1].expand(extra, -1)]).cuda()
    starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).cuda()
    kernels.prefill_attention_8bit(qkv, out, *cache, batch.table.cuda(), starts, torch.tensor(batch.lengths, dtype=torch.int32).cuda(),
                                   batch.page, batch.heads, batch.kv_heads, batch.dim, scale, window,
                                   None if sinks is None else sinks.cuda(), **more)
    return out


# ------------------------------------------------------------------------------------------------ the cache's writes
def run_store(qkv, slots, cache, batch):
    from libmir_b200 import kernels
    kernels.store_kv_8bit(qkv.cuda(), torch.tensor(slots, dtype=torch.int32).cuda(), *cache, batch.page, batch.heads, batch.kv_heads,
                          batch.dim)


def same_cache(batch, cache):
    k, v, ks, vs = (t.cpu() for t in cache)
    assert torch.equal(ks.double(), batch.k.scales) and torch.equal(vs.double(), batch.v.scales)
    for got, want in ((k, batch.k.rows()), (v, batch.v.rows())):
        got = got.float().double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def plain_store(batch, qkv, slots):
    h, g, d = batch.heads, batch.kv_heads, batch.dim
    batch.k.store(qkv[:, h * d:(h + g) * d].reshape(-1, g, d), slots)
    batch.v.store(qkv[:, (h + g) * d:(h + 2 * g) * d].reshape(-1, g, d), slots)


@pytest.mark.parametrize("dim, page, heads, kv_heads, new, before", [
    (128, 16, 32, 8, [1, 1, 1], [0, 15, 100]), (128, 16, 4, 1, [17, 1, 33], [5, 16, 0]), (64, 8, 3, 3, [40, 7], [3, 1]),
    (64, 5, 2, 2, [13], [4]), (128, 128, 8, 4, [300, 1], [100, 127]), (128, 1, 2, 2, [3], [2]), (128, 48, 28, 4, [1100], [31]),
    (128, 16, 0, 17, [20], [9])])
def test_store_keeps_the_least_scale_and_takes_a_page_along(dim, page, heads, kv_heads, new, before):
    lengths = [n + b for n, b in zip(new, before)]
    batch = Batch(3, lengths, heads, kv_heads, dim, page)
    cache = batch.on_gpu()
    slots, rows = [], []
    for r, (n, b) in enumerate(zip(new, before)):
        slots += [int(batch.table[r, p // page]) * page + p % page for p in range(b, b + n)]
    qkv = torch.randn(len(slots) + 2, (heads + 2 * kv_heads) * dim + 24, generator=batch.g) \
        * torch.exp2(torch.randint(-6, 7, (len(slots) + 2, 1), generator=batch.g).float())
    qkv = qkv.bfloat16()
    slots = slots + [-1, batch.pool * page]                           # no slot, and one that is not there
    plain_store(batch, qkv, slots)
    run_store(qkv, slots, cache, batch)
    same_cache(batch, cache)
    run_store(qkv, slots, cache, batch)                               # the same step again changes nothing
    plain_store(batch, qkv, slots)
    same_cache(batch, cache)


def test_store_of_single_tokens_until_pages_are_full():
    """Token by token, each louder than the last: the page is taken along every time."""
    batch = Batch(4, [32], 4, 2, 128, 16)
    cache = batch.on_gpu()
    for place in range(16):
        qkv = (torch.randn(1, 8 * 128, generator=batch.g) * 2.0 ** (place - 8)).bfloat16()
        slots = [int(batch.table[0, 1]) * 16 + place]
        run_store(qkv, slots, cache, batch)
        plain_store(batch, qkv, slots)
        same_cache(batch, cache)


def test_store_of_what_is_not_finite_zeros_and_the_smallest_and_largest():
    batch = Batch(5, [64], 2, 2, 64, 16)
    cache = batch.on_gpu()
    qkv = torch.randn(20, 6 * 64, generator=batch.g)
    qkv[3, 130], qkv[4, 140], qkv[5, 150] = math.inf, -math.inf, math.nan
    qkv[16:18] = 0.0
    qkv[18, 128:] *= 1e-39
    qkv[19, 128:192], qkv[19, 192:] = 3.3e38, 1e-38
    qkv = qkv.bfloat16()
    page = [int(p) for p in batch.table[0]]
    slots = [page[0] * 16 + i for i in range(16)] + [page[1] * 16, page[1] * 16 + 1, page[2] * 16 + 3, page[3] * 16]
    run_store(qkv, slots, cache, batch)
    plain_store(batch, qkv, slots)
    same_cache(batch, cache)


# ------------------------------------------------------------------------------------------------ single tokens
SIZES = [(32, 8, 128, 16), (64, 8, 128, 16), (28, 4, 128, 32), (8, 8, 128, 8), (40, 2, 128, 64), (20, 1, 128, 128), (16, 4, 64, 16),
         (6, 6, 64, 24), (4, 2, 128, 5), (100, 1, 64, 16)]


@pytest.mark.parametrize("heads, kv_heads, dim, page", SIZES)
@pytest.mark.parametrize("window", [None, 70])
def test_decode_attention(heads, kv_heads, dim, page, window):
    lengths = [1, 300, 2, 127, 128, 129]
    batch = Batch(11, lengths, heads, kv_heads, dim, page)
    positions = [n - 1 for n in lengths]
    positions[2] = -1                                                  # a padding row
    out = run_decode(batch, batch.on_gpu(), positions, dim ** -0.5, window)
    want, size = batch.decode(positions, dim ** -0.5, window)
    rows = [0, 1, 3, 4, 5]
    close(out[rows], want[rows], attention_bound(want, size)[rows])
    assert (out[2] == 7.0).all()


@pytest.mark.parametrize("heads, kv_heads, dim, page, context", [(8, 2, 128, 16, 5000), (8, 2, 64, 16, 3001), (32, 2, 128, 64, 9000),
                                                                 (4, 4, 128, 24, 2000)])
def test_decode_attention_of_a_long_context_in_many_partitions(heads, kv_heads, dim, page, context):
    from libmir_b200 import kernels
    batch = Batch(12, [context, 3], heads, kv_heads, dim, page)
    assert kernels.decode_attention_8bit_plan(2, heads, kv_heads, dim, page, context)[1] > 4
    positions = [context - 1, 2]
    for sinks in (None, torch.linspace(-3, 5, heads)):
        out = run_decode(batch, batch.on_gpu(), positions, dim ** -0.5, None, sinks)
        close(out, *with_bound(batch.decode(positions, dim ** -0.5, None, sinks)))


def with_bound(found):
    want, size = found
    return want, attention_bound(want, size)


@pytest.mark.parametrize("dim", [64, 128])
def test_decode_attention_with_loud_and_quiet_pages(dim):
    """Scales of neighbouring pages 2^40 apart, the loud page's keys hardly weighted; one page of zeros with the least scale."""
    batch = Batch(13, [400], 8, 2, dim, 16)
    batch.v.scales[:] = torch.exp2(torch.randint(-30, 10, batch.v.scales.shape, generator=batch.g).double())
    loud = int(batch.table[0, 3])
    batch.v.scales[loud] = 2.0 ** 30
    batch.k.codes[loud] = -batch.k.codes[loud].abs()
    batch.qkv[:, :8 * dim] = batch.qkv[:, :8 * dim].abs()
    for page in (4, 20):
        batch.v.codes[int(batch.table[0, page])] = 0.0
        batch.v.scales[int(batch.table[0, page])] = 2.0 ** plain.LEAST
    out = run_decode(batch, batch.on_gpu(), [399], dim ** -0.5)
    close(out, *with_bound(batch.decode([399], dim ** -0.5)))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("exponent", [-118, -70, 60, 100])
def test_decode_attention_with_values_of_extreme_scales(dim, exponent):
    """All values at one extreme scale: the weights' sum must not suffer from it (a long context: many weights near 1)."""
    batch = Batch(14, [1500], 4, 2, dim, 16)
    batch.v.scales[:] = 2.0 ** exponent
    batch.k.scales *= 2.0 ** -6                                         # flat weights
    out = run_decode(batch, batch.on_gpu(), [1499], dim ** -0.5)
    want, size = batch.decode([1499], dim ** -0.5)
    close(out, want, attention_bound(want, size) + 2.0 ** -133)


@pytest.mark.parametrize("dim", [64, 128])
def test_decode_attention_peaks_and_queries_of_all_sizes(dim):
    """Scores up to some hundreds (one key takes it all) and a query of zeros (all keys weigh the same)."""
    batch = Batch(15, [700, 700, 700], 4, 2, dim, 16)
    batch.qkv[0] *= 60.0
    batch.qkv[1] *= 0.0
    batch.qkv[2] *= 1e-6
    batch.k.scales *= 0.25
    out = run_decode(batch, batch.on_gpu(), [699] * 3, dim ** -0.5)
    want, size = batch.decode([699] * 3, dim ** -0.5)
    # row 0: scores of some hundreds, 32-bit sums of 128 products: 2^-24 of their magnitudes times a few
    magnitude = (batch.qkv[0, :4 * dim].double().abs().sum() * batch.k.values().abs().max() * dim ** -0.5)
    bound = attention_bound(want, size)
    bound[0] += size[0] * float(magnitude) * 2.0 ** -22
    close(out, want, bound)


@pytest.mark.parametrize("dim", [64, 128])
def test_decode_attention_hides_missing_pages_and_what_lies_there(dim):
    """Entries of -1 and beyond the pool, and a table that ends before the context: those keys are not seen, and a row that
    has no page at all gives zeros.  NaN codes behind the context and in unused pages change nothing."""
    batch = Batch(16, [290, 290, 290], 8, 4, dim, 16)
    batch.table[0, 5], batch.table[0, 9] = -1, batch.pool
    batch.table[0, 17:] = -1
    batch.table[1, :] = -1
    used = {int(p) for p in batch.table.flatten()}
    for page in range(batch.pool):
        if page not in used:
            batch.k.codes[page], batch.v.codes[page] = math.nan, math.nan
    last = int(batch.table[2, 18])
    batch.k.codes[last, 2:], batch.v.codes[last, 2:] = math.nan, math.nan
    batch.k.scales[last + 1 if last + 1 < batch.pool else 0] = 1.0
    cache = batch.on_gpu()
    positions = [289, 289, 289]
    want, size = batch.decode(positions, dim ** -0.5)
    for table in (batch.table, batch.table[:, :19].contiguous()):
        out = run_decode(batch, cache, positions, dim ** -0.5, table=table.cuda())
        assert (out[1] == 0).all()
        close(out, want, attention_bound(want, size))


@pytest.mark.parametrize("heads, kv_heads, rows, longest", [(32, 8, 90, 300), (16, 16, 70, 130), (20, 1, 600, 260), (8, 8, 150, 500)])
def test_decode_attention_of_many_short_contexts(heads, kv_heads, rows, longest):
    """More requests and kv heads than CTAs, each of one to four tiles of keys: every CTA takes several, and parts of some.
    More rows than a CTA keeps positions of; padding rows anywhere."""
    from libmir_b200 import kernels
    g = seeded(rows)
    lengths = torch.randint(1, longest + 1, (rows,), generator=g).tolist()
    batch = Batch(19, lengths, heads, kv_heads, 128, 16)
    positions = [n - 1 if i % 7 else -1 for i, n in enumerate(lengths)]
    out = run_decode(batch, batch.on_gpu(), positions, 0.09)
    picked = [i for i in range(rows) if i % (rows // 30) == 0 and positions[i] >= 0]
    some = [positions[i] if i in picked else -1 for i in range(rows)]
    want, size = batch.decode(some, 0.09)
    close(out[picked], want[picked], attention_bound(want, size)[picked])
    padding = [i for i in range(rows) if positions[i] < 0]
    assert (out[padding] == 7.0).all()
    assert kernels.eight_bit_error() == 0


def test_decode_attention_of_a_context_longer_than_its_table_reads_what_is_there():
    batch = Batch(17, [64], 8, 2, 128, 16)
    out = run_decode(batch, batch.on_gpu(), [1000], 0.1)
    close(out, *with_bound(batch.decode([1000], 0.1)))


def test_decode_attention_with_a_plan_for_a_longer_context_and_strided_rows():
    batch = Batch(18, [40, 700], 32, 8, 128, 16)
    wide = torch.zeros(2, batch.qkv.shape[1] + 64, dtype=torch.bfloat16, device="cuda")
    wide[:, :batch.qkv.shape[1]] = batch.qkv[:2].cuda()
    want, bound = with_bound(batch.decode([39, 699], 0.09))
    for longest in (700, 20000):
        close(run_decode(batch, batch.on_gpu(), [39, 699], 0.09, plan_context=longest, qkv=wide), want, bound)


# ------------------------------------------------------------------------------------------------ portions
@pytest.mark.parametrize("heads, kv_heads, dim, page", SIZES)
@pytest.mark.parametrize("window", [None, 50])
def test_prefill_attention(heads, kv_heads, dim, page, window):
    new, lengths = [1, 70, 3, 129], [1, 100, 203, 129]
    batch = Batch(21, lengths, heads, kv_heads, dim, page)
    sinks = torch.linspace(-2, 3, heads) if window else None
    out = run_prefill(batch, batch.on_gpu(), new, dim ** -0.5, window, sinks, extra=3)
    want, size = batch.prefill(new, dim ** -0.5, window, sinks)
    close(out[:sum(new)], want, attention_bound(want, size))
    assert (out[sum(new):] == 7.0).all()                               # rows that no request has


@pytest.mark.parametrize("heads, kv_heads, dim, page, new, lengths", [
    (4, 2, 128, 16, [300], [300]), (2, 1, 128, 128, [257, 40], [700, 1000]), (4, 4, 64, 16, [200], [450]),
    (4, 1, 128, 32, [5], [1500]), (2, 2, 128, 16, [0, 33, 0], [0, 90, 17]), (2, 1, 128, 8, [130, 130], [260, 131])])
def test_prefill_attention_of_longer_portions(heads, kv_heads, dim, page, new, lengths):
    batch = Batch(22, lengths, heads, kv_heads, dim, page)
    out = run_prefill(batch, batch.on_gpu(), new, dim ** -0.5)
    close(out, *with_bound(batch.prefill(new, dim ** -0.5)))
    out = run_prefill(batch, batch.on_gpu(), new, dim ** -0.5, max_context=max(lengths),
                      alloc=lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda"))
    close(out, *with_bound(batch.prefill(new, dim ** -0.5)))


@pytest.mark.parametrize("dim", [64, 128])
def test_prefill_attention_with_loud_pages_missing_pages_and_rows_that_see_nothing(dim):
    batch = Batch(23, [200, 150, 60], 4, 2, dim, 16)
    batch.v.scales[:] = torch.exp2(torch.randint(-30, 30, batch.v.scales.shape, generator=batch.g).double())
    batch.k.scales[int(batch.table[0, 2])] *= 2.0 ** 6
    batch.table[0, 4], batch.table[0, 7], batch.table[1, 0], batch.table[2, :] = -1, batch.pool + 5, -1, -1
    used = {int(p) for p in batch.table.flatten()}
    for page in range(batch.pool):
        if page not in used:
            batch.k.codes[page], batch.v.codes[page] = math.nan, math.nan
    last = int(batch.table[0, 12])
    batch.k.codes[last, 8:], batch.v.codes[last, 8:] = math.nan, math.nan
    new = [140, 150, 60]
    out = run_prefill(batch, batch.on_gpu(), new, dim ** -0.5)
    want, size = batch.prefill(new, dim ** -0.5)
    close(out, want, attention_bound(want, size))
    assert (out[140:156] == 0).all() and (out[290:] == 0).all()


# ------------------------------------------------------------------------------------------------ products
def product_bound(x, weight, out_dtype, extra):
    """Of sums of exact products in 32 bits (see the head of this file)."""
    size = plain.rounded_rows(x).abs() @ weight.abs().t() + extra.abs()
    terms = 128 + 2 * -(-x.shape[1] // 128) + 4
    return lambda want: size * terms * 2.0 ** -24 + want.abs() * (2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -24) + 1e-35


@pytest.mark.parametrize("m, k, n", [(1, 128, 128), (1, 16, 1), (2, 4096, 200), (7, 144, 333), (8, 2560, 1024), (17, 1040, 129),
                                     (33, 4048, 257), (64, 512, 512), (65, 512, 640), (128, 272, 384), (130, 384, 255), (300, 1024, 520)])
@pytest.mark.parametrize("form", ["bfloat16", "float32 bias", "accumulate", "bfloat16 bias strided"])
def test_linear(m, k, n, form):
    from libmir_b200 import kernels
    g = seeded(m * 1000 + n)
    x = torch.randn(m, k, generator=g)
    x[:, ::37] *= 30.0
    x[0, :min(k, 128)] = 0.0                                           # a block of zeros
    x = x.bfloat16()
    codes = (torch.randn(n, k, generator=g) * 100).clamp(-448, 448).to(E4M3)
    scales = torch.rand(-(-n // 128), -(-k // 128), generator=g) * 1e-3 + 1e-5
    scales[0, 0] *= -1.0
    weight = plain.weight_values(codes, scales)
    dtype = torch.bfloat16 if form.startswith("bfloat16") else torch.float32
    bias = (torch.randn(n, generator=g) * 3).to(dtype) if "bias" in form else None
    start = torch.randn(m, n, generator=g).to(dtype)
    if "strided" in form:
        buffer = torch.full((m, n + 13), 5.0, dtype=dtype, device="cuda")
        out = buffer[:, :n]
        xs = torch.zeros(m, k + 8, dtype=torch.bfloat16, device="cuda")
        xs[:, :k] = x.cuda()
        xs = xs[:, :k]
    else:
        out, xs = start.cuda(), x.cuda()
    kernels.linear_8bit(xs, codes.cuda(), scales.cuda(), out, None if bias is None else bias.cuda(), accumulate=form == "accumulate")
    extra = torch.zeros(1, dtype=torch.float64) if bias is None else bias.double()[None]
    if form == "accumulate":
        extra = start.double()
    want = plain.rounded_rows(x) @ weight.t() + extra
    close(out, want, product_bound(x, weight, dtype, extra)(want), form)
    if "strided" in form:
        assert (buffer[:, n:] == 5.0).all()


def test_linear_of_extreme_rows():
    """Rows of the smallest and largest numbers, infinities (448 times the scale) and NaN (that row alone)."""
    from libmir_b200 import kernels
    g = seeded(5)
    x = torch.randn(6, 256, generator=g)
    x[1] *= 1e-37
    x[2] *= 1e30
    x[3, 7] = math.inf
    x[4, 200] = math.nan
    x[5] = 0.0
    x = x.bfloat16()
    codes = (torch.randn(130, 256, generator=g) * 100).clamp(-448, 448).to(E4M3)
    scales = torch.rand(2, 2, generator=g) * 1e-3
    out = torch.empty(6, 130, device="cuda")
    kernels.linear_8bit(x.cuda(), codes.cuda(), scales.cuda(), out)
    weight = plain.weight_values(codes, scales)
    finite = torch.where(x.isnan(), torch.zeros_like(x), x)
    want = plain.rounded_rows(finite) @ weight.t()
    rows = [0, 1, 2, 3, 5]
    assert out[4].isnan().all()
    # (row 1: what is below 2^-127 of the block of tiny numbers is lost to the least scale's grid, 2^-128 a term)
    bound = product_bound(finite, weight, torch.float32, torch.zeros(1, dtype=torch.float64))(want)
    close(out[rows], want[rows], bound[rows])


@pytest.mark.parametrize("rows, columns", [(128, 128), (1, 16), (200, 300), (257, 144)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_weight(rows, columns, dtype):
    from libmir_b200 import kernels
    weight = (torch.randn(rows, columns, generator=seeded(rows)) * 0.02).to(dtype)
    weight[0, :] = 0.0
    codes, scales = kernels.quantize_weight_8bit(weight.cuda())
    assert codes.shape == (rows, columns) and scales.shape == (-(-rows // 128), -(-columns // 128))
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            block = weight[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128].float()
            scale = block.abs().max() / 448.0 if block.abs().max() > 0 else torch.tensor(1.0)
            assert scales[i, j].cpu() == scale
            want = (block / scale).clamp(-448, 448).to(E4M3).float()
            assert torch.equal(codes[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128].cpu().float(), want)
