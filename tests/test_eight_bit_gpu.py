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


# ------------------------------------------------------------------------------------------------ together, as they would be used
def test_a_generation_over_the_8bit_cache():
    """Two prompts in portions, then decoded tokens: norm and rotation in place, the cache's write, attention over it and the
    output projection with 8-bit weights, every operator against the plain one on what the GPU gave it."""
    from libmir_b200 import kernels
    heads, kv_heads, dim, page, hidden = 8, 2, 128, 16, 512
    g = seeded(31)
    lengths = [150, 37]
    steps = [[100, 37], [50, 0]] + [[1, 1]] * 20                       # tokens of each request in each step
    batch = Batch(32, [n + 20 for n in lengths], heads, kv_heads, dim, page)
    batch.k, batch.v = plain.Cache(batch.pool, page, kv_heads, dim), plain.Cache(batch.pool, page, kv_heads, dim)
    cache = batch.on_gpu()
    table = batch.table.cuda()
    weight = torch.randn(hidden, heads * dim, generator=g) * 0.03
    codes, scales = kernels.quantize_weight_8bit(weight.cuda())
    values = plain.weight_values(codes.cpu(), scales.cpu())
    inv_freq = (1e4 ** (-torch.arange(0, dim, 2).float() / dim)).cuda()
    q_norm, k_norm = (torch.rand(2, dim, generator=g) + 0.5).cuda()
    done = [0, 0]
    for counts in steps:
        positions = [p for r in range(2) for p in range(done[r], done[r] + counts[r])]
        rows = [r for r in range(2) for _ in range(counts[r])]
        slots = [int(batch.table[r, p // page]) * page + p % page for r, p in zip(rows, positions)]
        qkv = (torch.randn(len(rows), (heads + 2 * kv_heads) * dim, generator=g)).bfloat16().cuda()
        at = torch.tensor(positions, dtype=torch.int32).cuda()
        kernels.qk_rope_store(qkv, at, None, inv_freq, q_norm, k_norm, None, None, heads, kv_heads, dim, dim, 1e-6, keys_in_place=True)
        kernels.store_kv_8bit(qkv, torch.tensor(slots, dtype=torch.int32).cuda(), *cache, page, heads, kv_heads, dim)
        out = torch.empty(len(rows), heads * dim, dtype=torch.bfloat16, device="cuda")
        done = [d + c for d, c in zip(done, counts)]
        if max(counts) == 1:
            plan = kernels.decode_attention_8bit_plan(2, heads, kv_heads, dim, page, 200)
            kernels.decode_attention_8bit(qkv, out, *cache, table, at, page, heads, kv_heads, dim, 0.088, None, plan[0], plan[1],
                                          torch.empty(plan[2], device="cuda"))
        else:
            starts = torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32).cuda()
            kernels.prefill_attention_8bit(qkv, out, *cache, table, starts, torch.tensor(done, dtype=torch.int32).cuda(), page, heads,
                                           kv_heads, dim, 0.088, None)
        residual = torch.randn(len(rows), hidden, generator=g)
        result = residual.cuda()
        kernels.linear_8bit(out, codes, scales, result, accumulate=True)
        # the same, plainly
        plain_store(batch, qkv.cpu(), slots)
        same_cache(batch, cache)
        wants, sizes = [], []
        for r in range(2):
            mine = [i for i in range(len(rows)) if rows[i] == r]
            q = qkv[mine, :heads * dim].cpu().view(len(mine), heads, dim)
            o, s = plain.attention(q, batch.k.values(), batch.v.values(), page, batch.table[r].tolist(), [positions[i] for i in mine], 0.088)
            wants.append(o.flatten(1))
            sizes.append(s.flatten(1))
        want, size = torch.cat(wants), torch.cat(sizes)
        close(out, want, attention_bound(want, size))
        product = plain.rounded_rows(out.cpu()) @ values.t() + residual.double()
        close(result, product, product_bound(out.cpu(), values, torch.float32, residual.double())(product))
    assert kernels.eight_bit_error() == 0


def step_calls(batch, cache, qkv, slots, positions, table, codes, scales, out, result, scratch, plan):
    from libmir_b200 import kernels
    kernels.store_kv_8bit(qkv, slots, *cache, batch.page, batch.heads, batch.kv_heads, batch.dim)
    kernels.decode_attention_8bit(qkv, out, *cache, table, positions, batch.page, batch.heads, batch.kv_heads, batch.dim, 0.09, None,
                                  plan[0], plan[1], scratch)
    kernels.linear_8bit(out, codes, scales, result)


@pytest.mark.parametrize("dim", [64, 128])
def test_a_captured_step_replayed_for_growing_contexts(dim):
    """Two graphs of a decode step over caches of their own, replayed in turn with new positions, slots and queries, against eager
    calls: captured when contexts were short, replayed when they are long and a row has become padding."""
    from libmir_b200 import kernels
    heads, kv_heads, page, rows = 8, 2, 16, 3
    g = seeded(41)
    codes = (torch.randn(256, heads * dim, generator=g) * 100).clamp(-448, 448).to(E4M3).cuda()
    scales = (torch.rand(2, -(-heads * dim // 128), generator=g) * 1e-3).cuda()
    plan = kernels.decode_attention_8bit_plan(rows, heads, kv_heads, dim, page, 900)
    made = []
    for seed in (42, 43):
        batch = Batch(seed, [900, 700, 800], heads, kv_heads, dim, page)
        held = dict(cache=batch.on_gpu(), qkv=torch.zeros(rows, (heads + 2 * kv_heads) * dim, dtype=torch.bfloat16, device="cuda"),
                    slots=torch.full((rows,), -1, dtype=torch.int32, device="cuda"), table=batch.table.cuda(),
                    positions=torch.zeros(rows, dtype=torch.int32, device="cuda"), codes=codes, scales=scales,
                    out=torch.zeros(rows, heads * dim, dtype=torch.bfloat16, device="cuda"), result=torch.zeros(rows, 256, device="cuda"),
                    scratch=torch.empty(plan[2], device="cuda") if plan[2] else None, plan=plan)
        eager = dict(held, cache=tuple(t.clone() for t in held["cache"]), out=held["out"].clone(), result=held["result"].clone(),
                     scratch=torch.empty(plan[2], device="cuda") if plan[2] else None)
        step_calls(batch, **{**held, "cache": tuple(t.clone() for t in held["cache"])})        # (warm)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step_calls(batch, **held)
        made.append((batch, held, eager, graph))
    for positions in ([3, 0, 17], [130, 128, 255], [899, -1, 400], [512, 699, -1]):
        for batch, held, eager, graph in made:
            held["qkv"].copy_(torch.randn(held["qkv"].shape, generator=g).bfloat16())
            held["positions"].copy_(torch.tensor(positions, dtype=torch.int32))
            held["slots"].copy_(torch.tensor([int(batch.table[r, p // page]) * page + p % page if p >= 0 else -1
                                              for r, p in enumerate(positions)], dtype=torch.int32))
            graph.replay()
            step_calls(batch, **eager)
        torch.cuda.synchronize()
        for batch, held, eager, _ in made:
            for name in ("out", "result"):
                assert torch.equal(held[name], eager[name]), name
            for a, b in zip(held["cache"], eager["cache"]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert kernels.eight_bit_error() == 0


def test_calls_on_two_streams_at_once():
    """The same step on two streams, each with tensors of its own, gives what it gives alone."""
    from libmir_b200 import kernels
    heads, kv_heads, dim, page, rows = 8, 2, 128, 16, 3
    g = seeded(51)
    codes = (torch.randn(640, heads * dim, generator=g) * 100).clamp(-448, 448).to(E4M3).cuda()
    scales = (torch.rand(5, heads, generator=g) * 1e-3).cuda()
    plan = kernels.decode_attention_8bit_plan(rows, heads, kv_heads, dim, page, 3000)
    held = []
    for seed in (52, 53):
        batch = Batch(seed, [3000, 200, 1700], heads, kv_heads, dim, page)
        positions = [2999, 199, 1699]
        slots = [int(batch.table[r, p // page]) * page + p % page for r, p in enumerate(positions)]
        def state():
            return dict(cache=batch.on_gpu(), qkv=batch.qkv[:rows].cuda(), slots=torch.tensor(slots, dtype=torch.int32).cuda(),
                        table=batch.table.cuda(), positions=torch.tensor(positions, dtype=torch.int32).cuda(), codes=codes, scales=scales,
                        out=torch.zeros(rows, heads * dim, dtype=torch.bfloat16, device="cuda"), result=torch.zeros(rows, 640, device="cuda"),
                        scratch=torch.empty(plan[2], device="cuda"), plan=plan)
        held.append((batch, state(), state()))
    for batch, alone, _ in held:
        step_calls(batch, **alone)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for stream, (batch, _, both) in zip(streams, held):
            with torch.cuda.stream(stream):
                step_calls(batch, **both)
    torch.cuda.synchronize()
    for batch, alone, both in held:
        assert torch.equal(alone["out"], both["out"]) and torch.equal(alone["result"], both["result"])
    assert kernels.eight_bit_error() == 0


# ------------------------------------------------------------------------------------------------ offsets beyond 32 bits
@pytest.mark.parametrize("dim", [64, 128])
def test_pages_beyond_two_gigabytes(dim):
    """Pages at the end of a pool of more than 2^31 bytes: written and read as at its beginning."""
    from libmir_b200 import kernels
    heads, kv_heads, page = 16, 8, 16
    pool = (1 << 31) // (page * kv_heads * dim) + 5000
    batch = Batch(61, [600, 90], heads, kv_heads, dim, page)
    small = batch.on_gpu()
    shift = pool - batch.pool
    large = tuple(torch.zeros((pool * page, kv_heads, dim), dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2)) \
        + tuple(torch.zeros((pool, kv_heads), device="cuda") for _ in range(2))
    for a, b in zip(small[:2], large[:2]):
        b.view(torch.uint8)[shift * page:] = a.view(torch.uint8)
    for a, b in zip(small[2:], large[2:]):
        b[shift:] = a
    far = torch.where(batch.table >= 0, batch.table + shift, batch.table)
    qkv = batch.qkv[:40].cuda()
    for r in range(2):
        last = batch.lengths[r] - 1
        for cache, table in ((small, batch.table), (large, far)):
            slots = [int(table[r, p // page]) * page + p % page for p in range(last - 19, last + 1)]
            kernels.store_kv_8bit(qkv[r * 20:r * 20 + 20], torch.tensor(slots, dtype=torch.int32).cuda(), *cache, page, heads, kv_heads, dim)
    for a, b in zip(small[:2], large[:2]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)[shift * page:]) and not b.view(torch.uint8)[:1000].any()
    for a, b in zip(small[2:], large[2:]):
        assert torch.equal(a, b[shift:])
    positions = [599, 89]
    near = run_decode(batch, small, positions, 0.1, table=batch.table.cuda())
    assert torch.equal(near, run_decode(batch, large, positions, 0.1, table=far.cuda()))
    batch.table = far
    over = run_prefill(batch, large, [300, 50], 0.1)
    batch.table = far - shift * (far >= 0).int()
    assert torch.equal(over, run_prefill(batch, small, [300, 50], 0.1))


def test_products_beyond_two_to_the_31():
    """More than 2^31 elements of x and of the result: the last rows are right."""
    from libmir_b200 import kernels
    g = seeded(71)
    m, k, n = 70000, 32768, 136
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, k, generator=g).bfloat16().cuda()
    codes = (torch.randn(n, k, generator=g) * 100).clamp(-448, 448).to(E4M3)
    scales = torch.rand(2, k // 128, generator=g) * 1e-3
    weight = plain.weight_values(codes, scales)
    out = torch.full((m, n), 3.0, device="cuda")
    kernels.linear_8bit(x, codes.cuda(), scales.cuda(), out)
    want = plain.rounded_rows(x[-3:].cpu()) @ weight.t()
    close(out[-3:], want, product_bound(x[-3:].cpu(), weight, torch.float32, torch.zeros(1, dtype=torch.float64))(want))
    assert (out[:-3] == 0).all()
    del x, out
    m, k, n = 40000, 128, 60000
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.randn(k, generator=g).bfloat16().cuda()
    codes = (torch.randn(n, k, generator=g) * 100).clamp(-448, 448).to(E4M3)
    scales = torch.rand(-(-n // 128), 1, generator=g) * 1e-3
    out = torch.full((m, n), 3.0, dtype=torch.bfloat16, device="cuda")
    kernels.linear_8bit(x, codes.cuda(), scales.cuda(), out)
    weight = plain.weight_values(codes, scales)
    want = plain.rounded_rows(x[-1:].cpu()) @ weight.t()
    close(out[-1:], want, product_bound(x[-1:].cpu(), weight, torch.bfloat16, torch.zeros(1, dtype=torch.float64))(want))
    assert (out[-2] == 0).all() and (out[0] == 0).all()


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals_of_tensors_that_do_not_fit():
    from libmir_b200 import kernels
    from libmir_b200.errors import KernelError
    batch = Batch(81, [40], 4, 2, 64, 16)
    cache = batch.on_gpu()
    qkv = batch.qkv[:1].cuda()
    slots = torch.zeros(1, dtype=torch.int32).cuda()
    k, v, ks, vs = cache

    def store(**c):
        a = dict(qkv=qkv, slots=slots, k=k, v=v, ks=ks, vs=vs, page=16, heads=4, kv_heads=2, dim=64)
        a.update(c)
        kernels.store_kv_8bit(*a.values())
    store()
    for change in (dict(k=k.view(torch.uint8)), dict(v=v[:-16]), dict(ks=ks[:-1]), dict(vs=vs.double()), dict(page=7), dict(kv_heads=1),
                   dict(dim=32), dict(qkv=qkv.float()), dict(qkv=qkv[:, :-1]), dict(slots=slots.long()), dict(slots=slots[:0]),
                   dict(k=k.cpu()), dict(qkv=qkv.t().contiguous().t() if qkv.shape[0] > 1 else qkv[0])):
        with pytest.raises((KernelError, IndexError)):
            store(**change)
    table, positions = batch.table.cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    out = torch.empty(1, 256, dtype=torch.bfloat16, device="cuda")

    def decode(**c):
        plan = kernels.decode_attention_8bit_plan(1, 4, 2, 64, 16, 40)
        a = dict(qkv=qkv, out=out, k=k, v=v, ks=ks, vs=vs, table=table, positions=positions, page=16, heads=4, kv_heads=2, dim=64,
                 scale=0.1, window=None, partition=plan[0], parts=plan[1], scratch=None, sinks=None)
        a.update(c)
        kernels.decode_attention_8bit(*a.values())
    decode()
    for change in (dict(out=out.float()), dict(out=out[:, :128]), dict(table=table.long()), dict(table=table[:0]), dict(positions=positions[:0]),
                   dict(heads=3), dict(scale=0.0), dict(window=-3), dict(parts=2), dict(sinks=torch.zeros(3, device="cuda")),
                   dict(sinks=torch.zeros(4)), dict(partition=0), dict(k=k[..., :32]), dict(scratch=torch.zeros(8))):
        with pytest.raises(KernelError):
            decode(**change)
    starts, contexts = torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.tensor([40], dtype=torch.int32).cuda()

    def prefill(**c):
        a = dict(qkv=qkv, out=out, k=k, v=v, ks=ks, vs=vs, table=table, starts=starts, contexts=contexts, page=16, heads=4, kv_heads=2,
                 dim=64, scale=0.1, window=None)
        a.update(c)
        kernels.prefill_attention_8bit(*a.values())
    prefill()
    for change in (dict(starts=starts[:1]), dict(contexts=contexts.long()), dict(starts=starts.cpu()), dict(out=out[:, ::2]),
                   dict(qkv=qkv[:, 1:]), dict(scale=-1.0), dict(page=3)):
        with pytest.raises(KernelError):
            prefill(**change)
    codes, scales = torch.zeros(200, 128).to(E4M3).cuda(), torch.ones(2, 1).cuda()
    x, result = torch.zeros(3, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, 200, device="cuda")

    def linear(**c):
        a = dict(x=x, weight=codes, scales=scales, out=result, bias=None, accumulate=False)
        a.update(c)
        kernels.linear_8bit(*a.values())
    linear()
    for change in (dict(x=x.float()), dict(x=x[:, :64]), dict(weight=codes[:, :120].contiguous(), x=x[:, :120].contiguous()),
                   dict(scales=scales.t()), dict(scales=scales.double()), dict(out=result[:, :100]), dict(out=result.bfloat16(), accumulate=True),
                   dict(out=result.half()), dict(bias=torch.zeros(200, dtype=torch.bfloat16, device="cuda")), dict(bias=torch.zeros(199, device="cuda")),
                   dict(weight=codes.view(torch.uint8)), dict(x=x.cpu()), dict(weight=torch.zeros(128, 200).to(E4M3).cuda().t())):
        with pytest.raises(KernelError):
            linear(**change)
    linear(x=x[:0], out=result[:0])
    with pytest.raises(KernelError):
        kernels.quantize_weight_8bit(torch.zeros(4, 4, dtype=torch.float16, device="cuda"))


# ------------------------------------------------------------------------------------------------ numbers that are none
def close_with_nans(got, want, bound, what=""):
    """NaN exactly where the plain result is, and close elsewhere."""
    assert torch.equal(got.cpu().isnan(), want.isnan()), what
    close(got.cpu().double().nan_to_num(0.0), want.nan_to_num(0.0), bound.nan_to_num(1e-30), what)


@pytest.mark.parametrize("heads, kv_heads, dim, page", [(4, 2, 128, 16), (6, 2, 64, 16), (2, 2, 128, 12)])
@pytest.mark.parametrize("window", [None, 40])
def test_prefill_attention_shows_nan_only_to_the_queries_that_see_it(heads, kv_heads, dim, page, window):
    """NaN among the values and keys of the portions' own tokens, of the context before them and at the windows' edges; infinite and
    NaN queries."""
    new, lengths = [90, 40, 1, 150], [90, 170, 60, 150]
    batch = Batch(91, lengths, heads, kv_heads, dim, page)
    slot = lambda r, p: (int(batch.table[r, p // page]), p % page)
    for r, p, head, column in ((0, 30, 0, 5), (0, 89, 1, dim - 1), (0, 0, 1, 7), (1, 120, 0, 33), (1, 169, 1, 2), (1, 95, 1, 60),
                               (2, 59, 0, 1), (3, 128, 1, 9), (3, 127, 1, 8), (3, 3, 0, 4)):
        at, place = slot(r, p)
        batch.v.codes[at, place, head, column] = math.nan
    at, place = slot(0, 60)
    batch.k.codes[at, place, 0, 3] = math.nan                          # that head's queries from there on see it
    batch.qkv[10, 5], batch.qkv[20, dim + 3], batch.qkv[95, 1], batch.qkv[131, 0] = math.inf, math.nan, -math.inf, math.nan
    out = run_prefill(batch, batch.on_gpu(), new, dim ** -0.5, window)
    want, size = batch.prefill(new, dim ** -0.5, window)
    assert want.isnan().any() and not want.isnan().all()
    close_with_nans(out, want, attention_bound(want, size))


@pytest.mark.parametrize("heads, kv_heads, dim, page", [(4, 2, 128, 16), (6, 2, 64, 16), (20, 1, 128, 32)])
@pytest.mark.parametrize("window", [None, 40])
def test_decode_attention_shows_nan_only_to_the_rows_that_see_it(heads, kv_heads, dim, page, window):
    lengths = [300, 200, 500, 77, 1]
    batch = Batch(92, lengths, heads, kv_heads, dim, page)
    slot = lambda r, p: (int(batch.table[r, p // page]), p % page)
    for r, p, head, column in ((0, 299, 0, 5), (0, 258, 0, 6), (0, 261, kv_heads - 1, 7), (0, 260, 0, 8), (2, 100, 0, 1)):
        at, place = slot(r, p)
        batch.v.codes[at, place, head, column] = math.nan
    at, place = slot(3, 76)
    batch.k.codes[at, place, 0, 3] = math.nan
    batch.qkv[1, 5], batch.qkv[4, dim + 3] = math.inf, math.nan
    positions = [n - 1 for n in lengths]
    out = run_decode(batch, batch.on_gpu(), positions, dim ** -0.5, window)
    want, size = batch.decode(positions, dim ** -0.5, window)
    assert want.isnan().any() and not want.isnan().all()
    close_with_nans(out, want, attention_bound(want, size))


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_zero_queries_over_zero_keys(dim):
    """The least scales on both sides (their product is no 32-bit number): every visible key weighs the same."""
    batch = Batch(93, [70, 200], 4, 2, dim, 16)
    batch.k.codes[:], batch.k.scales[:] = 0.0, 2.0 ** -118
    batch.qkv[:, :4 * dim] = 0.0
    cache = batch.on_gpu()
    for scale in (0.1, 1e-12):
        close(run_decode(batch, cache, [69, 150], scale), *with_bound(batch.decode([69, 150], scale)))
        close(run_prefill(batch, cache, [30, 140], scale), *with_bound(batch.prefill([30, 140], scale)))


@pytest.mark.parametrize("dim", [64, 128])
def test_prefill_attention_ends_with_its_rows(dim):
    """Query starts beyond the rows there are: what has a row is worked out, nothing else is written."""
    from libmir_b200 import kernels
    batch = Batch(94, [60, 50], 4, 2, dim, 16)
    cache = batch.on_gpu()
    out = torch.full((60, 4 * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    starts, contexts = torch.tensor([0, 20, 75], dtype=torch.int32).cuda(), torch.tensor([60, 50], dtype=torch.int32).cuda()
    kernels.prefill_attention_8bit(batch.qkv[:40].cuda(), out[:40], *cache, batch.table.cuda(), starts, contexts, 16, 4, 2, dim, 0.1, None)
    want, bound = with_bound(batch.prefill([20, 20], 0.1))
    close(out[:40], want, bound)
    assert (out[40:] == 7.0).all()


def test_linear_of_a_long_row_with_few_parts():
    """A forced cut that would leave a CTA more blocks than it holds is made finer."""
    from libmir_b200 import kernels
    from libmir_b200.kernels.eight_bit import set_linear_8bit_splits
    g = seeded(95)
    for m in (3, 20):
        k, n = 128 * 170, 200
        x = torch.randn(m, k, generator=g).bfloat16()
        codes = (torch.randn(n, k, generator=g) * 100).clamp(-448, 448).to(E4M3)
        scales = torch.rand(2, k // 128, generator=g) * 1e-3
        weight = plain.weight_values(codes, scales)
        want = plain.rounded_rows(x) @ weight.t()
        bound = product_bound(x, weight, torch.float32, torch.zeros(1, dtype=torch.float64))(want)
        for splits in (1, 2, 4, 8, 0):
            set_linear_8bit_splits(splits)
            try:
                out = torch.zeros(m, n, device="cuda")
                kernels.linear_8bit(x.cuda(), codes.cuda(), scales.cuda(), out)
            finally:
                set_linear_8bit_splits(0)
            close(out, want, bound, f"{m} rows, {splits}")
    assert kernels.eight_bit_error() == 0


@pytest.mark.parametrize("dim, page, kv_heads, new, before", [
    (128, 256, 3, [400, 1], [100, 200]), (64, 24, 3, [2, 290, 1], [23, 7, 40]), (128, 16, 5, [1] * 700, [3, 15, 16, 31] * 175),
    (64, 130, 2, [1030, 5], [129, 3]), (128, 64, 2, [1] * 300, list(range(300)))])
def test_store_of_long_pages_and_many_tokens(dim, page, kv_heads, new, before):
    """Pages of more rows than a warp or a block holds, found and shared in each of the ways; later tokens louder than the page."""
    lengths = [n + b for n, b in zip(new, before)]
    batch = Batch(97, lengths, 4, kv_heads, dim, page)
    cache = batch.on_gpu()
    slots = [int(batch.table[r, p // page]) * page + p % page for r, (n, b) in enumerate(zip(new, before)) for p in range(b, b + n)]
    for loud in (0, 4):
        qkv = (torch.randn(len(slots), (4 + 2 * kv_heads) * dim, generator=batch.g)
               * torch.exp2(torch.randint(-6, 7, (len(slots), 1), generator=batch.g).float() + loud)).bfloat16()
        plain_store(batch, qkv, slots)
        run_store(qkv, slots, cache, batch)
        same_cache(batch, cache)


@pytest.mark.parametrize("dim", [64, 128])
def test_prefill_attention_of_many_short_portions(dim):
    """More requests than a warp looks at together, of no, one and a few tokens."""
    g = seeded(98)
    lengths = torch.randint(1, 60, (150,), generator=g).tolist()
    new = [min(n, int(c)) for n, c in zip(lengths, torch.randint(0, 40, (150,), generator=g))]
    batch = Batch(98, lengths, 4, 2, dim, 16)
    out = run_prefill(batch, batch.on_gpu(), new, 0.1, extra=2)
    want, bound = with_bound(batch.prefill(new, 0.1))
    close(out[:sum(new)], want, bound)
    assert (out[sum(new):] == 7.0).all()


@pytest.mark.parametrize("heads, kv_heads, dim, page", [(8, 2, 128, 16), (8, 2, 64, 16), (8, 2, 128, 24)])
def test_decode_attention_at_positions_far_beyond_the_table(heads, kv_heads, dim, page):
    batch = Batch(99, [96, 96, 96], heads, kv_heads, dim, page)
    want, bound = with_bound(batch.decode([95, 95, 95], 0.1))
    close(run_decode(batch, batch.on_gpu(), [95, 2 ** 31 - 1, 2 ** 31 - 2], 0.1, plan_context=2 ** 20), want, bound)
