"""Measured calls of the operators for serving in 8 bits: the product with 8-bit weights, the write into an 8-bit cache, and
attention over that cache for single tokens and for portions of prompts.

The cache holds e4m3 numbers in pages of `page` tokens, [pages * page, kv_heads, head_dim], and one 32-bit scale, a power of
two, per page and kv head; weights are e4m3 with one 32-bit scale per block of 128 x 128, and activations are rounded to e4m3
with a power of two per row and 128 columns on their way in.  `own` False computes every operator from elementary torch
operations in 32 bits, True calls libmir_b200.kernels."""

import math

import torch

own = False

LARGEST = 448.0             # of e4m3
LEAST_EXPONENT = -118       # of a scale
BLOCK = 128                 # of rows and columns of a weight's scales, and of columns of an activation's


def listed():
    return [
        # one token through the output projection of a 2,560-wide model: latency alone
        {"name": "linear one token", "op": "linear", "tokens": 1, "k": 2560, "n": 2560, "out": "bfloat16", "bias": False},
        # a decode step of 8 requests, packed gate and up projection of the same model: bound by the weights' bytes
        {"name": "linear decode 8", "op": "linear", "tokens": 8, "k": 2560, "n": 19456, "out": "bfloat16", "bias": False},
        # a short portion into a 32-bit result with a bias and sizes that fill no tile
        {"name": "linear odd", "op": "linear", "tokens": 37, "k": 4048, "n": 4001, "out": "float32", "bias": True},
        # a prompt of 2,048 through the packed q, k, v projection of a 4,096-wide model
        {"name": "linear prompt 2048", "op": "linear", "tokens": 2048, "k": 4096, "n": 6144, "out": "bfloat16", "bias": False},
        # the largest product of a 5,120-wide model, a step full of prompt tokens
        {"name": "linear prompt 4096", "op": "linear", "tokens": 4096, "k": 5120, "n": 25600, "out": "bfloat16", "bias": False},
        # one new token for each of 8 requests, somewhere inside a page
        {"name": "store decode 8", "op": "store", "requests": 8, "new": 1, "before": 1000, "ragged": True, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "scattered": True},
        # portions of three prompts that begin and end inside pages
        {"name": "store prompts 4000", "op": "store", "requests": 3, "new": 2001, "before": 333, "ragged": True, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "scattered": False},
        # one request in the middle of a chat
        {"name": "decode 1 of 1000", "op": "decode", "requests": 1, "context": 1000, "ragged": False, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "window": 0, "scattered": False},
        # the batch of a busy server, pages anywhere in the pool
        {"name": "decode 64 of 2048", "op": "decode", "requests": 64, "context": 2048, "ragged": True, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "window": 0, "scattered": True},
        # few requests with long documents
        {"name": "decode 4 of 32768", "op": "decode", "requests": 4, "context": 32768, "ragged": True, "heads": 64, "kv_heads": 8,
         "head_dim": 128, "page": 16, "window": 0, "scattered": False},
        # whole prompts of different lengths, packed
        {"name": "prompts 3 of 2048", "op": "prefill", "requests": 3, "new": 2048, "before": 0, "ragged": True, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "window": 0, "scattered": False},
        # a portion of a long prompt, its earlier portions in the cache
        {"name": "portion 512 at 16384", "op": "prefill", "requests": 1, "new": 512, "before": 16001, "ragged": False, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 16, "window": 0, "scattered": True},
    ]


HEADS = ((32, 8, 128), (64, 8, 128), (28, 4, 128), (16, 16, 128), (16, 4, 64), (32, 2, 128))


def spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("linear", "store", "decode", "prefill"))
    if op == "linear":
        case = {"op": op, "tokens": spread(rng, 1, 4096), "k": 16 * spread(rng, 8, 640), "n": spread(rng, 64, 25600),
                "out": rng.choice(("bfloat16", "float32")), "bias": rng.random() < 0.3}
        while case["tokens"] * case["k"] * case["n"] > 4096 * 5120 * 25600:
            case["tokens"] = max(1, case["tokens"] // 2)
        return case
    heads, kv_heads, head_dim = rng.choice(HEADS)
    case = {"op": op, "requests": spread(rng, 1, 64), "ragged": rng.random() < 0.7, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": rng.choice((8, 16, 16, 32, 64, 128)), "scattered": rng.random() < 0.5}
    if op == "store":
        case.update(new=1 if rng.random() < 0.4 else spread(rng, 1, 2048), before=rng.choice((0, spread(rng, 1, 4096))))
        while case["requests"] * (case["new"] + case["before"]) > 32768:
            case["requests"] = max(1, case["requests"] // 2)
            case["before"] //= 2
    elif op == "decode":
        case.update(context=spread(rng, 1, 32768), window=rng.choice((0, 0, 0, 256, 4096)))
        while case["requests"] * case["context"] * kv_heads > 131072 * 8:
            case["requests"] = max(1, case["requests"] // 2)
            case["context"] = max(1, case["context"] * 3 // 4)
    else:
        case.update(requests=spread(rng, 1, 12), new=spread(rng, 2, 2048), before=rng.choice((0, 0, spread(rng, 1, 16384))),
                    window=rng.choice((0, 0, 0, 256, 1000)))
        while case["requests"] * case["new"] * (case["new"] + case["before"]) * heads > 512 * 16513 * 32:
            case["requests"] = max(1, case["requests"] // 2)
            case["new"] = max(2, case["new"] * 3 // 4)
            case["before"] = case["before"] * 3 // 4
    return case


# ------------------------------------------------------------------------------------------------ sizes
def lengths(case):
    """(new tokens, cached tokens after them) of each request; `ragged`: down to half of the longest."""
    count = case["requests"]
    share = [1.0 - 0.5 * (i * 7 % count) / count if case["ragged"] else 1.0 for i in range(count)]
    if case["op"] == "decode":
        return [1] * count, [max(1, int(case["context"] * s)) for s in share]
    new = [max(1, int(case["new"] * s)) for s in share]
    return new, [n + int(case["before"] * s) for n, s in zip(new, share)]


def visible_pairs(case):
    """Pairs of a query and a key that it sees, and keys that some query of their request sees."""
    pairs = keys = 0
    window = case["window"]
    for new, total in zip(*lengths(case)):
        for_all = new * total - new * (new - 1) // 2
        if window:
            short = max(0, min(total, window) - (total - new))          # queries that see fewer keys than a window holds
            for_all = sum(range(total - new + 1, total - new + short + 1)) + (new - short) * window
        pairs += for_all
        keys += min(total, window + new - 1) if window else total
    return pairs, keys


def work(case):
    if case["op"] == "linear":
        m, n, k = case["tokens"], case["n"], case["k"]
        scales = 4 * (-(-n // BLOCK)) * (-(-k // BLOCK))
        size = 2 if case["out"] == "bfloat16" else 4
        return {"bytes": 2 * m * k + n * k + scales + size * m * n + (size * n if case["bias"] else 0), "flops": 2 * m * n * k}
    new, total = lengths(case)
    width = case["kv_heads"] * case["head_dim"]
    if case["op"] == "store":
        tokens = sum(new)
        pages = sum(-(-t // case["page"]) - (t - n) // case["page"] for n, t in zip(new, total))
        return {"bytes": tokens * (2 * 2 * width + 2 * width + 4) + pages * 2 * 4 * case["kv_heads"], "flops": 2 * tokens * width}
    pairs, keys = visible_pairs(case)
    rows = sum(new) * case["heads"] * case["head_dim"]
    scales = 2 * 4 * case["kv_heads"] * (keys // case["page"] + len(new))
    return {"bytes": 2 * keys * width + scales + 2 * 2 * rows, "flops": 4 * pairs * case["heads"] * case["head_dim"]}


# ------------------------------------------------------------------------------------------------ the numbers of the format
def scale_exponent(largest):
    """The least e >= LEAST_EXPONENT with largest <= 448 * 2^e."""
    mantissa, exponent = torch.frexp(largest)
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    return torch.where(largest > 0, e, LEAST_EXPONENT).clamp_min(LEAST_EXPONENT)


def power(exponent, dtype=torch.float32):
    return torch.exp2(exponent.to(dtype))


def rounded(x):
    return x.clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn)


def by_blocks(x):
    """The columns of x in blocks of 128 (the last one filled up with zeros)."""
    pad = -x.shape[-1] % BLOCK
    return torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, BLOCK))


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    if case["op"] == "linear":
        m, n, k = case["tokens"], case["n"], case["k"]
        # weights as a checkpoint holds them: rounded by blocks with scales that are no powers of two
        weight = torch.empty((n, k), dtype=torch.float8_e4m3fn, device="cuda")
        scales = torch.empty((-(-n // BLOCK), -(-k // BLOCK)), device="cuda")
        scales.copy_((0.5 + torch.rand(scales.shape, generator=g, device="cuda")) * (0.1 / LARGEST))
        for first in range(0, n, 4096):
            rows = min(4096, n - first)
            weight[first:first + rows] = rounded(normal(rows, k, dtype=torch.bfloat16).float() * 110.0)
        # activations with a few loud columns
        x = normal(m, k)
        x[:, torch.randint(k, (max(1, k // 200),), generator=g, device="cuda")] *= 20.0
        dtype = getattr(torch, case["out"])
        return {"case": case, "x": x.to(torch.bfloat16), "weight": weight, "scales": scales,
                "bias": normal(n).to(dtype) if case["bias"] else None}

    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    new, total = lengths(case)
    tokens, count = sum(new), len(new)
    per_request = [-(-t // page) for t in total]
    pool = sum(per_request) + 3
    order = torch.randperm(pool, generator=g, device="cuda") if case["scattered"] else torch.arange(pool, device="cuda")
    table = torch.full((count, max(per_request)), -1, dtype=torch.int32)
    order = order.cpu().to(torch.int32)
    at = 0
    for r, pages in enumerate(per_request):
        table[r, :pages] = order[at:at + pages]
        at += pages
    row_of = torch.repeat_interleave(torch.arange(count), torch.tensor(new))
    positions = torch.cat([torch.arange(t - n, t) for n, t in zip(new, total)])
    slots = table[row_of, positions // page].long() * page + positions % page
    # the cached keys and values: a loud channel here and there, pages louder than others
    channel = 1.0 + 7.0 * (torch.rand((2, kv_heads, dim), generator=g, device="cuda") < 0.03)
    pages, scales = [], []
    for which in range(2):
        loud = torch.exp2(normal(pool, 1, kv_heads, 1) * 0.7)
        values = normal(pool, page, kv_heads, dim, dtype=torch.bfloat16) * channel[which] * loud
        e = scale_exponent(values.abs().amax(dim=(1, 3)))
        pages.append(rounded(values * power(-e)[:, None, :, None]).view(pool * page, kv_heads, dim))
        scales.append(power(e))
    qkv = normal(tokens + (2 if case["op"] == "store" else 0), (heads + 2 * kv_heads) * dim)
    if case["op"] == "store":
        # behind the step's tokens two rows without a slot, as a padded batch has them
        qkv[:, heads * dim:] *= channel.flatten()
        slots = torch.cat([slots, torch.tensor([-1, -1])])
    state = {"case": case, "qkv": qkv.to(torch.bfloat16), "k_pages": pages[0], "v_pages": pages[1], "k_scales": scales[0],
             "v_scales": scales[1], "table": table.cuda(), "slots": slots.to(torch.int32).cuda(),
             "positions": positions.to(torch.int32).cuda(), "longest": max(total), "longest_new": max(new), "tokens": tokens}
    state["starts"] = torch.tensor([sum(new[:i]) for i in range(count + 1)], dtype=torch.int32, device="cuda")
    state["contexts"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"linear": run_linear, "store": run_store, "decode": run_decode, "prefill": run_prefill}[state["case"]["op"]](state)


def run_linear(state):
    x, weight, scales, bias = state["x"], state["weight"], state["scales"], state["bias"]
    dtype = getattr(torch, state["case"]["out"])
    if own:
        from libmir_b200 import kernels
        out = torch.empty((x.shape[0], weight.shape[0]), dtype=dtype, device=x.device)
        kernels.linear_8bit(x, weight, scales, out, bias)
        return out
    blocks = by_blocks(x.float())
    e = scale_exponent(blocks.abs().amax(dim=-1, keepdim=True))
    taken = (rounded(blocks * power(-e)).float() * power(e)).flatten(1)[:, :x.shape[1]]
    spread_scales = scales.repeat_interleave(BLOCK, 0)[:weight.shape[0]].repeat_interleave(BLOCK, 1)[:, :weight.shape[1]]
    result = taken @ (weight.float() * spread_scales).t()
    if bias is not None:
        result = result + bias.float()
    return result.to(dtype)


def run_store(state):
    case, qkv, slots = state["case"], state["qkv"], state["slots"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    if own:
        from libmir_b200 import kernels
        kernels.store_kv_8bit(qkv, slots, state["k_pages"], state["v_pages"], state["k_scales"], state["v_scales"], page, heads,
                              kv_heads, dim)
    else:
        k = qkv[:, heads * dim:(heads + kv_heads) * dim].unflatten(1, (kv_heads, dim)).float()
        v = qkv[:, (heads + kv_heads) * dim:].unflatten(1, (kv_heads, dim)).float()
        store_plain(k, slots.long(), state["k_pages"], state["k_scales"], page)
        store_plain(v, slots.long(), state["v_pages"], state["v_scales"], page)
    return {"k": state["k_pages"], "v": state["v_pages"], "k_scales": state["k_scales"], "v_scales": state["v_scales"]}


def store_plain(x, slots, pages, scales, page):
    count = scales.shape[0]
    # rows without a slot go to a page behind the last
    page_of = torch.where(slots >= 0, slots // page, count)
    place = torch.where(slots >= 0, slots % page, 0)
    size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(dim=-1)
    largest = torch.zeros((count + 1, x.shape[1]), device=x.device).index_reduce_(0, page_of, size, "amax")[:count]
    first = torch.full((count + 1,), page, device=x.device).index_reduce_(0, page_of, place, "amin")[:count, None]
    before = torch.where(scales > 0, torch.frexp(scales)[1] - 1, LEAST_EXPONENT)
    e = torch.where(first == 0, scale_exponent(largest), torch.maximum(before, scale_exponent(largest)))
    e = torch.where(first == page, before, e)
    again = torch.where(first == 0, 0, before - e)                           # what is there already is taken to the new scale
    held = pages.view(count, page, *pages.shape[1:]).float() * power(again)[:, None, :, None]
    codes = torch.cat([held.flatten(0, 1), torch.zeros_like(held[0])])
    put = torch.where(slots >= 0, slots, pages.shape[0])
    all_e = torch.cat([e, torch.zeros_like(e[:1])])
    codes[put] = (x * power(-all_e[page_of])[..., None]).clamp(-LARGEST, LARGEST)
    pages.copy_(codes[:pages.shape[0]].to(torch.float8_e4m3fn))
    scales.copy_(torch.where(first == page, scales, power(e)))


def gathered(state, which):
    """The cached keys or values of every request in 32 bits, [requests, longest, kv_heads, head_dim]."""
    page = state["case"]["page"]
    at = torch.arange(state["longest"], device="cuda")
    page_of = state["table"].long()[:, at // page].clamp_min(0)
    rows = state[which + "_pages"].view(torch.uint8)[page_of * page + at % page].view(torch.float8_e4m3fn)
    return rows.float() * state[which + "_scales"][page_of][..., None]


def attend_plain(state, q, positions):
    """q [requests, queries, heads, head_dim], positions [requests, queries] (below 0: a row that is not there)."""
    case = state["case"]
    group = case["heads"] // case["kv_heads"]
    k, v = gathered(state, "k"), gathered(state, "v")
    grouped = q.unflatten(2, (case["kv_heads"], group)).permute(0, 2, 3, 1, 4).flatten(2, 3)          # [r, kv, group * queries, d]
    scores = (grouped @ k.permute(0, 2, 3, 1)) / math.sqrt(case["head_dim"])
    at = torch.arange(state["longest"], device="cuda")
    hidden = at > positions[..., None]
    if case["window"]:
        hidden = hidden | (at <= positions[..., None] - case["window"])
    scores = scores.unflatten(2, (group, -1)).masked_fill_(hidden[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(dim=-1, keepdim=True)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    mixed = (scores.flatten(2, 3) @ v.transpose(1, 2)).unflatten(2, (group, -1)) / total
    return mixed.permute(0, 3, 1, 2, 4).flatten(2)                          # [requests, queries, heads * head_dim]


def run_decode(state):
    case, qkv = state["case"], state["qkv"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    if own:
        from libmir_b200 import kernels
        rows = case["requests"]
        partition, count, floats = kernels.decode_attention_8bit_plan(rows, heads, kv_heads, dim, case["page"], state["longest"])
        scratch = torch.empty((floats,), dtype=torch.float32, device=qkv.device) if floats else None
        out = torch.empty((rows, heads * dim), dtype=torch.bfloat16, device=qkv.device)
        kernels.decode_attention_8bit(qkv, out, state["k_pages"], state["v_pages"], state["k_scales"], state["v_scales"],
                                      state["table"], state["positions"], case["page"], heads, kv_heads, dim, 1.0 / math.sqrt(dim),
                                      case["window"] or None, partition, count, scratch)
        return out
    q = qkv[:, :heads * dim].float().unflatten(1, (heads, dim))[:, None]
    return attend_plain(state, q, state["positions"].long()[:, None])[:, 0].to(torch.bfloat16)


def run_prefill(state):
    case, qkv = state["case"], state["qkv"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    if own:
        from libmir_b200 import kernels
        out = torch.empty((state["tokens"], heads * dim), dtype=torch.bfloat16, device=qkv.device)
        kernels.prefill_attention_8bit(qkv, out, state["k_pages"], state["v_pages"], state["k_scales"], state["v_scales"],
                                       state["table"], state["starts"], state["contexts"], case["page"], heads, kv_heads, dim,
                                       1.0 / math.sqrt(dim), case["window"] or None)
        return out
    starts, contexts = state["starts"].long(), state["contexts"].long()
    new = starts[1:] - starts[:-1]
    at = torch.arange(state["longest_new"], device="cuda")
    there = at < new[:, None]
    token = torch.where(there, starts[:-1, None] + at, 0)
    # a row that is not there sees key 0, and nobody reads its result
    positions = torch.where(there, contexts[:, None] - new[:, None] + at, 0)
    q = qkv[:, :heads * dim].float().unflatten(1, (heads, dim))[token]
    mixed = attend_plain(state, q, positions).flatten(0, 1)
    request = torch.repeat_interleave(torch.arange(case["requests"], device="cuda"), new, output_size=state["tokens"])
    back = request * state["longest_new"] + torch.arange(state["tokens"], device="cuda") - starts[request]
    return mixed[back].to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "linear":
        return exact_linear(state)
    if case["op"] == "store":
        return exact_store(state)
    return exact_attention(state)


def exact_linear(state):
    x, weight = state["x"].double(), state["weight"]
    n, k = weight.shape
    result = torch.zeros((x.shape[0], n), dtype=torch.float64, device="cuda")
    for block in range(-(-k // BLOCK)):
        columns = slice(block * BLOCK, min(k, (block + 1) * BLOCK))
        part = x[:, columns]
        largest = part.abs().amax(dim=1, keepdim=True)
        e = torch.ceil(torch.log2(torch.clamp(largest, min=1e-30) / LARGEST))
        e = torch.where(largest > LARGEST * torch.exp2(e), e + 1, e)          # (the logarithm next to a border)
        e = torch.where(largest <= LARGEST * torch.exp2(e - 1), e - 1, e)
        e = torch.where(largest > 0, e, 0.0)
        codes = (part * torch.exp2(-e)).float().to(torch.float8_e4m3fn).double()
        scale = state["scales"][:, block].double().repeat_interleave(BLOCK)[:n]
        result.addmm_(codes * torch.exp2(e), (weight[:, columns].double() * scale[:, None]).t())
    if state["bias"] is not None:
        result += state["bias"].double()
    return result


def exact_store(state):
    """Page by page on the host."""
    case = state["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    slots = state["slots"].tolist()
    qkv = state["qkv"].cpu().double()
    found = {}
    for token, slot in enumerate(slots):
        if slot >= 0:
            found.setdefault(slot // page, []).append((token, slot % page))
    results = {}
    for which, offset in (("k", heads * dim), ("v", (heads + kv_heads) * dim)):
        x = qkv[:, offset:offset + kv_heads * dim].view(-1, kv_heads, dim)
        codes = state[which + "_pages"].cpu().double().view(-1, page, kv_heads, dim)
        scales = state[which + "_scales"].cpu().double()
        for b, entries in found.items():
            tokens, places = [t for t, _ in entries], [p for _, p in entries]
            largest = x[tokens].abs().amax(dim=(0, 2))
            new = torch.tensor([2.0 ** max(LEAST_EXPONENT, least_exponent(float(a))) for a in largest], dtype=torch.float64)
            if 0 not in places:
                new = torch.maximum(new, scales[b])
                codes[b] = rounded((codes[b] * (scales[b] / new)[:, None]).float()).double()
            codes[b, places] = rounded((x[tokens] / new[:, None]).float()).double()
            scales[b] = new
        results[which] = codes.flatten(0, 1)
        results[which + "_scales"] = scales
    return results


def least_exponent(largest):
    if largest == 0.0:
        return LEAST_EXPONENT
    e = math.frexp(largest)[1] - 10
    while largest > LARGEST * 2.0 ** e:
        e += 1
    return e


def exact_attention(state):
    case = state["case"]
    heads, kv_heads, dim, page, window = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["window"]
    new, total = lengths(case)
    result = torch.empty((sum(new), heads * dim), dtype=torch.float64, device="cuda")
    first = 0
    for r, (count, context) in enumerate(zip(new, total)):
        pages = state["table"][r, :-(-context // page)].long()
        k, v = ((state[w + "_pages"].view(torch.uint8).view(-1, page, kv_heads, dim)[pages].view(torch.float8_e4m3fn).double()
                 * state[w + "_scales"][pages].double()[:, None, :, None]).flatten(0, 1)[:context] for w in ("k", "v"))
        q = state["qkv"][first:first + count, :heads * dim].double().view(count, heads, dim)
        position = torch.arange(context - count, context, device="cuda")[:, None]
        key = torch.arange(context, device="cuda")
        seen = key <= position
        if window:
            seen = seen & (key > position - window)
        for h in range(heads):
            g = h // (heads // kv_heads)
            s = (q[:, h] @ k[:, g].t()) * dim ** -0.5
            p = torch.softmax(torch.where(seen, s, -math.inf), dim=1)
            result[first:first + count, h * dim:(h + 1) * dim] = p @ v[:, g]
        first += count
    return result
