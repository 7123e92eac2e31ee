"""The operators for serving in 8 bits, computed plainly in 64 bits on the CPU (the oracle of test_eight_bit*.py)."""

import math

import torch

LEAST = -118


def exponent(largest: float) -> int:
    """The least e >= -118 with largest <= 448 * 2^e."""
    if largest == 0.0:
        return LEAST
    e = math.frexp(largest)[1] - 11
    while largest > math.ldexp(448.0, e):
        e += 1
    return max(e, LEAST)


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """Rounded to nearest even to e4m3, beyond 448 to 448, as 64-bit numbers (from the format's definition)."""
    x = x.double()
    size = x.abs().clamp_max(1024.0)                                   # (infinities too; NaN stays NaN)
    step = torch.exp2(torch.floor(torch.log2(size.clamp_min(2.0 ** -20))).clamp_min(-6.0) - 3.0)
    step = torch.where(size >= 16 * step, step * 2, step)             # (a logarithm rounded down at a power of two)
    rounded = torch.round(size / step) * step                          # torch.round: halves to even
    return torch.where(x.isnan(), x, torch.copysign(rounded.clamp_max(448.0), x))


def finite_largest(x: torch.Tensor) -> float:
    x = x.double().abs()
    x = x[torch.isfinite(x)]
    return float(x.max()) if x.numel() else 0.0


class Cache:
    """Numbers and scales of keys or of values, [pages, page, kv_heads, dim] and [pages, kv_heads], in 64 bits."""

    def __init__(self, pages: int, page: int, kv_heads: int, dim: int):
        self.page = page
        self.codes = torch.zeros(pages, page, kv_heads, dim, dtype=torch.float64)
        self.scales = torch.zeros(pages, kv_heads, dtype=torch.float64)

    def store(self, x: torch.Tensor, slots) -> None:
        """x [tokens, kv_heads, dim]; a slot below 0 is no slot."""
        found = {}
        for token, slot in enumerate(slots):
            if 0 <= slot < self.codes.shape[0] * self.page:
                found.setdefault(slot // self.page, []).append((token, slot % self.page))
        for page, entries in found.items():
            tokens, places = [t for t, _ in entries], [p for _, p in entries]
            for head in range(self.codes.shape[2]):
                new = x[tokens, head].double()
                e = exponent(finite_largest(new))
                if 0 not in places:
                    scale = float(self.scales[page, head])
                    before = max(LEAST, math.frexp(scale)[1] - 1) if scale > 0 else LEAST
                    if before < e:
                        self.codes[page, :, head] = e4m3(self.codes[page, :, head] * 2.0 ** (before - e))
                    e = max(e, before)
                self.codes[page, places, head] = e4m3(new * 2.0 ** -e)
                self.scales[page, head] = 2.0 ** e

    def rows(self) -> torch.Tensor:
        return self.codes.flatten(0, 1)

    def values(self) -> torch.Tensor:
        return (self.codes * self.scales[:, None, :, None]).flatten(0, 1)


def attention(q, k_values, v_values, page: int, table, positions, scale: float, window=None, sinks=None):
    """q [queries, heads, dim] of ONE request with its block table (a list); k_values, v_values [slots, kv_heads, dim].
    The result [queries, heads, dim] and, for tolerances, the same weights applied to |v|."""
    q = q.double()
    heads, dim = q.shape[1], q.shape[2]
    pool = k_values.shape[0] // page
    out = torch.zeros_like(q)
    size = torch.zeros_like(q)
    for i, position in enumerate(positions):
        first = max(0, position - window + 1) if window else 0
        keys = [j for j in range(first, position + 1) if j // page < len(table) and 0 <= table[j // page] < pool]
        if not keys:
            continue
        rows = torch.tensor([table[j // page] * page + j % page for j in keys])
        k, v = k_values[rows], v_values[rows]                          # [keys, kv_heads, dim]
        group = heads // k.shape[1]
        for h in range(heads):
            s = (k[:, h // group] @ q[i, h]) * scale
            top = s.max()
            p = torch.exp(s - top)
            total = p.sum()
            if sinks is not None:
                total = total + torch.exp(sinks[h].double() - top)
            out[i, h] = (p @ v[:, h // group]) / total
            size[i, h] = (p @ v[:, h // group].abs()) / total
    return out, size


def rounded_rows(x: torch.Tensor) -> torch.Tensor:
    """Every row's runs of 128 columns rounded to e4m3 with a power of two."""
    x = x.double()
    out = torch.empty_like(x)
    for row in range(x.shape[0]):
        for first in range(0, x.shape[1], 128):
            part = x[row, first:first + 128]
            e = exponent(finite_largest(part))
            out[row, first:first + 128] = e4m3(part * 2.0 ** -e) * 2.0 ** e
    return out


def weight_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    n, k = codes.shape
    return codes.double() * scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
