"""The 8-bit cache's write and attention in float64 (CPU), and the bound of the attention's rounding."""

from __future__ import annotations

import torch

E4M3 = torch.float8_e4m3fn


def e4m3_round(x: torch.Tensor) -> torch.Tensor:
    """E4M3 codes of float32 values in range, by torch's conversion (ties to even); infinities are NaN."""
    return torch.where(x.isinf(), torch.nan, x).to(E4M3)


def needed_scale(largest: float) -> float:
    power = -126
    while largest > 448.0 * 2.0 ** power:
        power += 1
    return 2.0 ** power


def write(key, value, cache, scales, starts, seq_lens, table):
    """Updates ``cache`` (E4M3) and ``scales`` (float32) as the operator does; loops over pages."""
    page_tokens = cache.size(3)
    raw = cache.view(torch.uint8)
    for b in range(len(seq_lens)):
        begin, n = int(starts[b]), int(starts[b + 1] - starts[b])
        history = max(0, int(seq_lens[b]) - n)
        i = 0
        while i < n:
            page, slot = divmod(history + i, page_tokens)
            count = min(n - i, page_tokens - slot)
            block = int(table[b, page]) if page < table.size(1) else -1
            if 0 <= block < cache.size(1):
                for plane, rows in enumerate((key, value)):
                    for head in range(cache.size(2)):
                        x = rows[begin + i:begin + i + count, head].float()
                        finite = x[x.isfinite()].abs()
                        need = needed_scale(float(finite.max()) if finite.numel() else 0.0)
                        old = float(scales[plane, block, head])
                        scale = old if slot and old >= need else need
                        if slot and scale > old:
                            ratio = torch.tensor(old) / torch.tensor(scale)
                            kept = raw[plane, block, head, :slot].view(E4M3).float() * ratio
                            raw[plane, block, head, :slot] = e4m3_round(kept).view(torch.uint8)
                        raw[plane, block, head, slot:slot + count] = e4m3_round(x / scale).view(torch.uint8)
                        scales[plane, block, head] = scale
            i += count


def attend(query, key, value, cache, scales, starts, seq_lens, table, scale):
    """(output, bound) float64 [rows, heads, D]; rows of no request are NaN in both.

    The bound: one BF16 rounding of the output (2^-8 of it), and on the sum of p |v|: the
    weights' split into two BF16 parts (2^-16), the error of a score (D products summed in
    float32, the scales and the logarithm's factor: (D + 8) 2^-24 of the sum of |q k|, on
    numerator and denominator), of the exponential (2^-21) and of the sums over the tokens
    (2^-24 for each of 64 and every 16th token, numerator and denominator).
    """
    rows, heads, dim = query.shape
    kv_heads, page_tokens = key.size(1), cache.size(3)
    out = torch.full((rows, heads, dim), torch.nan, dtype=torch.float64)
    bound = out.clone()
    for b in range(len(seq_lens)):
        begin, n = int(starts[b]), int(starts[b + 1] - starts[b])
        history = min(max(0, int(seq_lens[b]) - n), table.size(1) * page_tokens)
        positions = [t for t in range(history) if 0 <= int(table[b, t // page_tokens]) < cache.size(1)]
        blocks = torch.tensor([int(table[b, t // page_tokens]) for t in positions], dtype=torch.long)
        slots = torch.tensor([t % page_tokens for t in positions], dtype=torch.long)
        for head in range(heads):
            group = head // (heads // kv_heads)
            planes = []
            for plane, new in enumerate((key, value)):
                held = cache[plane, :, group].view(torch.uint8)[blocks, slots].view(E4M3).double()
                held = held * scales[plane, blocks, group].double()[:, None]
                planes.append(torch.cat([held, new[begin:begin + n, group].double()]))
            for i in range(n):
                count = len(positions) + i + 1
                k, v = planes[0][:count], planes[1][:count]
                q = query[begin + i, head].double()
                scores = k @ q * scale
                weights = torch.exp(scores - scores.max())
                weights = torch.where(scores == -torch.inf, 0.0, weights)
                weights = weights / weights.sum()
                out[begin + i, head] = weights @ v
                size = float((k.abs() @ q.abs()).max()) * scale
                share = 2.0 ** -16 + 2 * (dim + 8) * 2.0 ** -24 * size + 2.0 ** -21 + 2 * (64 + count / 16) * 2.0 ** -24
                bound[begin + i, head] = 2.0 ** -8 * out[begin + i, head].abs() + share * (weights @ v.abs()) + 1e-37
    return out, bound
