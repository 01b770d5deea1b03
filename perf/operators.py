"""Operators of a decode step with an 8-bit cache and 4-bit weights, as cases that can be timed and compared.

Four kinds, each through the package's public entry points where ``own`` is
true and in elementary torch operations where it is not:

- ``attend``: attention over a paged cache held in 8 bits (E4M3) with one
  scale per page and head (``paged_attention_fp8``): one new row per request,
  a few, or a prompt chunk, causal among the new rows;
- ``write``: a call's new K/V tokens written into such a cache
  (``quantize_fp8``): pages that gain a larger value get a larger scale, and
  the codes they hold are rounded again;
- ``project``: a projection with 4-bit weights and group scales
  (``linear_rows_int4``);
- ``logprobs``: log probabilities of given tokens, the entropy and the top
  alternatives of logits (``token_logprobs``).

``exact`` restates each in float64.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = torch.device("cuda:0")
E4M3_MAX = 448.0


def listed():
    return [
        # One user's next token on a short conversation: launches and latency.
        {"name": "attend_single", "kind": "attend", "batch": 1, "shortest": 2047, "longest": 2047, "rows": 1,
         "ragged": False, "mix": 0, "heads": 16, "kv_heads": 16, "dim": 128, "page": 16},
        # The headline batch: 32 requests of 8192 tokens, 16 heads of 128 channels.
        {"name": "attend_batch", "kind": "attend", "batch": 32, "shortest": 8192, "longest": 8192, "rows": 1,
         "ragged": False, "mix": 0, "heads": 16, "kv_heads": 16, "dim": 128, "page": 16},
        # A serving batch as it really is, heads in groups of four.
        {"name": "attend_grouped", "kind": "attend", "batch": 24, "shortest": 0, "longest": 8000, "rows": 1,
         "ragged": False, "mix": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32},
        # 55 heads of 96 channels, a few draft rows to verify for some of the requests.
        {"name": "attend_drafts", "kind": "attend", "batch": 8, "shortest": 1001, "longest": 4096, "rows": 5,
         "ragged": True, "mix": 2, "heads": 55, "kv_heads": 55, "dim": 96, "page": 16},
        # The next chunk of two long prompts over their cached prefixes.
        {"name": "attend_chunk", "kind": "attend", "batch": 2, "shortest": 2000, "longest": 6000, "rows": 509,
         "ragged": False, "mix": 5, "heads": 16, "kv_heads": 16, "dim": 128, "page": 16},
        # The new tokens of one decode step, in pages that are partly filled.
        {"name": "write_step", "kind": "write", "batch": 32, "shortest": 1, "longest": 8000, "rows": 1,
         "ragged": False, "mix": 3, "kv_heads": 16, "dim": 128, "page": 16},
        # A prefill batch of chat prompts, some behind a cached prefix.
        {"name": "write_prompts", "kind": "write", "batch": 12, "shortest": 0, "longest": 700, "rows": 1500,
         "ragged": True, "mix": 6, "kv_heads": 16, "dim": 128, "page": 16},
        # The fused Q/K/V projection of one user's token.
        {"name": "project_qkv", "kind": "project", "rows": 1, "out": 6144, "in": 2048, "group": 32},
        # The MLP's down projection of a small batch.
        {"name": "project_down", "kind": "project", "rows": 12, "out": 2048, "in": 5632, "group": 128},
        # The vocabulary projection of a batch of 32.
        {"name": "project_vocab", "kind": "project", "rows": 32, "out": 49152, "in": 2048, "group": 64},
        # The logits of a decode step, eight alternatives; part of the vocabulary is ruled out.
        {"name": "logprobs_step", "kind": "logprobs", "rows": 4, "vocab": 49152, "pad": 0, "top": 8, "bits": 16,
         "masked": 0.3},
        # Every token of a prompt scored, as a perplexity run does; an odd vocabulary in padded rows.
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 2041, "vocab": 50257, "pad": 47, "top": 1, "bits": 16,
         "masked": 0.0},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "write", "project", "project", "logprobs"])
    if kind == "project":
        rows, group = _log_uniform(rng, 1, 64), rng.choice([32, 64, 128])
        features = group * _log_uniform(rng, max(1, 256 // group), 8192 // group)
        most = min(49152, 49152 * 2048 * 32 // (features * max(rows, 32)))
        return {"kind": kind, "rows": rows, "out": _log_uniform(rng, 100, most), "in": features, "group": group}
    if kind == "logprobs":
        bits = rng.choice([16, 16, 32])
        vocab = _log_uniform(rng, 1000, 151_000)
        return {"kind": kind, "rows": _log_uniform(rng, 1, min(2041, 100_000_000 * 16 // (vocab * bits))),
                "vocab": vocab, "pad": rng.choice([0, 0, rng.randint(1, 64)]), "top": rng.choice([0, 1, 5, 20, 32]),
                "bits": bits, "masked": rng.choice([0.0, 0.0, rng.uniform(0.05, 0.95)])}
    heads, kv_heads, dim = rng.choice([(16, 16, 128), (32, 8, 128), (24, 2, 96), (55, 55, 96)])
    case = {"kind": kind, "mix": rng.randrange(1 << 20), "ragged": rng.random() < 0.5, "kv_heads": kv_heads,
            "dim": dim, "page": rng.choice([16, 32])}
    longest = _log_uniform(rng, 16, 8192)
    case |= {"longest": longest, "shortest": rng.choice([0, rng.randint(1, longest)])}
    most = max(1, 120_000 * 16 * 128 // (kv_heads * dim * longest))  # history tokens of the whole batch
    if kind == "write":
        case["rows"] = rng.choice([1, _log_uniform(rng, 2, 2048)])
        return case | {"batch": min(most, _log_uniform(rng, 1, 48), max(1, 6000 // case["rows"]))}
    case["rows"] = rng.choice([1, 1, _log_uniform(rng, 2, 16), _log_uniform(rng, 17, 500)])
    case["heads"] = heads
    return case | {"batch": min(most, _log_uniform(rng, 1, 48), max(1, 1000 * 16 // (case["rows"] * heads)))}


def _histories(case):
    """Cached tokens per request: log-uniform, the longest among them; one request without any where ``shortest`` is 0."""
    rng = random.Random(case["mix"])
    lengths = [_log_uniform(rng, max(1, case["shortest"]), case["longest"]) for _ in range(case["batch"])]
    lengths[rng.randrange(case["batch"])] = case["longest"]
    if case["shortest"] == 0 and case["batch"] > 1:
        lengths[lengths.index(min(lengths))] = 0
    return lengths


def _new_rows(case):
    """New rows per request: all alike, or anything up to ``rows`` (the most among them)."""
    rng = random.Random(case["mix"] + 1)
    rows = [rng.randint(0, case["rows"]) if case["ragged"] else case["rows"] for _ in range(case["batch"])]
    rows[rng.randrange(case["batch"])] = case["rows"]
    return rows


# ---------------------------------------------------------------- prepare


def _keys(shape, generator):
    """N(0, 1) with a few strong channels, as keys have; BF16."""
    x = torch.randn(shape, generator=generator, device=DEVICE)
    x[..., :: shape[-1] // 4] *= 8.0
    return x.to(torch.bfloat16)


def _values(shape, generator):
    return torch.randn(shape, generator=generator, device=DEVICE).to(torch.bfloat16)


def _prepare_cache(case, seed):
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    histories, rows = _histories(case), _new_rows(case)
    seq_lens = [h + n for h, n in zip(histories, rows)]
    pages = (max(seq_lens) + page - 1) // page
    blocks = case["batch"] * pages
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    # Pages full of tokens, also behind the last of a request: a pool that is in use.
    cache = torch.empty((2, blocks, heads, page, dim), dtype=torch.float8_e4m3fn, device=DEVICE)
    scales = torch.empty((2, blocks, heads), dtype=torch.float32, device=DEVICE)
    chunk = max(1, (1 << 26) // (heads * page * dim))
    for start in range(0, blocks, chunk):
        shape = (min(chunk, blocks - start), heads, page, dim)
        for plane, make in enumerate((_keys, _values)):
            x = make(shape, generator).float()
            scale = _power(_exponent(x.abs().amax(dim=(2, 3))))
            scales[plane, start:start + chunk] = scale
            cache[plane, start:start + chunk] = (x / scale[..., None, None]).to(torch.float8_e4m3fn)
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    total = starts[-1]
    state = {
        "case": case, "cache": cache, "scales": scales, "most_rows": max(rows),
        "key": _keys((total, heads, dim), generator), "value": _values((total, heads, dim), generator),
        "starts": torch.tensor(starts, dtype=torch.int32, device=DEVICE),
        "seq_lens": torch.tensor(seq_lens, dtype=torch.int32, device=DEVICE),
        "table": torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).view(case["batch"], pages).to(
            torch.int32).to(DEVICE),
    }
    if case["kind"] == "attend":
        state["query"] = torch.randn((total, case["heads"], dim), generator=generator, device=DEVICE).to(torch.bfloat16)
        state["output"] = torch.empty_like(state["query"])
    return state


def _project_inputs(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    shape = (case["out"], case["in"] // case["group"], case["group"])
    weight = torch.randn(shape, generator=generator, device=DEVICE) / math.sqrt(case["in"])
    scales = (weight.abs().amax(dim=2) / 7).to(torch.bfloat16)
    codes = torch.round(weight / scales.float()[..., None]).clamp(-8, 7).to(torch.int8)
    x = torch.randn((case["rows"], case["in"]), generator=generator, device=DEVICE).to(torch.bfloat16)
    return x, codes.view(case["out"], case["in"]), scales


def _prepare_project(case, seed):
    x, codes, scales = _project_inputs(case, seed)
    if own:  # the weights as a model holds them, laid out once
        from residualquant_amd import step_ops

        return {"case": case, "x": x, "weight": step_ops.pack_weight_int4(codes, scales)}
    return {"case": case, "x": x, "codes": codes, "scales": scales}


def _prepare_logprobs(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.randn((rows, vocab + case["pad"]), generator=generator, device=DEVICE) * 2.5
    logits = logits.to(torch.bfloat16 if case["bits"] == 16 else torch.float32)[:, :vocab]
    tokens = torch.randint(0, vocab, (rows,), generator=generator, device=DEVICE)
    if case["masked"]:
        ruled_out = torch.rand(vocab, generator=generator, device=DEVICE) < case["masked"]
        ruled_out[tokens] = False
        logits.masked_fill_(ruled_out, -math.inf)
    return {"case": case, "logits": logits, "tokens": tokens}


def prepare(case, seed):
    return {"attend": _prepare_cache, "write": _prepare_cache, "project": _prepare_project,
            "logprobs": _prepare_logprobs}[case["kind"]](case, seed)


# ---------------------------------------------------------------- plain forms


def _exponent(largest):
    """The least e >= -126 with largest <= 448 x 2^e (largest finite, not negative)."""
    mantissa, exponent = torch.frexp(largest)  # largest = mantissa x 2^exponent, 448 = 0.875 x 2^9
    return torch.where(largest > 0, exponent - 9 + (mantissa > 0.875), -126).clamp(min=-126)


def _power(exponent):
    """2^exponent in float32, from its bits (exponent >= -126)."""
    return ((exponent + 127).int() << 23).view(torch.float32)


def _row_places(state):
    """Per flat row: its request and its place among the request's new rows."""
    starts = state["starts"].long()
    row = torch.arange(state["key"].size(0), device=DEVICE)
    request = torch.searchsorted(starts[1:], row, right=True)
    return request, row - starts[request]


def _plain_attend(state):
    query, page = state["query"], state["case"]["page"]
    batch, table = state["seq_lens"].numel(), state["table"].long()
    heads, (_, kv_heads, dim) = query.size(1), state["key"].shape
    group, most = heads // kv_heads, state["most_rows"]
    counts = (state["starts"][1:] - state["starts"][:-1]).long()
    histories = state["seq_lens"].long() - counts
    request, place = _row_places(state)

    def padded(x):
        out = torch.zeros((batch, most) + x.shape[1:], device=DEVICE)
        out[request, place] = x.float()
        return out.transpose(1, 2)  # [batch, heads, most, dim]

    def tokens(plane, new):
        pages = state["cache"][plane].view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
        pages = pages * state["scales"][plane][table][..., None, None]
        history = pages.transpose(1, 2).reshape(batch, kv_heads, -1, dim)
        return torch.cat([history, padded(new)], dim=2)

    keys, values = tokens(0, state["key"]), tokens(1, state["value"])
    span = table.size(1) * page
    old = torch.arange(span, device=DEVICE)[None, :] < histories[:, None]
    new = torch.arange(most, device=DEVICE)
    mask = torch.cat([old[:, None, :].expand(batch, most, span), (new[None, :] <= new[:, None]).expand(batch, most, most)],
                     dim=2)[:, None, None]  # [batch, 1, 1, most, span + most]
    q = padded(query).reshape(batch, kv_heads, group * most, dim) * dim ** -0.5
    scores = torch.matmul(q, keys.transpose(2, 3)).view(batch, kv_heads, group, most, span + most)
    scores = scores.masked_fill_(~mask, -math.inf)
    weights = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    weights = weights / weights.sum(dim=-1, keepdim=True)
    out = torch.matmul(weights.view(batch, kv_heads, group * most, -1), values)
    out = out.view(batch, heads, most, dim).transpose(1, 2)[request, place]
    return out.to(torch.bfloat16)


def _plain_write(state):
    page = state["case"]["page"]
    cache, scales, table = state["cache"].view(torch.uint8), state["scales"], state["table"].long()
    _, blocks, heads, _, dim = cache.shape
    counts = (state["starts"][1:] - state["starts"][:-1]).long()
    histories = state["seq_lens"].long() - counts
    request, place = _row_places(state)
    position = histories[request] + place
    block, slot = table[request, position // page], position % page
    # Tokens that a block holds already: the partly filled page of each request with new rows.
    partly = (histories % page > 0) & (counts > 0)
    last = table.gather(1, (histories // page).clamp(max=table.size(1) - 1)[:, None])[:, 0]
    kept = torch.zeros(blocks, dtype=torch.long, device=DEVICE)
    kept[last[partly]] = (histories % page)[partly]
    touched = torch.zeros(blocks, dtype=torch.bool, device=DEVICE)
    touched[block] = True
    new = torch.stack([state["key"], state["value"]]).float()  # [2, rows, heads, dim]
    largest = torch.zeros((2, blocks, heads), device=DEVICE)
    largest.scatter_reduce_(1, block[None, :, None].expand(2, -1, heads), new.abs().amax(dim=3), "amax")
    need = _power(_exponent(largest))
    grown = torch.where((kept > 0)[None, :, None], torch.maximum(scales, need), need)
    grown = torch.where(touched[None, :, None], grown, scales)
    old = cache[:, last[partly]].view(torch.float8_e4m3fn).float()
    again = old * (scales / grown)[:, last[partly]][..., None, None]
    mine = torch.arange(page, device=DEVICE)[None, :] < kept[last[partly]][:, None]
    again = torch.where(mine[None, :, None, :, None], again, old)
    cache[:, last[partly]] = again.to(torch.float8_e4m3fn).view(torch.uint8)
    codes = (new / grown[:, block][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    cache[:, block, :, slot] = codes.transpose(0, 1)
    scales.copy_(grown)
    return {"cache": state["cache"], "scales": scales}


def _plain_project(state):
    codes, scales = state["codes"], state["scales"]
    weight = codes.view(scales.size(0), scales.size(1), -1).float() * scales.float()[..., None]
    return torch.matmul(state["x"].float(), weight.view(codes.shape).t()).to(torch.bfloat16)


def _plain_logprobs(state):
    x, top = state["logits"].float(), state["case"]["top"]
    largest = x.amax(dim=1, keepdim=True)
    shifted = x - largest
    weights = torch.exp(shifted)
    total = weights.sum(dim=1)
    log_total = torch.log(total)
    entropy = log_total - torch.where(weights > 0, weights * shifted, 0.0).sum(dim=1) / total
    logprob = shifted.gather(1, state["tokens"][:, None])[:, 0] - log_total
    values, order = torch.sort(shifted, dim=1, descending=True, stable=True) if top else (shifted, state["tokens"][:, None])
    return {"logprob": logprob, "entropy": entropy, "top_logprobs": values[:, :top] - log_total[:, None],
            "top_tokens": order[:, :top]}


# ---------------------------------------------------------------- run


def run(state):
    kind = state["case"]["kind"]
    if own:
        from residualquant_amd import ops, step_ops

        if kind == "attend":
            ops.paged_attention_fp8(state["query"], state["key"], state["value"], state["cache"], state["scales"],
                                    state["output"], state["starts"], state["seq_lens"], state["table"])
            return state["output"]
        if kind == "write":
            ops.quantize_fp8(state["key"], state["value"], state["cache"], state["scales"], state["starts"],
                             state["seq_lens"], state["table"])
            return {"cache": state["cache"], "scales": state["scales"]}
        if kind == "project":
            return step_ops.linear_rows_int4(state["x"], state["weight"])
        result = step_ops.token_logprobs(state["logits"], state["tokens"], top=state["case"]["top"])
        return {"logprob": result.logprob, "entropy": result.entropy, "top_logprobs": result.top_logprobs,
                "top_tokens": result.top_tokens}
    return {"attend": _plain_attend, "write": _plain_write, "project": _plain_project,
            "logprobs": _plain_logprobs}[kind](state)


# ---------------------------------------------------------------- work


def work(case):
    kind = case["kind"]
    if kind == "project":
        rows, out, features = case["rows"], case["out"], case["in"]
        return {"bytes": out * features // 2 + 2 * out * features // case["group"] + 2 * rows * (out + features),
                "flops": 2 * rows * out * features}
    if kind == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * (vocab * case["bits"] // 8 + 16 + 12 * case["top"]), "flops": 5 * rows * vocab}
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    histories, rows = _histories(case), _new_rows(case)
    if kind == "write":
        # Each new value read and written, a scale per touched page.
        pages = sum((h + n - 1) // page - h // page + 1 for h, n in zip(histories, rows) if n)
        return {"bytes": 2 * kv_heads * (3 * sum(rows) * dim + 8 * pages), "flops": 4 * kv_heads * dim * sum(rows)}
    heads = case["heads"]
    read = [h for h, n in zip(histories, rows) if n]
    return {"bytes": 2 * kv_heads * (dim * sum(read) + 4 * sum((h + page - 1) // page for h in read))
            + 2 * 2 * dim * (heads + kv_heads) * sum(rows),
            "flops": 4 * dim * heads * sum(n * h + n * (n + 1) // 2 for h, n in zip(histories, rows))}


# ---------------------------------------------------------------- exact


def _exact_attend(case, state):
    histories, rows, page = _histories(case), _new_rows(case), case["page"]
    group, out, row = case["heads"] // case["kv_heads"], [], 0
    for b, (h, n) in enumerate(zip(histories, rows)):
        if n == 0:
            continue
        used = state["table"][b, :(h + page - 1) // page].tolist()
        planes = []
        for plane, new in enumerate((state["key"], state["value"])):
            held = [state["cache"][plane, block].double() * state["scales"][plane, block].double()[:, None, None]
                    for block in used]
            held = torch.cat(held, dim=1)[:, :h] if held else new.double().transpose(0, 1)[:, :0]
            planes.append(torch.cat([held, new[row:row + n].double().transpose(0, 1)], dim=1))
        keys, values = (x.repeat_interleave(group, dim=0) for x in planes)
        q = state["query"][row:row + n].double().transpose(0, 1)
        scores = q @ keys.transpose(1, 2) / math.sqrt(case["dim"])
        later = torch.ones((n, n), device=DEVICE).triu(1).bool()
        scores[:, :, h:].masked_fill_(later, -math.inf)
        out.append((torch.softmax(scores, dim=2) @ values).transpose(0, 1))
        row += n
    return torch.cat(out)


def _power64(exponent):
    """2^exponent in float64, from its bits (the device's exp2 and ldexp may be off by a rounding)."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _exact_e4m3(x):
    """Float64 values rounded to E4M3, ties to even (|x| <= 448)."""
    _, exponent = torch.frexp(x)
    quantum = _power64((exponent - 1).clamp(min=-6) - 3)
    return torch.round(x / quantum) * quantum


def _exact_write(case, state):
    histories, rows, page = _histories(case), _new_rows(case), case["page"]
    cache, scales, row = state["cache"].double(), state["scales"].double(), 0
    new = [state["key"].double(), state["value"].double()]
    for b, (h, n) in enumerate(zip(histories, rows)):
        for first in range(h // page, (h + n - 1) // page + 1 if n else 0):
            block = int(state["table"][b, first])
            begin, end = max(h, first * page), min(h + n, first * page + page)
            kept = begin - first * page
            for plane in range(2):
                x = new[plane][row + begin - h:row + end - h].transpose(0, 1)
                largest = x.abs().amax(dim=(1, 2)).clamp(min=2.0 ** -150)
                power = torch.floor(torch.log2(largest)) - 8  # 2^8 <= 448 < 2^9
                power = torch.where(largest > E4M3_MAX * _power64(power), power + 1, power).clamp(min=-126)
                scale = _power64(power)
                if kept:
                    before = scales[plane, block].clone()
                    scale = torch.maximum(scale, before)
                    cache[plane, block, :, :kept] = _exact_e4m3(cache[plane, block, :, :kept]
                                                                * (before / scale)[:, None, None])
                scales[plane, block] = scale
                cache[plane, block, :, kept:kept + end - begin] = _exact_e4m3(x / scale[:, None, None])
        row += n
    return {"cache": cache, "scales": scales}


def _exact_project(case, seed):
    x, codes, scales = _project_inputs(case, seed)
    scales = scales.double().repeat_interleave(case["group"], dim=1)
    parts = [x.double() @ (codes[k:k + 4096].double() * scales[k:k + 4096]).t() for k in range(0, case["out"], 4096)]
    return torch.cat(parts, dim=1)


def _exact_logprobs(case, state):
    found = []
    for row in range(0, case["rows"], 64):
        x = state["logits"][row:row + 64].double()
        logp = x - torch.logsumexp(x, dim=1, keepdim=True)
        order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :case["top"]]
        found.append((logp.gather(1, state["tokens"][row:row + 64, None])[:, 0],
                      -torch.special.xlogy(logp.exp(), logp.exp()).sum(dim=1), logp.gather(1, order), order))
    return dict(zip(("logprob", "entropy", "top_logprobs", "top_tokens"), (torch.cat(x) for x in zip(*found))))


def exact(case, seed):
    if case["kind"] == "project":
        return _exact_project(case, seed)
    return {"attend": _exact_attend, "write": _exact_write, "logprobs": _exact_logprobs}[case["kind"]](
        case, prepare(case, seed))
