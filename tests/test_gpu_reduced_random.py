"""Seeded random calls of the 8-bit cache, the 4-bit projections and the log probabilities, against the
references and bounds of their own tests."""

from __future__ import annotations

import math
import random

import pytest
import torch

from residualquant_amd import step_ops

from . import test_gpu_fp8_cache as fp8
from . import test_gpu_linear_int4 as int4
from . import test_gpu_logprobs as scores

pytestmark = pytest.mark.gpu


def _spread(rng, low, high):
    """Spread evenly over the logarithm of low..high."""
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def _requests(rng, work):
    """Histories and rows of 1 to 90 requests of at most ``work`` row x token pairs each."""
    requests = _spread(rng, 1, 90)
    longest, most = _spread(rng, 1, 3000), rng.choice([1, 1, 6, 40, 200])
    most = max(1, min(most, work // (longest + 1)))
    histories = [rng.choice([0, _spread(rng, 1, longest), longest]) for _ in range(requests)]
    rows = [most if rng.random() < 0.5 else rng.randint(0, most) for _ in range(requests)]
    rows[rng.randrange(requests)] = most
    return histories, rows


@pytest.mark.parametrize("seed", range(32))
def test_attention_random_calls(device, seed):
    rng = random.Random(seed)
    histories, rows = _requests(rng, 200000)
    kv_heads, group = rng.choice([1, 2, 3]), rng.choice([1, 1, 2, 3, 8])
    dim, page = rng.choice([96, 128]), rng.choice([16, 32])
    print(f"requests={len(rows)} rows={max(rows)} longest={max(histories)} heads={kv_heads}x{group} D={dim} PT={page}", flush=True)
    case = fp8._case(histories, rows, kv_heads * group, kv_heads, dim, page, seed=seed, extra_pages=rng.randint(0, 3))
    fp8._check_attention(case, fp8._attend(fp8._to(case, device), device))


@pytest.mark.parametrize("seed", range(16))
def test_write_random_calls(device, seed):
    rng = random.Random(100 + seed)
    histories, rows = _requests(rng, 40000)
    kv_heads, dim, page = rng.choice([1, 2, 5]), rng.choice([96, 128]), rng.choice([16, 32])
    print(f"requests={len(rows)} rows={max(rows)} longest={max(histories)} heads={kv_heads} D={dim} PT={page}", flush=True)
    case = fp8._case(histories, rows, kv_heads, kv_heads, dim, page, seed=seed, outlier=rng.choice([0.01, 1.0, 100.0]))
    fp8._check_write(case, device, repeat=rng.choice([1, 2]))


@pytest.mark.parametrize("seed", range(32))
def test_linear_random_shapes(device, seed):
    rng = random.Random(200 + seed)
    group = rng.choice([32, 64, 128])
    rows, features = rng.randint(1, 64), group * _spread(rng, 1, 9000 // group)
    out = _spread(rng, 1, 24000000 // features if features > 1000 else 24000)
    out = min(out, 24000)
    print(f"rows={rows} out={out} in={features} group={group}", flush=True)
    codes, scales = int4._weight(out, features, group, seed=seed)
    x = torch.randint(-4, 5, (rows, features), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
    scales = torch.exp2(scales.float().log2().round()).to(torch.bfloat16)
    got = step_ops.linear_rows_int4(x.to(device), step_ops.pack_weight_int4(codes.to(device), scales.to(device)))
    # Integers times powers of two: 2^-10 to 2^-5, sums below 2^24 of the least unit are exact in any order.
    want = x.float() @ (codes.float() * scales.float().repeat_interleave(group, dim=1)).t()
    assert torch.equal(got.cpu(), want.to(torch.bfloat16))


@pytest.mark.parametrize("seed", range(32))
def test_logprobs_random_calls(device, seed):
    rng = random.Random(300 + seed)
    vocab = _spread(rng, 1, 160000)
    rows = _spread(rng, 1, max(1, min(700, 4000000 // vocab)))
    top, pad = rng.randint(0, min(32, vocab)), rng.choice([0, 1, 7, 40])
    dtype = rng.choice([torch.bfloat16, torch.float32])
    print(f"rows={rows} vocab={vocab} top={top} pad={pad} {dtype}", flush=True)
    logits, tokens = scores._logits(rows, vocab + pad, dtype, seed, scale=rng.choice([0.1, 3.0, 40.0]))
    if rng.random() < 0.5 and vocab > 1:
        logits[torch.rand(logits.shape, generator=torch.Generator().manual_seed(seed)) < 0.4] = -torch.inf
        logits[:, rng.randrange(vocab)] = 1.0
    tokens = tokens % vocab
    moved = logits.to(device)[:, :vocab]
    got = step_ops.token_logprobs(moved, tokens.to(device), top=top)
    scores._check(logits[:, :vocab], tokens, top, device, got=got)


def test_calls_on_two_streams_at_once(device):
    """Two streams issue attention, projections and log probabilities at the same time; each gets its own results."""
    cases = [fp8._to(fp8._case([2500, 40, 1200], [1, 5, 120], 4, 2, 128, 16, seed=9), device),
             fp8._to(fp8._case([1900, 700], [1, 1], 4, 4, 96, 32, seed=10), device)]
    codes, scales = int4._weight(5000, 2048, 64, seed=11)
    weight = step_ops.pack_weight_int4(codes.to(device), scales.to(device))
    x = [torch.randn((n, 2048), generator=torch.Generator().manual_seed(n)).to(torch.bfloat16).to(device) for n in (3, 50)]
    logits = [torch.randn((n, 30000), generator=torch.Generator().manual_seed(n)).to(torch.bfloat16).to(device) for n in (2, 300)]
    tokens = [torch.arange(row.size(0), device=device) for row in logits]

    def run(k):
        scored = step_ops.token_logprobs(logits[k], tokens[k], top=5)
        return [fp8._attend(cases[k], device), step_ops.linear_rows_int4(x[k], weight), *scored]

    want = [run(0), run(1)]
    streams = [torch.cuda.Stream(device=device) for _ in range(2)]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream(device))
    got = [[], []]
    for _ in range(8):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(run(k))
    torch.cuda.synchronize(device)
    for k in range(2):
        for results in got[k]:
            assert all(torch.equal(mine, first) for mine, first in zip(results, want[k]))
