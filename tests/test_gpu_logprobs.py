"""Log probabilities of tokens, entropy and top alternatives (step_ops.token_logprobs) against float64."""

from __future__ import annotations

import pytest
import torch

from residualquant_amd import step_ops

pytestmark = pytest.mark.gpu


def _reference(logits, tokens, top):
    """Values and their bounds in float64.  A float32 sum over n entries of a row: each thread adds at
    least every 256th, then a tree; the exponential is off by 2^-22 and by the rounding of x - m.  A
    log probability is x - m and log S, each rounded, and their difference."""
    x = logits.double()
    n = x.size(1)
    m = x.amax(dim=1, keepdim=True)
    d = x - m
    w = torch.where(x == -torch.inf, 0.0, torch.exp(d))
    s = w.sum(dim=1)
    log_s = torch.log(s)
    inside = (tokens >= 0) & (tokens < n)
    at = d.gather(1, tokens.clamp(0, n - 1)[:, None])[:, 0]
    logprob = torch.where(inside, at - log_s, torch.nan)
    terms = torch.where(w > 0, w * d, 0.0)
    entropy = log_s - terms.sum(dim=1) / s
    order = torch.argsort(x.nan_to_num(nan=torch.inf, posinf=torch.inf, neginf=-torch.inf), dim=1, descending=True,
                          stable=True)[:, :top]
    values = d.gather(1, order) - log_s[:, None]
    summed = (n / 256 + 64) * 2.0 ** -24 + 2.0 ** -21
    spread = torch.where(w > 0, w * d.abs() * (1 + d.abs()), 0.0).sum(dim=1) / s
    bound = summed * (1 + spread) + 2.0 ** -22 * (log_s.abs() + 1)
    return {"logprob": (logprob, bound + 2.0 ** -23 * (at.abs() + logprob.abs())),
            "entropy": (entropy, bound + 2.0 ** -23 * entropy.abs()),
            "top_logprobs": (values, bound[:, None] + 2.0 ** -23 * (values.abs() + d.gather(1, order).abs())),
            "top_tokens": order}


def _check(logits, tokens, top, device, got=None):
    got = got or step_ops.token_logprobs(logits.to(device), tokens.to(device), top=top)
    want = _reference(logits, tokens, top)
    assert torch.equal(got.top_tokens.cpu(), want.pop("top_tokens"))
    for name, (value, bound) in want.items():
        mine = getattr(got, name).cpu().double()
        assert torch.equal(mine.isnan(), value.isnan()), name
        assert torch.equal(mine.isneginf(), value.isneginf()), name
        off = (mine - value).abs()[value.isfinite()]
        assert bool((off <= bound[value.isfinite()]).all()), (name, (off / bound[value.isfinite()]).max())


def _logits(rows, vocab, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g) * scale).to(dtype), torch.randint(0, vocab, (rows,), generator=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (2, 7, 7), (5, 33, 32), (1, 256, 5),
                                            (2, 257, 20), (9, 1000, 3), (4, 4099, 32), (1, 49152, 8), (3, 50257, 20),
                                            (300, 777, 1), (2, 131075, 32), (70, 8192, 0)])
def test_logprobs(device, dtype, rows, vocab, top):
    print(f"rows={rows} vocab={vocab} top={top} {dtype}", flush=True)
    logits, tokens = _logits(rows, vocab, dtype, seed=rows + vocab + top)
    _check(logits, tokens, top, device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (3, 2), (5, 7), (0, 40)])
def test_row_alignment(device, dtype, offset, pad):
    """Rows that start at any element; what lies beside them is not read."""
    logits, tokens = _logits(6, 5001, dtype, seed=offset + pad)
    wide = torch.full((6, 5001 + offset + pad), torch.nan, dtype=dtype)
    wide[:, offset:offset + 5001] = logits
    on = wide.to(device)[:, offset:offset + 5001]
    _check(logits, tokens, 9, device, got=step_ops.token_logprobs(on, tokens.to(device), top=9))


@pytest.mark.parametrize("vocab", [100, 5000, 70001])
def test_order_of_equal_and_sorted_logits(device, vocab):
    """Ties go to the lower token, in rows where many or all are equal, rising, falling or in blocks."""
    index = torch.arange(vocab)
    rows = torch.stack([torch.zeros(vocab), index.float(), -index.float(), (index % 3).float(), -(index % 1024).float(),
                        (index // 8 % 64).float(), torch.where(index % 2 == 0, 0.0, -0.0),
                        (index == vocab - 1).float(), (index % 512 < 8).float() * index.float(),
                        (index % 64 == 63).float() * (1 + index.float())])
    tokens = torch.randint(0, vocab, (rows.size(0),), generator=torch.Generator().manual_seed(vocab))
    for top in (1, 32):
        _check(rows, tokens, top, device)
        _check(rows.to(torch.bfloat16), tokens, top, device)


def test_ruled_out_tokens(device):
    logits, tokens = _logits(6, 3001, torch.float32, seed=8)
    logits[0, 1:] = -torch.inf           # one token left
    tokens[0] = 0
    logits[1, ::2] = -torch.inf
    tokens[1] = 2                        # a ruled-out token: -inf
    logits[2, 5:2990] = -torch.inf       # fewer left than alternatives asked for
    logits[3] = -torch.inf               # none left: NaN
    logits[4] = torch.finfo(torch.float32).min  # the lowest value is no mask
    logits[5] = torch.finfo(torch.float32).min
    logits[5, 17] = 0.0
    _check(logits, tokens, 20, device)


def test_nan_and_infinity(device):
    logits, tokens = _logits(3, 2000, torch.bfloat16, seed=9)
    logits[0, 900] = torch.nan
    logits[1, 1999] = torch.inf
    got = step_ops.token_logprobs(logits.to(device), tokens.to(device), top=4)
    assert bool(got.logprob[:2].isnan().all()) and bool(got.entropy[:2].isnan().all())
    assert bool(got.top_logprobs[:2].isnan().all())
    assert int(got.top_tokens[0, 0]) == 900 and int(got.top_tokens[1, 0]) == 1999
    _check(logits[2:], tokens[2:], 4, device)


def test_wide_range(device):
    """Logits of thousands apart, and far from zero."""
    logits, tokens = _logits(4, 4000, torch.float32, seed=10, scale=2000.0)
    logits[1] += 1e6
    logits[2] -= 1e6
    _check(logits, tokens, 5, device)


def test_tokens_outside_the_vocabulary(device):
    logits, tokens = _logits(5, 500, torch.bfloat16, seed=11)
    tokens[0], tokens[2], tokens[3] = -1, 500, 1 << 40
    _check(logits, tokens, 3, device)


def test_streams_graphs_and_refusals(device):
    logits, tokens = _logits(3, 20001, torch.bfloat16, seed=12)
    x, t = logits.to(device), tokens.to(device)
    want = step_ops.token_logprobs(x, t, top=8)
    stream = torch.cuda.Stream(device=device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        other = step_ops.token_logprobs(x, t, top=8)
    torch.cuda.current_stream(device).wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step_ops.token_logprobs(x, t, top=8)
        graphs.append((graph, captured))
    for step in range(3):
        fresh, drawn = _logits(3, 20001, torch.bfloat16, seed=20 + step)
        x.copy_(fresh)
        t.copy_(drawn)
        for graph, _ in graphs:
            graph.replay()
        eager = step_ops.token_logprobs(x, t, top=8)
        torch.cuda.synchronize()
        for _, captured in graphs:
            assert all(torch.equal(a, b) for a, b in zip(captured, eager)), f"replay {step}"
    empty = step_ops.token_logprobs(x[:0], t[:0], top=3)
    assert empty.logprob.shape == (0,) and empty.top_tokens.shape == (0, 3)
    for wrong in (dict(top=33), dict(top=-1), dict(tokens=t[:2]), dict(tokens=t.int()), dict(logits=x.half()),
                  dict(logits=x.t().contiguous().t()), dict(logits=x[0])):
        with pytest.raises(RuntimeError):
            step_ops.token_logprobs(**{"logits": x, "tokens": t, "top": 2, **wrong})


def test_expanded_rows_are_refused(device):
    """Rows that share memory (stride 0) are not rows of vocab logits; one row may have any stride."""
    row, tokens = torch.randn(1, 500, device=device), torch.zeros(4, dtype=torch.int64, device=device)
    with pytest.raises(RuntimeError, match="unit column stride"):
        step_ops.token_logprobs(row.expand(4, 500), tokens)
    with pytest.raises(RuntimeError, match="unit column stride"):
        step_ops.token_logprobs(torch.randn(2000, device=device).as_strided((4, 500), (100, 1)), tokens)
    odd = torch.randn(2000, device=device).as_strided((1, 500), (3, 1))
    _check(odd.cpu().contiguous(), tokens[:1].cpu(), 3, device, got=step_ops.token_logprobs(odd, tokens[:1], top=3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 32, 33, 3001])
def test_nan_ranks_first_wherever_it_is(device, dtype, vocab):
    """NaN at token 0, at the last and everywhere, beside infinities, with as many alternatives as there are tokens."""
    logits, tokens = _logits(6, vocab, dtype, seed=vocab)
    logits[0, 0] = torch.nan
    logits[1, vocab - 1] = torch.nan
    logits[2] = torch.nan
    logits[3, ::2] = torch.nan
    logits[4] = -torch.inf
    logits[4, 0] = torch.nan
    logits[5, vocab // 2] = torch.inf
    top = min(32, vocab)
    print(f"vocab={vocab} top={top} {dtype}", flush=True)
    got = step_ops.token_logprobs(logits.to(device), tokens.to(device), top=top)
    for row in range(6):
        x = logits[row].float()
        order = sorted(range(vocab), key=lambda i: (not x[i].isnan(), -x[i] if not x[i].isnan() else 0.0, i))
        assert got.top_tokens[row].tolist() == order[:top], row
    assert bool(got.logprob.isnan().all()) and bool(got.entropy.isnan().all())
    assert bool(got.top_logprobs.isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [900, 50257])
def test_logits_far_from_zero(device, dtype, vocab):
    """Rows around +-5e9 and more, where log2(e) x has a rounding of hundreds: the maximum has e^0 all the same."""
    for k, at in enumerate((5e9, 1e10, 2e10, 1e20, 1e30, 3e38, -5e10, -1e11, -1e12, -1e30, -3e38, 2.0 ** 100, -2.0 ** 100)):
        logits, tokens = _logits(4, vocab, dtype, seed=30 + k)
        logits = logits.float()
        logits[0] += at                        # equal, or a unit apart
        logits[1] = at * (1 + logits[1].abs() * 2.0 ** -10).clamp(max=1.1)
        logits[2] = at
        logits[3] = at * 0.75
        logits[3, vocab // 3] = at
        tokens[3] = vocab // 3
        _check(logits.clamp(-3.38e38, 3.38e38).to(dtype), tokens, 3, device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask", [-1e4, -1e10, -1e20, -1e30, -2.0 ** 120, -2.0 ** 126, -1e38, -2e38, -3.38e38])
def test_finite_masks(device, dtype, mask):
    """Ruled-out tokens held as a finite value, in stretches that whole threads see nothing else of, first, last or all."""
    logits, tokens = _logits(6, 20011, dtype, seed=44)
    logits[0, 5000:] = mask
    logits[1, :15000] = mask
    logits[2, torch.rand(20011, generator=torch.Generator().manual_seed(3)) < 0.9] = mask
    logits[3, 4096:] = mask
    logits[3, :4096:2] = mask
    logits[4] = mask
    logits[5] = mask
    logits[5, 777] = 2.0
    _check(logits, tokens, 4, device)


def test_finite_masks_are_as_infinite_ones(device):
    """A row masked with a finite value gives what the row masked with -inf gives, where neither value has a weight."""
    logits, tokens = _logits(3, 49152, torch.float32, seed=45)
    out = torch.rand(49152, generator=torch.Generator().manual_seed(4)) < 0.3
    out[tokens] = False
    want = step_ops.token_logprobs(logits.masked_fill(out, -torch.inf).to(device), tokens.to(device), top=8)
    for mask in (-1e4, -1e10, -1e30, -1e38):
        got = step_ops.token_logprobs(logits.masked_fill(out, mask).to(device), tokens.to(device), top=8)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), mask


def test_more_rows_than_one_launch_takes(device):
    """2^24 and some rows of two logits."""
    rows = (1 << 24) + 3
    g = torch.Generator(device=device).manual_seed(7)
    logits = torch.randn((rows, 2), generator=g, device=device).to(torch.bfloat16)
    tokens = torch.randint(0, 2, (rows,), generator=g, device=device)
    got = step_ops.token_logprobs(logits, tokens, top=1)
    # Against the small calls, which the tests above check: the last rows, and some around the launches' borders.
    for first in (0, (1 << 22) - 20, (1 << 23) - 1, (1 << 24) - 30, rows - 40):
        part = slice(first, first + 40)
        want = step_ops.token_logprobs(logits[part], tokens[part], top=1)
        assert all(torch.equal(a[part], b) for a, b in zip(got, want)), first
    assert torch.equal(got.top_tokens[:, 0], (logits[:, 1] > logits[:, 0]).long())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [9, 28, 200, 3001])
def test_maxima_of_both_signs(device, dtype, vocab):
    """Positive logits far above stretches of negative ones, wherever they stand: the row's maximum is the positive one."""
    g = torch.Generator().manual_seed(vocab)
    logits, tokens = [], []
    for gap in (3.0, 40.0, 80.0, 84.0, 85.5, 87.0, 100.0, 1000.0):
        for place in sorted({0, 1, vocab // 2, vocab - 1, *torch.randint(0, vocab, (6,), generator=g).tolist()}):
            row = -gap * 0.5 - torch.rand(vocab, generator=g) * 3
            row[place] = gap * 0.5
            logits.append(row)
            tokens.append(place)
    logits, tokens = torch.stack(logits).to(dtype), torch.tensor(tokens)
    _check(logits, tokens, min(3, vocab), device)
    _check(logits, (tokens + 1) % vocab, 1, device)
    only = torch.full((8, vocab), -torch.inf)
    only[:, 0] = torch.arange(8) * 12.0
    only[:, -1] = -3.0
    _check(only.to(dtype), torch.zeros(8, dtype=torch.int64), 2, device)
