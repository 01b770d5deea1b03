"""Verification of drafted tokens (step_ops.verify_drafts) against the definition in float64."""

from __future__ import annotations

import math
import random

import pytest
import torch

from residualquant_amd import step_ops

pytestmark = pytest.mark.gpu


def reference(target, tokens, uniforms, starts, draft):
    """(accepted, tokens) by the definition; float64 sums in the tokens' order."""
    def clean(x):
        x = x.double()
        return torch.where((x > 0) & x.isfinite(), x, 0.0)

    rows, vocab = target.shape
    following, accepted = [-1] * rows, []
    for first, stop in zip(starts, starts[1:]):
        if first == stop:
            accepted.append(0)
            continue
        row = first
        while row < stop - 1:
            t = int(tokens[row + 1])
            inside = 0 <= t < vocab
            p = float(clean(target[row, t])) if inside else 0.0
            q = 1.0 if draft is None or not inside else float(clean(draft[row, t]))
            if not float(uniforms[row]) * q < p:
                break
            following[row] = t
            row += 1
        accepted.append(row - first)
        weight = clean(target[row])
        if row < stop - 1:
            if draft is not None:
                weight = (weight - clean(draft[row])).clamp(min=0.0)
            elif 0 <= int(tokens[row + 1]) < vocab:
                weight[int(tokens[row + 1])] = 0.0
        sums = torch.cumsum(weight, 0)
        limit = float(uniforms[stop - 1]) * float(sums[-1])
        positive = torch.nonzero(weight > 0)[:, 0]
        above = torch.nonzero((weight > 0) & (sums > limit))[:, 0]
        following[row] = int(above[0]) if len(above) else int(positive[-1]) if len(positive) else -1
    return accepted, following


def make(counts, vocab, dtype, seed, kept=1.0, pad=0, given=True):
    g = torch.Generator().manual_seed(seed)
    rows = sum(counts)

    def cut(x):
        if kept < 1.0:
            least = torch.kthvalue(x, max(1, int(vocab * (1 - kept))), dim=1, keepdim=True).values
            x = x.masked_fill(x < least, -math.inf)
        return torch.softmax(x, 1).to(dtype)

    logits = torch.randn((rows, vocab), generator=g) * 3
    target, draft = cut(logits), cut(logits + torch.randn((rows, vocab), generator=g) * 0.6)
    drawn = torch.multinomial(draft.float(), 1, generator=g)[:, 0] if given else draft.float().argmax(1)
    tokens = torch.cat([torch.zeros(1, dtype=torch.int64), drawn[:-1]]) if rows else drawn
    wide = torch.full((rows, vocab + pad), torch.nan, dtype=dtype)
    wide[:, :vocab] = target
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return wide[:, :vocab], tokens, torch.rand(rows, generator=g), starts, draft if given else None


def check(device, target, tokens, uniforms, starts, draft, **more):
    want_accepted, want = reference(target, tokens, uniforms, starts, draft)
    on = target.as_strided(target.shape, target.stride()).to(device)
    got = step_ops.verify_drafts(on, tokens.to(device), uniforms.to(device),
                                 torch.tensor(starts, dtype=torch.int32, device=device),
                                 draft=None if draft is None else draft.to(device), **more)
    assert got.accepted.dtype is torch.int32 and got.tokens.dtype is torch.int64
    assert got.accepted.tolist() == want_accepted
    assert got.tokens.tolist() == want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("given", [True, False])
@pytest.mark.parametrize("counts,vocab", [([1], 1), ([2], 1), ([1, 2, 3], 7), ([5], 1000), ([3, 0, 1, 9], 2048),
                                          ([4] * 9, 2049), ([1, 17, 70, 130], 333), ([2, 5], 49152), ([6] * 3, 50257),
                                          ([2] * 100, 511), ([5, 1, 3], 151000)])
def test_verify(device, counts, vocab, given, dtype):
    print(f"{counts} vocab={vocab} given={given} {dtype}", flush=True)
    for seed, kept in ((1, 1.0), (2, 0.1)):
        check(device, *make(counts, vocab, dtype, seed, kept=kept, given=given))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad", [1, 3, 40])
def test_padded_rows(device, dtype, pad):
    """Rows that start at any element; what lies beside them is not read."""
    target, tokens, uniforms, starts, draft = make([3, 4, 1], 5001, dtype, seed=pad, pad=pad)
    want = reference(target, tokens, uniforms, starts, draft)
    memory = torch.full((8, 5001 + pad), torch.nan, dtype=dtype)
    memory[:, pad:] = target
    wide = torch.full((8, 5001 + 2 * pad), torch.nan, dtype=dtype)
    wide[:, pad // 2:pad // 2 + 5001] = draft
    got = step_ops.verify_drafts(memory.to(device)[:, pad:], tokens.to(device), uniforms.to(device),
                                 torch.tensor(starts, dtype=torch.int32, device=device),
                                 draft=wide.to(device)[:, pad // 2:pad // 2 + 5001])
    assert (got.accepted.tolist(), got.tokens.tolist()) == want


@pytest.mark.parametrize("vocab", [5, 4096, 70001])
def test_borders(device, vocab):
    """Equal weights, whose sums are exact: random numbers on a border take the token behind it."""
    count = min(vocab, 4096)
    rows = 65
    target = torch.zeros((rows, vocab))
    place = torch.randperm(vocab, generator=torch.Generator().manual_seed(vocab))[:count].sort().values
    target[:, place] = 0.25
    uniforms = torch.tensor([k / 64 for k in range(rows)])  # 1.0 among them: the last of positive weight
    tokens = torch.zeros(rows, dtype=torch.int64)
    check(device, target, tokens, uniforms, list(range(rows + 1)), None)
    below = torch.nextafter(uniforms, torch.tensor(-1.0))
    check(device, target, tokens, below, list(range(rows + 1)), None)


def test_random_numbers_that_are_none(device):
    target, tokens, uniforms, starts, draft = make([3, 3, 3, 3], 900, torch.float32, seed=3)
    uniforms[[2, 5]] = torch.tensor([torch.nan, 2.0])
    uniforms[[8, 11]] = torch.tensor([-1.0, 0.0])
    uniforms[0], uniforms[3], uniforms[6], uniforms[9] = torch.nan, 1.0, 0.0, -0.5
    check(device, target, tokens, uniforms, starts, draft)
    check(device, target, tokens, uniforms, starts, None)


@pytest.mark.parametrize("given", [True, False])
def test_what_is_no_probability(device, given):
    """Negative entries, NaN and infinities count as 0; rows that hold nothing else give no token."""
    target, tokens, uniforms, starts, draft = make([2, 2, 2, 1, 1, 3], 1500, torch.float32, seed=4)
    g = torch.Generator().manual_seed(2)
    for x in (target, draft):
        bad = torch.rand(x.shape, generator=g) < 0.2
        x[bad] = torch.tensor([torch.nan, torch.inf, -torch.inf, -0.3, -0.0])[torch.randint(0, 5, (int(bad.sum()),), generator=g)]
    target[1], target[6], target[7] = 0.0, torch.nan, -1.0
    target[8], target[9] = torch.inf, 0.0  # a draft refused with nothing to draw from
    target[6, 1499] = 1e-38
    check(device, target, tokens, uniforms, starts, draft if given else None)


@pytest.mark.parametrize("given", [True, False])
def test_tokens_outside_the_vocabulary(device, given):
    target, tokens, uniforms, starts, draft = make([4, 4, 4], 800, torch.bfloat16, seed=5)
    tokens[2], tokens[5], tokens[9] = -1, 800, 2 ** 40
    check(device, target, tokens, uniforms, starts, draft if given else None)


def test_all_taken_and_none(device):
    target, tokens, uniforms, starts, draft = make([6, 6, 1], 3000, torch.float32, seed=6)
    check(device, draft, tokens, uniforms, starts, draft)  # like distributions: every draft is taken
    uniforms[:5] = 0.0
    check(device, target, tokens, uniforms, starts, draft)
    uniforms[:5] = 1.0
    target[range(5), tokens[1:6]] = 0.0
    check(device, target, tokens, uniforms, starts, draft)


def test_uneven_sizes_of_weights(device):
    """Weights of all sizes, down to subnormals: sums in float64 find the same token as in order."""
    g = torch.Generator().manual_seed(7)
    target = torch.exp2(torch.rand((40, 20000), generator=g) * 140 - 140)
    target[20:] = target[20:].sort(dim=1).values
    target[30:] = target[30:].flip(1)
    uniforms = torch.rand(40, generator=g)
    check(device, target, torch.zeros(40, dtype=torch.int64), uniforms, list(range(41)), None)


def test_rows_outside_the_requests(device):
    target, tokens, uniforms, _, draft = make([20], 600, torch.float32, seed=8)
    for starts in ([3, 5, 5, 12], [0, 20], [19, 20], [4, 4], [0, 0, 1]):
        check(device, target, tokens, uniforms, starts, draft)


def test_no_requests_and_no_rows(device):
    target, tokens, uniforms, _, draft = make([4], 600, torch.float32, seed=8)
    got = step_ops.verify_drafts(target.to(device), tokens.to(device), uniforms.to(device),
                                 torch.zeros(1, dtype=torch.int32, device=device))
    assert got.accepted.numel() == 0 and got.tokens.tolist() == [-1] * 4
    got = step_ops.verify_drafts(target[:0].to(device), tokens[:0].to(device), uniforms[:0].to(device),
                                 torch.zeros(3, dtype=torch.int32, device=device))
    assert got.accepted.tolist() == [0, 0] and got.tokens.numel() == 0


def test_draws_follow_the_distribution(device):
    """One draft drawn from q, judged against p: the tokens that follow are distributed as p, whatever q is.  Of n
    draws a token's share is off by more than 6 sqrt(p (1 - p) / n) once in 10^8."""
    n, vocab = 40000, 12
    g = torch.Generator().manual_seed(9)
    p, q = torch.softmax(torch.randn(vocab, generator=g), 0), torch.softmax(torch.randn(vocab, generator=g), 0)
    drafts = torch.multinomial(q, n, replacement=True, generator=g)
    tokens = torch.stack([torch.zeros(n, dtype=torch.int64), drafts], 1).flatten()
    got = step_ops.verify_drafts(p.expand(2 * n, vocab).contiguous().to(device), tokens.to(device),
                                 torch.rand(2 * n, generator=g).to(device),
                                 torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=device),
                                 draft=q.expand(2 * n, vocab).contiguous().to(device))
    share = torch.bincount(got.tokens.view(n, 2)[:, 0].cpu(), minlength=vocab).double() / n
    p = p.double() / p.double().sum()
    assert bool(((share - p).abs() <= 6 * torch.sqrt(p * (1 - p) / n)).all())


def test_captured_and_replayed_in_one_workspace(device):
    counts, vocab = [3, 1, 5], 40000
    target, tokens, uniforms, starts, draft = [x if isinstance(x, list) else x.contiguous().to(device)
                                               for x in make(counts, vocab, torch.float32, 10)]
    starts = torch.tensor(starts, dtype=torch.int32, device=device)
    memory = torch.full((step_ops.verify_drafts_workspace_bytes(3, vocab) + 9,), 0xff, dtype=torch.uint8, device=device)
    workspace = memory[9:]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step_ops.verify_drafts(target, tokens, uniforms, starts, draft=draft, workspace=workspace)
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for given in (draft, None):  # two graphs that share the workspace, one after the other
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step_ops.verify_drafts(target, tokens, uniforms, starts, draft=given, workspace=workspace)
        graphs.append((graph, got, given is not None))
    for seed in range(4):
        fresh = make(counts, vocab, torch.float32, 30 + seed)
        for held, new in zip((target, tokens, uniforms, draft), (fresh[0], fresh[1], fresh[2], fresh[4])):
            held.copy_(new)
        for graph, got, given in graphs:
            graph.replay()
            step_ops.verify_drafts(target, tokens, uniforms, starts, draft=draft)
            torch.cuda.synchronize()
            want = reference(fresh[0], fresh[1], fresh[2], fresh[3], fresh[4] if given else None)
            assert (got.accepted.tolist(), got.tokens.tolist()) == want


def test_two_streams_at_once(device):
    calls = [make(counts, vocab, torch.float32, seed) for seed, (counts, vocab) in
             enumerate((([4] * 8, 30000), ([2], 100000), ([1, 5, 3], 50257)))]
    on = [[x if x is None or isinstance(x, list) else x.to(device) for x in call] for call in calls]
    starts = [torch.tensor(call[3], dtype=torch.int32, device=device) for call in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for call, start, stream in zip(on, starts, streams):
            with torch.cuda.stream(stream):
                got.append(step_ops.verify_drafts(call[0], call[1], call[2], start, draft=call[4]))
    torch.cuda.synchronize()
    wants = [reference(*call) for call in calls]
    for k, result in enumerate(got):
        assert (result.accepted.tolist(), result.tokens.tolist()) == wants[k % 3]


def test_seeded_random_calls(device):
    rng = random.Random(11)
    for k in range(40):
        counts = [rng.choice([0, 1, rng.randint(1, 12)]) for _ in range(rng.randint(1, 12))]
        if sum(counts) == 0:
            counts[0] = 1
        vocab, dtype = int(math.exp(rng.uniform(0, math.log(20000)))), rng.choice([torch.float32, torch.bfloat16])
        given, kept, pad = rng.random() < 0.6, rng.choice([1.0, 0.05, 0.5]), rng.choice([0, 1, 8])
        print(k, counts, vocab, dtype, given, kept, pad, flush=True)
        check(device, *make(counts, vocab, dtype, 100 + k, kept=kept, pad=pad, given=given))


def test_refusals(device):
    target, tokens, uniforms, starts, draft = [x if isinstance(x, list) else x.to(device)
                                               for x in make([3, 2], 100, torch.float32, 1)]
    good = dict(target=target, tokens=tokens, uniforms=uniforms, draft=draft,
                query_start_loc=torch.tensor(starts, dtype=torch.int32, device=device))
    step_ops.verify_drafts(**good)
    for wrong in (dict(target=target.half()), dict(target=target.t().contiguous().t()), dict(target=target.cpu()),
                  dict(target=target[:1].expand(5, 100), draft=None), dict(draft=draft.to(torch.bfloat16)),
                  dict(draft=draft[:4]), dict(draft=draft[:, :99]), dict(draft=draft.cpu()), dict(tokens=tokens.int()),
                  dict(tokens=tokens[:4]), dict(uniforms=uniforms.double()), dict(uniforms=uniforms[:4]),
                  dict(uniforms=uniforms[:, None]), dict(query_start_loc=good["query_start_loc"].long()),
                  dict(query_start_loc=good["query_start_loc"][:0]),
                  dict(workspace=torch.empty(100, dtype=torch.uint8, device=device))):
        with pytest.raises(RuntimeError):
            step_ops.verify_drafts(**{**good, **wrong})
