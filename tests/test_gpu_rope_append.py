"""Rotation of a call's q and k with K/V appended to a paged cache (ops.rope_append)."""

from __future__ import annotations

import random

import pytest
import torch

from residualquant_amd import ops, step_ops

pytestmark = pytest.mark.gpu


def tables(positions, rotary, device):
    half = rotary // 2
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(half, dtype=torch.float64) / half)
    return angles.cos().float().to(device), angles.sin().float().to(device)


def rotated(x, cos, sin, interleaved):
    """BF16 [rows, heads, D]; products and sums rounded to float32, then BF16: the definition, bit for bit."""
    half = cos.size(1)
    turned = x[..., :2 * half].float()
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    c, s = cos[:, None], sin[:, None]
    parts = (a * c - b * s, b * c + a * s)
    turned = torch.stack(parts, -1).flatten(-2) if interleaved else torch.cat(parts, -1)
    return torch.cat([turned.to(torch.bfloat16), x[..., 2 * half:]], -1)


class Call:
    def __init__(self, device, histories, rows, heads, kv_heads, dim, page, eight, seed=0, lead=0, tail=0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page, self.eight = heads, kv_heads, dim, page, eight
        self.histories, self.rows = histories, rows
        total = lead + sum(rows) + tail
        x = torch.randn((total, heads + 2 * kv_heads, dim), generator=g)
        x[:, heads:heads + kv_heads, ::32] *= 9.0
        self.qkv = x.to(torch.bfloat16).view(total, -1).to(device)
        starts = [lead]
        for n in rows:
            starts.append(starts[-1] + n)
        self.starts = torch.tensor(starts, dtype=torch.int32, device=device)
        self.seq_lens = torch.tensor([h + n for h, n in zip(histories, rows)], dtype=torch.int32, device=device)
        self.positions = torch.tensor([h + k for h, n in zip(histories, rows) for k in range(n)])
        pages = max(1, max(-(-(h + n) // page) for h, n in zip(histories, rows)))
        blocks = len(rows) * pages + 2
        self.table = torch.randperm(blocks, generator=g)[:len(rows) * pages].view(len(rows), pages).to(torch.int32).to(device)
        shape = (2, blocks, kv_heads, page, dim)
        values = torch.randn(shape, generator=g)
        if eight:
            self.scales = torch.exp2(torch.randint(-9, -5, shape[:3], generator=g).float()).to(device)
            self.cache = (values * 90).to(torch.float8_e4m3fn).to(device)
        else:
            self.scales, self.cache = None, values.to(torch.bfloat16).to(device)

    def parts(self):
        x = self.qkv.view(-1, self.heads + 2 * self.kv_heads, self.dim).cpu()
        return x[:, :self.heads], x[:, self.heads:self.heads + self.kv_heads], x[:, self.heads + self.kv_heads:]

    def bytes(self):
        return self.cache.view(torch.uint8 if self.eight else torch.int16).cpu()


def check(call, device, rotary, interleaved, positions=None, max_positions=None, **more):
    lead, total = int(call.starts[0]), call.qkv.size(0)
    n = sum(call.rows)
    inside = slice(lead, lead + n)
    most = max_positions or int(call.positions.max()) + 1 if n else 1
    cos, sin = tables(most, rotary, device)
    at = (call.positions if positions is None else positions.cpu()[inside]).clamp(0, most - 1)
    q, k, v = call.parts()
    want_q = rotated(q[inside], cos.cpu()[at], sin.cpu()[at], interleaved)
    want_k = rotated(k[inside], cos.cpu()[at], sin.cpu()[at], interleaved)
    # The cache as the separate writers leave it.
    cache, scales = call.cache.clone(), None if call.scales is None else call.scales.clone()
    if call.eight:
        key = torch.zeros((total, call.kv_heads, call.dim), dtype=torch.bfloat16)
        key[inside] = want_k
        ops.quantize_fp8(key.to(device), v.contiguous().to(device), cache, scales, call.starts, call.seq_lens, call.table)
    else:
        row = 0
        for b, (h, count) in enumerate(zip(call.histories, call.rows)):
            for t in range(h, h + count):
                if t // call.page < call.table.size(1):
                    block = int(call.table[b, t // call.page])
                    if 0 <= block < cache.size(1):
                        cache[0, block, :, t % call.page] = want_k[row].to(device)
                        cache[1, block, :, t % call.page] = v[lead + row].to(device)
                row += 1
    query = torch.full((total, call.heads, call.dim), 5.0, dtype=torch.bfloat16, device=device)
    key = torch.full((total, call.kv_heads, call.dim), 6.0, dtype=torch.bfloat16, device=device)
    for _ in range(2):  # (a repeated call writes the same)
        got_q, got_k, got_v = ops.rope_append(call.qkv, cos, sin, call.cache, call.scales, call.starts, call.seq_lens,
                                              call.table, positions=positions, interleaved=interleaved, query=query,
                                              key=key, **more)
        assert torch.equal(got_q[inside].cpu(), want_q) and torch.equal(got_k[inside].cpu(), want_k)
        assert torch.equal(got_v.cpu(), v) and got_v.data_ptr() == call.qkv.data_ptr() + 2 * (call.heads + call.kv_heads) * call.dim
        for x, fill in ((query, 5.0), (key, 6.0)):
            assert bool((x[:lead] == fill).all()) and bool((x[lead + n:] == fill).all())
        assert torch.equal(call.bytes(), cache.view(call.bytes().dtype).cpu())
        if call.eight:
            assert torch.equal(call.scales, scales)


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,page,rotary", [(4, 4, 128, 16, 128), (8, 2, 128, 32, 64), (5, 5, 96, 16, 96),
                                                            (6, 1, 96, 32, 32), (1, 3, 128, 16, 16)])
def test_append(device, heads, kv_heads, dim, page, rotary, interleaved, eight):
    print(f"{heads}/{kv_heads} x {dim} page {page} rotary {rotary} interleaved {interleaved} eight {eight}", flush=True)
    for histories, rows in (([0], [1]), ([15, 16, 17, 0, 31], [1, 1, 1, 1, 1]), ([3, 0, 40, 33], [0, 50, 5, 17]),
                            ([1000], [130]), ([7] * 70, [1] * 70)):
        check(Call(device, histories, rows, heads, kv_heads, dim, page, eight, seed=len(rows)), device, rotary, interleaved)


@pytest.mark.parametrize("eight", [True, False])
def test_rows_outside_the_requests(device, eight):
    check(Call(device, [5, 16], [3, 20], 4, 2, 128, 16, eight, lead=3, tail=6), device, 128, False)


@pytest.mark.parametrize("eight", [True, False])
def test_given_positions(device, eight):
    """Positions of any kind; those outside the tables take their ends."""
    call = Call(device, [5, 100], [3, 20], 4, 2, 128, 16, eight)
    g = torch.Generator().manual_seed(1)
    positions = torch.randint(-5, 300, (23,), generator=g)
    positions[0], positions[1] = 2 ** 62, -2 ** 62
    check(call, device, 128, True, positions=positions.to(device), max_positions=200)
    check(call, device, 64, False, max_positions=50)


@pytest.mark.parametrize("eight", [True, False])
def test_pages_that_are_not_there(device, eight):
    """Tokens without a page, or on an invalid block, are rotated and not stored."""
    call = Call(device, [10, 20, 30], [10, 40, 3], 4, 4, 128, 16, eight)
    call.table = call.table[:, :3].contiguous()
    call.table[0, 0], call.table[1, 2] = -1, 1000
    if not eight:
        check(call, device, 128, False)
        return
    check(call, device, 128, False)


def test_strided_rows(device):
    """qkv, query and key as parts of wider rows, on 8-byte boundaries."""
    call = Call(device, [5, 33], [4, 9], 4, 2, 96, 16, True)
    wide = torch.full((13, call.qkv.size(1) + 12), 7.0, dtype=torch.bfloat16, device=device)
    wide[:, 4:4 + call.qkv.size(1)] = call.qkv
    cos, sin = tables(50, 96, device)
    cache, scales = call.cache.clone(), call.scales.clone()
    want = ops.rope_append(call.qkv, cos, sin, cache, scales, call.starts, call.seq_lens, call.table)
    both = torch.full((13, 6 * 96 + 4), 9.0, dtype=torch.bfloat16, device=device)
    apart = torch.full((13, 2 * 96 + 4), 9.0, dtype=torch.bfloat16, device=device)
    query, key = both[:, 4:4 + 4 * 96].view(13, 4, 96), apart[:, :2 * 96].view(13, 2, 96)
    got = ops.rope_append(wide[:, 4:4 + call.qkv.size(1)], cos, sin, call.cache, call.scales, call.starts, call.seq_lens,
                          call.table, query=query, key=key)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(call.bytes(), cache.view(torch.uint8).cpu()) and torch.equal(call.scales, scales)
    assert bool((both[:, :4] == 9).all()) and bool((both[:, 4 + 4 * 96:] == 9).all()) and bool((apart[:, 2 * 96:] == 9).all())


def test_values_that_are_not_finite(device):
    call = Call(device, [5, 33], [4, 9], 4, 2, 128, 16, True)
    call.qkv.view(13, 8, 128)[2, 5, 3] = torch.nan
    call.qkv.view(13, 8, 128)[6, 4, 70] = torch.inf
    call.qkv.view(13, 8, 128)[7, 7, 9] = -torch.inf
    cos, sin = tables(50, 128, device)
    cache, scales = call.cache.clone(), call.scales.clone()
    q, k, v = ops.rope_append(call.qkv, cos, sin, cache, scales, call.starts, call.seq_lens, call.table)
    ops.quantize_fp8(k, v.contiguous(), call.cache, call.scales, call.starts, call.seq_lens, call.table)
    assert torch.equal(call.bytes(), cache.view(torch.uint8).cpu()) and torch.equal(call.scales, scales)
    assert bool(k[2].isnan().any()) and bool(scales.isfinite().all())


def test_like_the_separate_rotation(device):
    """As step_ops.rope_qkv up to the last rounding (whose products may be fused): one BF16 step of the larger channel."""
    call = Call(device, [40], [30], 4, 4, 128, 16, False)
    cos, sin = tables(70, 128, device)
    q, k = step_ops.rope_qkv(call.qkv, call.positions.to(device), cos, sin, 4, 128)
    query, key, _ = ops.rope_append(call.qkv, cos, sin, call.cache, None, call.starts, call.seq_lens, call.table)
    for a, b in ((q, query), (k, key)):
        size = torch.maximum(a.float().abs(), b.float().abs())
        sizes = call.qkv.float().abs().max() * 2.0 ** -22
        assert bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * size + sizes).all())


def test_seeded_random_calls(device):
    rng = random.Random(5)
    for k in range(30):
        heads, kv_heads, dim = rng.choice([(4, 4, 128), (8, 2, 128), (3, 1, 96), (5, 5, 96)])
        batch = rng.randint(1, 9)
        histories = [rng.choice([0, rng.randint(0, 200)]) for _ in range(batch)]
        rows = [rng.choice([0, 1, rng.randint(1, 80)]) for _ in range(batch)]
        if sum(rows) == 0:
            rows[0] = 1
        page, eight = rng.choice([16, 32]), rng.random() < 0.6
        rotary, interleaved = rng.choice([16, 48, 96]), rng.random() < 0.5
        print(k, histories, rows, heads, kv_heads, dim, page, eight, rotary, interleaved, flush=True)
        check(Call(device, histories, rows, heads, kv_heads, dim, page, eight, seed=k, lead=rng.choice([0, 2]),
                   tail=rng.choice([0, 3])), device, rotary, interleaved)


@pytest.mark.parametrize("eight", [True, False])
def test_captured_and_replayed(device, eight):
    call = Call(device, [5, 33, 16], [1, 9, 2], 4, 2, 128, 16, eight)
    cos, sin = tables(60, 128, device)
    arguments = (call.qkv, cos, sin, call.cache, call.scales, call.starts, call.seq_lens, call.table)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.rope_append(*arguments)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, k, v = ops.rope_append(*arguments)
    for seed in range(4):
        other = Call(device, [5, 33, 16], [1, 9, 2], 4, 2, 128, 16, eight, seed=seed + 50)
        call.qkv.copy_(other.qkv)
        call.seq_lens.add_(1 if seed else 0)
        cache, scales = call.cache.clone(), None if call.scales is None else call.scales.clone()
        want = ops.rope_append(call.qkv, cos, sin, cache, scales, call.starts, call.seq_lens, call.table)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        assert torch.equal(call.bytes(), cache.view(call.bytes().dtype).cpu())
        assert scales is None or torch.equal(call.scales, scales)


def test_query_and_key_side_by_side(device):
    call = Call(device, [5, 33], [4, 9], 4, 2, 128, 16, True)
    cos, sin = tables(50, 128, device)
    before, scales = call.cache.clone(), call.scales.clone()
    rest = (call.starts, call.seq_lens, call.table)
    query, key, _ = ops.rope_append(call.qkv, cos, sin, call.cache, call.scales, *rest)
    both = torch.full((13, 6 * 128 + 4), 7.0, dtype=torch.bfloat16, device=device)
    ops.rope_append(call.qkv, cos, sin, before, scales, *rest, query=both[:, :512].view(13, 4, 128), key=both[:, 512:768].view(13, 2, 128))
    assert torch.equal(both[:, :512], query.reshape(13, -1)) and torch.equal(both[:, 512:768], key.reshape(13, -1))
    assert torch.equal(before.view(torch.uint8), call.cache.view(torch.uint8)) and torch.equal(scales, call.scales)
    assert bool((both[:, 768:] == 7.0).all())


def test_refusals(device):
    call = Call(device, [5, 33], [4, 9], 4, 2, 128, 16, True)
    cos, sin = tables(50, 128, device)
    good = dict(qkv=call.qkv, cos=cos, sin=sin, cache=call.cache, scales=call.scales, query_start_loc=call.starts,
                seq_lens=call.seq_lens, block_table=call.table)
    ops.rope_append(**good)
    narrow = call.qkv[:, :-128]
    in_place = call.qkv[:, :4 * 128].view(13, 4, 128)
    for wrong in (dict(qkv=call.qkv.float()), dict(qkv=narrow[:, :-100]), dict(qkv=call.qkv[:, :3 * 128]),
                  dict(cos=cos[:, :60].contiguous()), dict(cos=cos.double(), sin=sin.double()), dict(sin=sin.cpu()),
                  dict(cos=cos[:, :12].contiguous(), sin=sin[:, :12].contiguous()), dict(scales=None),
                  dict(scales=call.scales[:1]), dict(cache=call.cache.view(torch.uint8)),
                  dict(cache=call.cache.float().to(torch.bfloat16)), dict(positions=call.positions[:5].to(device)),
                  dict(positions=call.positions.int().to(device)), dict(query=in_place), dict(seq_lens=call.seq_lens[:1]),
                  dict(key=torch.empty((13, 3, 128), dtype=torch.bfloat16, device=device)),
                  dict(query=torch.empty((13, 4, 128), device=device)), dict(block_table=call.table.long())):
        with pytest.raises(RuntimeError):
            ops.rope_append(**{**good, **wrong})
    both = torch.empty((13, 6, 128), dtype=torch.bfloat16, device=device)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.rope_append(**good, query=both.view(-1)[:13 * 4 * 128].view(13, 4, 128), key=both.view(-1)[512:512 + 13 * 256].view(13, 2, 128))
