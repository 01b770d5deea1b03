"""The paged cache held in 8 bits (ops.quantize_fp8, ops.paged_attention_fp8) against float64 and byte-exact references."""

from __future__ import annotations

import pytest
import torch

from residualquant_amd import ops

from . import fp8_reference as reference

pytestmark = pytest.mark.gpu


def _case(histories, rows, heads, kv_heads, dim, page, seed, extra_pages=0, outlier=1.0):
    g = torch.Generator().manual_seed(seed)
    pages = max(1, -(-max(h + n for h, n in zip(histories, rows)) // page)) + extra_pages
    batch = len(histories)
    blocks = batch * pages + 3
    total = sum(rows)
    x = torch.randn((2, blocks, kv_heads, page, dim), generator=g) * outlier
    scales = torch.exp2(torch.randint(-8, -5, (2, blocks, kv_heads), generator=g).float())
    cache = (x / scales[..., None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    make = lambda h, scale=1.0: (torch.randn((total, h, dim), generator=g) * scale).to(torch.bfloat16)  # noqa: E731
    return {
        "query": make(heads, 1.5), "key": make(kv_heads), "value": make(kv_heads), "cache": cache, "scales": scales,
        "starts": torch.tensor(starts, dtype=torch.int32),
        "seq_lens": torch.tensor([h + n for h, n in zip(histories, rows)], dtype=torch.int32),
        "table": torch.randperm(blocks, generator=g)[:batch * pages].view(batch, pages).to(torch.int32),
    }


def _to(case, device):
    return {k: v.view(torch.uint8).to(device).view(torch.float8_e4m3fn) if v.dtype == torch.float8_e4m3fn
            else v.to(device) for k, v in case.items()}


def _attend(d, device, softmax_scale=None, workspace=None, output=None):
    out = torch.full_like(d["query"], torch.nan) if output is None else output
    ops.paged_attention_fp8(d["query"], d["key"], d["value"], d["cache"], d["scales"], out, d["starts"],
                            d["seq_lens"], d["table"], softmax_scale=softmax_scale, workspace=workspace)
    return out


def _check_attention(case, got, scale=None):
    dim = case["query"].size(2)
    want, bound = reference.attend(case["query"], case["key"], case["value"], case["cache"], case["scales"],
                                   case["starts"], case["seq_lens"], case["table"],
                                   dim ** -0.5 if scale is None else scale)
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), "NaN in other places"
    over = ((got - want).abs() / bound).nan_to_num(0.0)
    assert over.max() <= 1.0, f"{over.max():.2f} times the bound, {int((over > 1).sum())} of {over.numel()} over it"


ATTENTION = [
    # histories, new rows, heads, kv_heads, dim, page
    ([0], [1], 4, 4, 128, 16),
    ([1], [1], 1, 1, 128, 16),
    ([15, 16, 17], [1, 1, 1], 3, 3, 128, 16),
    ([31, 32, 33, 0, 100], [1, 1, 1, 1, 1], 5, 5, 96, 32),
    ([700, 3, 129, 64, 257], [1, 1, 1, 1, 1], 8, 2, 128, 32),
    ([333, 90], [1, 1], 24, 2, 96, 16),
    ([1500], [1], 2, 2, 128, 16),
    ([40, 0, 311], [3, 1, 0], 4, 4, 128, 16),
    ([77, 200], [7, 16], 4, 2, 96, 16),
    ([50, 0, 1], [33, 17, 64], 3, 3, 128, 32),
    ([130], [70], 8, 2, 96, 32),
    ([0, 0], [40, 5], 2, 1, 128, 16),
    ([257], [130], 2, 2, 128, 16),
    ([2050], [1], 16, 1, 128, 32),
    ([5], [300], 1, 1, 96, 16),
    ([1500], [100], 2, 2, 128, 16),
    ([2500, 70], [64, 130], 2, 1, 96, 32),
    ([1300, 1200], [40, 25], 1, 1, 128, 16),
    ([1700], [9], 4, 2, 96, 16),
]


@pytest.mark.parametrize("histories,rows,heads,kv_heads,dim,page", ATTENTION)
def test_attention(device, histories, rows, heads, kv_heads, dim, page):
    print(f"histories={histories} rows={rows} heads={heads}/{kv_heads} D={dim} PT={page}", flush=True)
    case = _case(histories, rows, heads, kv_heads, dim, page, seed=sum(histories) + 7 * sum(rows) + dim)
    _check_attention(case, _attend(_to(case, device), device))


def test_attention_of_many_requests(device):
    """More requests than a wave has lanes, some without rows."""
    g = torch.Generator().manual_seed(5)
    histories = torch.randint(0, 200, (131,), generator=g).tolist()
    rows = torch.randint(0, 3, (131,), generator=g).tolist()
    case = _case(histories, rows, 2, 2, 96, 16, seed=6)
    _check_attention(case, _attend(_to(case, device), device))


@pytest.mark.parametrize("rows", [[1, 1], [20, 9]])
def test_attention_softmax_scale_and_any_scales(device, rows):
    case = _case([90, 210], rows, 4, 2, 128, 16, seed=21)
    case["scales"] *= 0.7 + 0.3 * torch.rand(case["scales"].shape, generator=torch.Generator().manual_seed(1))
    _check_attention(case, _attend(_to(case, device), device, softmax_scale=0.31), scale=0.31)


@pytest.mark.parametrize("rows", [[1, 1], [4, 37]])
def test_attention_scales_far_apart(device, rows):
    """Value pages of very different sizes: no page's rounding shows in another's share."""
    case = _case([300, 180], rows, 4, 4, 128, 16, seed=22)
    g = torch.Generator().manual_seed(2)
    case["scales"][1] *= torch.exp2(torch.randint(-40, 40, case["scales"].shape[1:], generator=g).float())
    _check_attention(case, _attend(_to(case, device), device))
    # One page of huge values that no row attends to (its keys point away from every query).
    case = _case([64], [rows[1]], 1, 1, 128, 16, seed=23)
    case["query"] = case["query"].abs()
    first = int(case["table"][0, 1])
    case["cache"][0, first] = torch.full((1, 16, 128), -448.0).to(torch.float8_e4m3fn)
    case["scales"][1, first] = 2.0 ** 60
    _check_attention(case, _attend(_to(case, device), device))


@pytest.mark.parametrize("rows", [[1, 1, 1], [5, 1, 40]])
def test_attention_ignores_what_it_must_not_read(device, rows):
    """NaN bytes in slots past a history and in blocks of no request, and NaN scales of unused pages."""
    case = _case([35, 0, 96], rows, 4, 2, 128, 16, seed=31, extra_pages=2)
    page = 16
    used = torch.zeros(case["cache"].shape[1:4], dtype=torch.bool)
    for b, h in enumerate([35, 0, 96]):
        for t in range(h):
            used[int(case["table"][b, t // page]), :, t % page] = True
    raw = case["cache"].view(torch.uint8)
    raw[:, ~used] = 0x7F
    case["scales"][:, ~used.any(dim=2)] = torch.nan
    _check_attention(case, _attend(_to(case, device), device))


@pytest.mark.parametrize("rows", [[1, 1], [3, 30]])
def test_attention_skips_invalid_blocks(device, rows):
    case = _case([70, 50], rows, 2, 2, 128, 16, seed=32)
    case["table"][0, 1] = -1
    case["table"][0, 3] = case["cache"].size(1)
    case["table"][1, 0] = 1 << 30
    _check_attention(case, _attend(_to(case, device), device))


@pytest.mark.parametrize("rows", [[1, 1], [6, 21]])
def test_attention_leaves_rows_outside_alone(device, rows):
    case = _case([20, 90], rows, 2, 2, 96, 16, seed=33)
    d = _to(case, device)
    d |= {k: torch.cat([d[k][:2], d[k], d[k][:1], d[k][:2]]) for k in ("query", "key", "value")}
    d["starts"] = d["starts"] + 2
    out = torch.full_like(d["query"], 7.0)
    _attend(d, device, output=out)
    assert bool((out[:2] == 7.0).all()) and bool((out[-3:] == 7.0).all())
    _check_attention(case, out[2:-3])


@pytest.mark.parametrize("rows", [[1, 1], [4, 50]])
def test_attention_strided_tokens(device, rows):
    """Q/K/V as parts of one fused projection's rows, the output as part of wider rows."""
    case = _case([100, 30], rows, 4, 2, 128, 16, seed=34)
    d = _to(case, device)
    total = sum(rows)
    fused = torch.cat([d["query"].flatten(1), d["key"].flatten(1), d["value"].flatten(1),
                       torch.zeros((total, 4), dtype=torch.bfloat16, device=device)], dim=1)
    d["query"] = fused[:, :512].unflatten(1, (4, 128))
    d["key"] = fused[:, 512:768].unflatten(1, (2, 128))
    d["value"] = fused[:, 768:1024].unflatten(1, (2, 128))
    out = torch.zeros((total, 600), dtype=torch.bfloat16, device=device)
    _attend(d, device, output=out[:, 4:516].unflatten(1, (4, 128)))
    _check_attention(case, out[:, 4:516].unflatten(1, (4, 128)))
    assert bool((out[:, :4] == 0).all()) and bool((out[:, 516:] == 0).all())


@pytest.mark.parametrize("where", ["query", "key", "value", "cache", "late"])
@pytest.mark.parametrize("rows", [[1, 1], [3, 18]])
def test_attention_nan_and_infinity(device, where, rows):
    """A NaN reaches the rows that attend to it and no others; scores of -inf have no weight."""
    case = _case([40, 33], rows, 2, 2, 128, 16, seed=35)
    if where == "cache":
        raw = case["cache"].view(torch.uint8)
        raw[1, int(case["table"][0, 1]), 0, 2, 5] = 0x7F  # a value channel of one head
    elif where == "query":
        case["query"][0, 1, 3] = torch.nan
    elif where == "key":
        case["query"][:, :, 9] = case["query"][:, :, 9].abs() + 0.5
        case["key"][0, 1, 9] = -torch.inf
    elif where == "value":
        case["value"][0, 1, 9] = torch.inf
    else:  # the last of the request's new rows: earlier rows do not see it
        last = rows[0] - 1
        case["key"][last, 0, 3] = torch.nan
        case["value"][last, 1, 9], case["value"][last, 1, 64] = -torch.inf, torch.nan
    got = _attend(_to(case, device), device).cpu().double()
    want, bound = reference.attend(case["query"], case["key"], case["value"], case["cache"], case["scales"],
                                   case["starts"], case["seq_lens"], case["table"], 128 ** -0.5)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf())
    finite = want.isfinite()
    if where != "key":
        assert bool(((got - want).abs() <= bound)[finite].all())
    else:  # (the bound counts |q k|, which is infinite here)
        assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12)[finite].all())


def test_attention_past_the_page_table(device):
    """A history longer than the page table: what the table holds counts."""
    case = _case([96], [1], 2, 2, 128, 16, seed=36)
    case["seq_lens"] = case["seq_lens"] + 1000
    _check_attention(case, _attend(_to(case, device), device))


def test_attention_is_repeatable_and_takes_any_workspace(device):
    case = _case([3000, 60, 900], [1, 1, 1], 4, 4, 128, 16, seed=37)
    d = _to(case, device)
    first = _attend(d, device)
    needed = ops.paged_attention_fp8_workspace_bytes(3, 4, 4, 128, d["table"].size(1), 16)
    buffer = torch.full((needed + 64,), 0xFF, dtype=torch.uint8, device=device)
    for offset in (0, 1, 12):
        for _ in range(3):
            assert torch.equal(first, _attend(d, device, workspace=buffer[offset:offset + needed]))
    with pytest.raises(RuntimeError, match="Attention workspace of"):
        _attend(d, device, workspace=buffer[:needed - 1])
    _check_attention(case, first)


def test_attention_of_many_requests_with_many_columns(device):
    """More requests than a wave has lanes, with 0 to 90 rows: several tiles, whole and with splits."""
    g = torch.Generator().manual_seed(50)
    for longest, seed in ((40, 51), (700, 52)):
        histories = torch.randint(0, longest, (66,), generator=g).tolist()
        rows = torch.randint(0, 91, (66,), generator=g).tolist()
        rows[65] = 300
        case = _case(histories, rows, 2, 1, 96, 16, seed=seed)
        _check_attention(case, _attend(_to(case, device), device))


def test_attention_of_a_chunk_in_graphs_that_share_a_workspace(device):
    """Two graphs and eager calls, of one row and of many, take turns with one workspace; another stream."""
    many = _to(_case([1800, 700], [120, 300], 2, 2, 128, 16, seed=53), device)
    few = _to(_case([2000, 900, 4], [1, 1, 1], 2, 2, 128, 16, seed=54), device)
    needed = max(ops.paged_attention_fp8_workspace_bytes(d["query"].size(0), 2, 2, 128, d["table"].size(1), 16)
                 for d in (many, few))
    workspace = torch.full((needed,), 0xFF, dtype=torch.uint8, device=device)
    want = [_attend(d, device) for d in (many, few)]
    outs = [torch.zeros_like(d["query"]) for d in (many, few)]
    graphs = []
    for d, out in zip((many, few), outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _attend(d, device, workspace=workspace, output=out)
        graphs.append(graph)
    for turn in range(4):
        for k in ((0, 1), (1, 0), (0, 0), (1, 1))[turn]:
            outs[k].fill_(torch.nan)
            graphs[k].replay()
            assert torch.equal(outs[k], want[k]), f"turn {turn}"
            other = (many, few)[1 - k]
            assert torch.equal(_attend(other, device, workspace=workspace), want[1 - k]), f"eager, turn {turn}"
    stream = torch.cuda.Stream(device=device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        got = _attend(many, device, workspace=workspace)
    torch.cuda.current_stream(device).wait_stream(stream)
    assert torch.equal(got, want[0])


def test_attention_of_a_padded_batch(device):
    """Rows behind the last request keep what they held; requests of no tokens are none's."""
    case = _case([700, 0, 90, 0], [140, 0, 1, 0], 2, 2, 96, 32, seed=55)
    d = _to(case, device)
    pad = lambda t: torch.cat([t, torch.full((9, *t.shape[1:]), torch.nan, dtype=t.dtype, device=device)])  # noqa: E731
    d |= {k: pad(d[k]) for k in ("query", "key", "value")}
    out = torch.full_like(d["query"], 7.0)
    _attend(d, device, output=out)
    _check_attention(case, out[:141])
    assert bool((out[141:] == 7.0).all())


def test_attention_far_block(device):
    """A page whose byte offset passes 2^32."""
    blocks = (1 << 32) // (16 * 128) + 40  # one head: 2 KiB a page, two planes of over 4 GiB
    cache = torch.zeros((2, blocks, 1, 16, 128), dtype=torch.float8_e4m3fn, device=device)
    scales = torch.ones((2, blocks, 1), device=device)
    small = _case([40], [1], 1, 1, 128, 16, seed=38)
    d = _to(small, device)
    places = torch.tensor([blocks - 1, 3, blocks - 17])
    for i, place in enumerate(places.tolist()):
        source = int(small["table"][0, i])
        cache.view(torch.uint8)[:, place] = d["cache"].view(torch.uint8)[:, source]
        scales[:, place] = d["scales"][:, source]
    d |= {"cache": cache, "scales": scales, "table": places[None].to(torch.int32).to(device)}
    _check_attention(small, _attend(d, device))
    ops.quantize_fp8(d["key"], d["value"], cache, scales, d["starts"], d["seq_lens"], d["table"])
    want_cache, want_scales = small["cache"].clone(), small["scales"].clone()
    reference.write(small["key"], small["value"], want_cache, want_scales, small["starts"], small["seq_lens"],
                    small["table"])
    last = int(small["table"][0, 2])
    assert torch.equal(cache.view(torch.uint8)[:, blocks - 17].cpu(), want_cache.view(torch.uint8)[:, last])
    assert torch.equal(scales[:, blocks - 17].cpu(), want_scales[:, last])


def test_attention_on_another_stream_and_graph(device):
    """The call follows the current stream; a captured call replays on new inputs."""
    case = _case([500, 20], [1, 1], 4, 4, 128, 16, seed=39)
    d = _to(case, device)
    want = _attend(d, device)
    stream = torch.cuda.Stream(device=device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        other = _attend(d, device)
    torch.cuda.current_stream(device).wait_stream(stream)
    assert torch.equal(want, other)
    graphs, outs = [], []
    for _ in range(2):
        out = torch.zeros_like(d["query"])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _attend(d, device, output=out)
        graphs.append(graph)
        outs.append(out)
    for step in range(3):
        second = _case([500 - step, 20 + step], [1, 1], 4, 4, 128, 16, seed=40 + step)
        fresh = _to(second, device)
        for k in ("query", "key", "value", "scales", "starts", "seq_lens", "table"):
            d[k][tuple(slice(0, s) for s in fresh[k].shape)].copy_(fresh[k])
        d["cache"].view(torch.uint8)[:, :fresh["cache"].size(1)].copy_(fresh["cache"].view(torch.uint8))
        for graph, out in zip(graphs, outs):
            graph.replay()
        eager = _attend(d, device)
        torch.cuda.synchronize()
        for out in outs:
            assert torch.equal(out, eager), f"replay {step}"


# ---------------------------------------------------------------- write


def _check_write(case, device, repeat=1):
    d = _to(case, device)
    for _ in range(repeat):
        ops.quantize_fp8(d["key"], d["value"], d["cache"], d["scales"], d["starts"], d["seq_lens"], d["table"])
    cache, scales = case["cache"].clone(), case["scales"].clone()
    reference.write(case["key"], case["value"], cache, scales, case["starts"], case["seq_lens"], case["table"])
    assert torch.equal(d["scales"].cpu(), scales)
    got, want = d["cache"].view(torch.uint8).cpu(), cache.view(torch.uint8)
    nan = (got & 0x7F == 0x7F) & (want & 0x7F == 0x7F)  # a NaN's sign is free
    assert bool(((got == want) | nan).all()), int(((got != want) & ~nan).sum())
    return d


WRITES = [
    ([0], [1], 1, 128, 16), ([15], [1], 2, 128, 16), ([16], [1], 2, 96, 16), ([3, 31, 32, 0], [1, 1, 1, 1], 3, 96, 32),
    ([0], [40], 2, 128, 16), ([5, 0, 9], [50, 0, 3], 4, 128, 16), ([30, 1], [33, 64], 2, 96, 32),
    ([100] * 70, [1] * 70, 1, 128, 16), ([7] * 3, [16, 9, 25], 5, 96, 16),
]


@pytest.mark.parametrize("outlier", [1.0, 100.0])
@pytest.mark.parametrize("histories,rows,heads,dim,page", WRITES)
def test_write(device, histories, rows, heads, dim, page, outlier):
    print(f"histories={histories[:5]} rows={rows[:5]} heads={heads} D={dim} PT={page} outlier={outlier}", flush=True)
    case = _case(histories, rows, heads, heads, dim, page, seed=sum(histories) + dim + page, extra_pages=1)
    case["key"] = (case["key"].float() * outlier).to(torch.bfloat16)
    _check_write(case, device)
    _check_write(case, device, repeat=2)  # the same bytes again


def test_write_special_values(device):
    case = _case([4, 20], [9, 3], 2, 2, 128, 16, seed=51)
    key, value = case["key"], case["value"]
    key[0, 0, 0], key[1, 0, 1], key[2, 0, 2] = torch.nan, torch.inf, -torch.inf
    key[:, 1] = 0.0                                  # a page of zeros
    value[0, 0] = torch.tensor(3.3e38)               # the top of BF16
    value[:, 1] = 1e-40                              # subnormal values alone
    key[9:, 0] = torch.nan                           # no finite value in the page's new rows
    value[9:, 0, 0], value[9:, 0, 1] = 448.0, 449.0  # at and just over a power of two's range
    _check_write(case, device)


def test_write_every_code(device):
    """Every finite E4M3 value and every midpoint of two, both signs, at several scales, as the conversion rounds them."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    points = torch.cat([codes, (codes[1:] + codes[:-1]) / 2])
    points = torch.cat([points, -points])
    points = torch.cat([points, torch.zeros(512 - points.numel())])
    for power in (-20, -3, 0, 11):
        case = _case([0], [4], 1, 1, 128, 16, seed=52)
        case["key"] = (points * 2.0 ** power).to(torch.bfloat16).view(4, 1, 128)
        case["key"][0, 0, 0] = 448.0 * 2.0 ** power
        case["value"] = case["key"] * 0.5
        _check_write(case, device)


def test_write_rescales_every_code(device):
    """A larger value makes the scale grow by 1 to 20 powers of two: older codes of every value are rounded again."""
    for power in (1, 2, 3, 7, 20):
        case = _case([4], [1], 1, 1, 128, 16, seed=53)
        block = int(case["table"][0, 0])
        codes = (torch.arange(512) % 256).to(torch.uint8)
        codes[codes & 0x7F == 0x7F] = 0
        case["cache"].view(torch.uint8)[:, block, 0, :4] = codes.view(4, 128)
        case["scales"][:, block] = 1.0
        case["key"][0, 0, 0] = case["value"][0, 0, 7] = 448.0 * 2.0 ** power
        _check_write(case, device)


def test_write_skips_what_has_no_page(device):
    case = _case([30, 14], [20, 10], 2, 2, 128, 16, seed=54)
    case["table"][0, 2] = -1
    case["table"][1, 1] = case["cache"].size(1) + 7
    _check_write(case, device)
    case = _case([30], [20], 2, 2, 128, 16, seed=55)
    case["table"] = case["table"][:, :3].contiguous()  # positions 48 and 49 lie past the table
    _check_write(case, device)


def test_write_rows_outside_and_strides(device):
    case = _case([9, 0], [12, 30], 2, 2, 96, 16, seed=56)
    wide = torch.randn((42 + 6, 2 * 2 * 96 + 8), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    case["key"], case["value"] = wide[:, :192].unflatten(1, (2, 96)), wide[:, 192:384].unflatten(1, (2, 96))
    case["starts"] = case["starts"] + 4
    d = _to({k: v for k, v in case.items() if k not in ("key", "value")}, device)
    on = wide.to(device)
    d["key"], d["value"] = on[:, :192].unflatten(1, (2, 96)), on[:, 192:384].unflatten(1, (2, 96))
    ops.quantize_fp8(d["key"], d["value"], d["cache"], d["scales"], d["starts"], d["seq_lens"], d["table"])
    cache, scales = case["cache"].clone(), case["scales"].clone()
    reference.write(case["key"], case["value"], cache, scales, case["starts"], case["seq_lens"], case["table"])
    assert torch.equal(d["cache"].view(torch.uint8).cpu(), cache.view(torch.uint8))
    assert torch.equal(d["scales"].cpu(), scales)


def test_refusals_on_the_device(device):
    d = _to(_case([20], [1], 4, 2, 128, 16, seed=57), device)
    call = lambda **other: _attend({**d, **other}, device)  # noqa: E731
    for wrong in (dict(cache=d["cache"].view(torch.uint8)), dict(scales=d["scales"].double()),
                  dict(scales=d["scales"][:, :, :1]), dict(cache=d["cache"].cpu()), dict(key=d["key"].float()),
                  dict(starts=d["starts"].long()), dict(seq_lens=d["seq_lens"].cpu()), dict(table=d["table"].long()),
                  dict(value=d["value"][:, :1])):
        with pytest.raises(RuntimeError):
            call(**wrong)
    with pytest.raises(RuntimeError, match="multiple of key/value heads"):
        three = torch.zeros((1, 3, 128), dtype=torch.bfloat16, device=device)
        call(query=three)
    with pytest.raises(RuntimeError):
        ops.quantize_fp8(d["key"], d["value"][:, :1], d["cache"], d["scales"], d["starts"], d["seq_lens"], d["table"])


# ---------------------------------------------------------------- attention at the ends of the range


@pytest.mark.parametrize("histories,rows", [([300, 181], [1, 1]), ([300, 181], [4, 37]), ([3000], [1]), ([2000, 60], [100, 130]),
                                            ([0, 40], [1, 90])])
def test_attention_of_huge_values(device, histories, rows):
    """Values up to 2^127, all of one sign, whose sum passes FP32 and whose average does not; the heads beside
    hold values of 1 and of 2^-100."""
    print(f"histories={histories} rows={rows}", flush=True)
    case = _case(histories, rows, 6, 3, 128, 16, seed=61)
    raw = case["cache"].view(torch.uint8)
    raw[1] &= 0x7F  # positive values
    for head, power in enumerate((2.0 ** 124, 1.0, 2.0 ** -100)):
        case["scales"][1, :, head] *= power
        case["value"][:, head] = (case["value"][:, head].float().abs() * power).to(torch.bfloat16)
    _check_attention(case, _attend(_to(case, device), device))


@pytest.mark.parametrize("rows", [[1], [5], [40], [150]])
@pytest.mark.parametrize("where", ["early", "late", "new"])
def test_attention_of_huge_values_in_one_place(device, rows, where):
    """One page or one new row of values near the top of BF16 among ordinary ones, seen by one wave or split only."""
    case = _case([2600], rows, 2, 2, 96, 32, seed=62)
    if where == "new":
        case["value"][rows[0] // 2] = (case["value"][rows[0] // 2].float().abs() * 2.0 ** 125).to(torch.bfloat16)
    else:
        block = int(case["table"][0, 1 if where == "early" else 2600 // 32 - 2])
        case["scales"][1, block] *= 2.0 ** 124
    _check_attention(case, _attend(_to(case, device), device))


@pytest.mark.parametrize("rows", [[1, 1], [3, 30], [90, 1]])
@pytest.mark.parametrize("size", [1e6, 1e10, 1e14, 1e25])
def test_attention_of_large_scores(device, rows, size):
    """Scores of 10^7 and more, whose largest stands alone: its value comes out."""
    case = _case([300, 181], rows, 2, 2, 128, 16, seed=63)
    case["query"] = (case["query"].float() * size).to(torch.bfloat16)
    query, scales, table = case["query"].double(), case["scales"].double(), case["table"]
    want, gaps = torch.zeros_like(query), []
    for b, (h, n) in enumerate(zip([300, 181], rows)):
        begin = sum(rows[:b])
        blocks = table[b, [t // 16 for t in range(h)]].long()
        slots = torch.tensor([t % 16 for t in range(h)])
        for head in range(2):
            held = [case["cache"].view(torch.uint8)[p, blocks, head, slots].view(torch.float8_e4m3fn).double()
                    * scales[p, blocks, head][:, None] for p in range(2)]
            for i in range(n):
                k, v = (torch.cat([x, case[name][begin:begin + i + 1, head].double()]) for x, name in zip(held, ("key", "value")))
                q = query[begin + i, head]
                scores = k @ q * 128 ** -0.5
                first, second = scores.topk(2).values
                # Its lead over the rounding of a score: 128 products summed in float32, and a factor.
                gaps.append((first - second) - 2 * 140 * 2.0 ** -24 * float((k.abs() @ q.abs()).max()) * 128 ** -0.5)
                want[begin + i, head] = v[scores.argmax()]
    clear = torch.tensor(gaps).view(-1) > 30
    assert clear.float().mean() > 0.9
    # (In the order of the gaps: request, head, row.)
    order = [(sum(rows[:b]) + i, head) for b, n in enumerate(rows) for head in range(2) for i in range(n)]
    got = _attend(_to(case, device), device).cpu().double()
    for (row, head), sure in zip(order, clear.tolist()):
        if sure:  # one BF16 rounding, and weights of two BF16 parts
            assert bool(((got[row, head] - want[row, head]).abs() <= 2.0 ** -7 * want[row, head].abs() + 2.0 ** -10).all()), (row, head)
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("rows", [[1], [40]])
def test_attention_of_large_equal_scores(device, rows):
    """Equal keys: equal weights, whatever the size of the scores."""
    for sign, power in ((1, 12), (1, 30), (-1, 30), (1, 60), (-1, 60), (1, 100)):
        case = _case([333], rows, 1, 1, 128, 16, seed=64)
        case["cache"][0] = torch.ones(case["cache"][0].shape).to(torch.float8_e4m3fn)
        case["scales"][0] = 2.0 ** -3
        case["query"] = torch.full_like(case["query"], sign * 1.5 * 2.0 ** power)
        case["key"] = torch.full_like(case["key"], -3.0 if sign > 0 else 6.0)  # far below the others
        blocks = case["table"][0, [t // 16 for t in range(333)]].long()
        slots = torch.tensor([t % 16 for t in range(333)])
        v = case["cache"].view(torch.uint8)[1, blocks, 0, slots].view(torch.float8_e4m3fn).double()
        v = v * case["scales"][1, blocks, 0].double()[:, None]
        got = _attend(_to(case, device), device).cpu().double()
        bound = 2.0 ** -8 * v.mean(0).abs() + (2.0 ** -16 + 100 * 2.0 ** -23) * v.abs().mean(0)
        assert bool(((got[:, 0] - v.mean(0)).abs() <= bound).all()), (sign, power)


@pytest.mark.parametrize("rows", [[1, 1], [3, 90]])
def test_attention_of_scores_that_vanish(device, rows):
    """A softmax scale so small that a page's scale times it underflows: every token has the same weight."""
    case = _case([300, 181], rows, 2, 2, 128, 16, seed=65)
    case["scales"][0] *= 2.0 ** -20
    for scale in (1e-30, 1e-38, 1e-44):
        _check_attention(case, _attend(_to(case, device), device, softmax_scale=scale), scale=scale)
