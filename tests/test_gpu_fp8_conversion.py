"""Every BF16 value as an E4M3 code, at every power-of-two scale and at others, by each operator that converts."""

from __future__ import annotations

import pytest
import torch

from residualquant_amd import ops, step_ops

from . import fp8_reference

pytestmark = pytest.mark.gpu

# All finite BF16 values: 15 rows of 34 heads of 128.
FINITE = torch.arange(1 << 16, dtype=torch.int32).to(torch.uint16).view(torch.bfloat16)
FINITE = FINITE[FINITE.isfinite()]
HEADS, DIM, PAGE = 34, 128, 16
POWERS = [2.0 ** p for p in range(-126, 121)]
# What no writer makes, but a caller may: powers past 2^120 and other numbers.
OTHERS = [2.0 ** 121, 2.0 ** 125, 2.0 ** 127, 3.0 * 2.0 ** 100, 1.1, 0.7 * 2.0 ** -100, 5.0 * 2.0 ** -120, 448.0, 1.5 * 2.0 ** 120, torch.inf]


def _pages(scales, device):
    """A page per scale with one token in it, and the 15 rows to append: every finite value that the power of two
    at or below the scale keeps within 448 (so that the page's scale stays), else 0."""
    scales = torch.tensor(scales)
    values = FINITE.view(1, 15, HEADS, DIM).expand(len(scales), -1, -1, -1)
    power = torch.where(scales.isfinite(), torch.exp2(torch.frexp(scales.double()).exponent.double() - 1), torch.inf)
    fits = values.double().abs() <= 448.0 * power[:, None, None, None]
    key = torch.where(fits, values, torch.zeros((), dtype=torch.bfloat16))
    held = torch.full((2, len(scales), HEADS, PAGE, DIM), 0x38, dtype=torch.uint8)
    return dict(key=key, value=key.flip(3), scales=scales[None, :, None].expand(2, -1, HEADS).contiguous().to(device),
                cache=held.view(torch.float8_e4m3fn).to(device),
                starts=torch.arange(0, 15 * len(scales) + 1, 15, dtype=torch.int32, device=device),
                seq_lens=torch.full((len(scales),), 16, dtype=torch.int32, device=device),
                table=torch.arange(len(scales), dtype=torch.int32, device=device)[:, None].contiguous())


def _check(pages, given):
    scales = given.cpu()
    assert torch.equal(pages["scales"].cpu(), scales)  # (the page's own is large enough)
    got = pages["cache"].view(torch.uint8).cpu()
    assert bool((got[:, :, :, 0] == 0x38).all())
    for plane, rows in enumerate((pages["key"], pages["value"])):
        want = fp8_reference.e4m3_round(rows.float() / scales[plane, :, None, :, None]).view(torch.uint8)
        assert torch.equal(got[plane, :, :, 1:].transpose(1, 2), want)


@pytest.mark.parametrize("which", ["powers", "others"])
def test_quantize_every_value_at_every_scale(device, which):
    pages = _pages(POWERS if which == "powers" else OTHERS, device)
    given = pages["scales"].clone()
    ops.quantize_fp8(pages["key"].flatten(0, 1).to(device), pages["value"].flatten(0, 1).to(device), pages["cache"],
                     pages["scales"], pages["starts"], pages["seq_lens"], pages["table"])
    _check(pages, given)


@pytest.mark.parametrize("which", ["powers", "others"])
def test_append_every_value_at_every_scale(device, which):
    """Keys turned by an angle of 0: a x 1 - b x 0 is a."""
    pages = _pages(POWERS if which == "powers" else OTHERS, device)
    given, rows = pages["scales"].clone(), 15 * pages["key"].size(0)
    query = torch.zeros((rows, 2, DIM), dtype=torch.bfloat16)
    qkv = torch.cat([query, pages["key"].flatten(0, 1), pages["value"].flatten(0, 1)], 1).view(rows, -1).to(device)
    cos, sin = torch.ones((16, 8), device=device), torch.zeros((16, 8), device=device)
    _, key, _ = ops.rope_append(qkv, cos, sin, pages["cache"], pages["scales"], pages["starts"], pages["seq_lens"], pages["table"])
    # (A rotated 0 may have lost its sign.)
    assert torch.equal(key.cpu(), pages["key"].flatten(0, 1))
    pages["key"] = key.cpu().view(pages["key"].shape)
    _check(pages, given)


def test_project_every_value_at_every_scale(device):
    """Rows of 127 values and one of 448 x 2^p through the unit matrix: each value as its code times 2^p."""
    rows = -(-FINITE.numel() // 127)
    values = torch.zeros(rows * 127, dtype=torch.bfloat16)
    values[:FINITE.numel()] = FINITE
    unit = step_ops.quantize_weight_fp8(torch.eye(128, dtype=torch.bfloat16, device=device))
    for p in range(-126, 120):
        most = 448.0 * 2.0 ** p
        x = torch.full((rows, 128), most).to(torch.bfloat16)
        x[:, 1:] = torch.where(values.double().abs() <= most, values, torch.zeros((), dtype=torch.bfloat16)).view(rows, 127)
        x = x.roll(p, dims=1)  # (the largest in every place)
        want = fp8_reference.e4m3_round(x.float() / 2.0 ** p).double() * 2.0 ** p
        parts = [step_ops.linear_fp8(x.to(device), unit), step_ops.linear_fp8(x[:40].to(device), unit)]
        for got in parts:
            got, expected = got.double().cpu(), want[:got.size(0)]
            # (Below the normal range of FP32 a result may be 0.)
            low = expected.abs() < 2.0 ** -126
            assert torch.equal(torch.where(low, 0.0, got), torch.where(low, 0.0, expected)), p
            assert bool((got[low].abs() <= 2.0 ** -126).all()), p


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,page", [(128, 16), (96, 32)])
def test_append_against_the_formula(device, dim, page, interleaved):
    """The pages of a few requests by the definition on the host, which no kernel has a part in."""
    g = torch.Generator().manual_seed(dim + page)
    histories, rows, heads, kv_heads = [0, 5, 31, 40], [3, 30, 1, 17], 3, 2
    total, half = sum(rows), 32
    starts = torch.tensor([0] + [sum(rows[:b + 1]) for b in range(len(rows))], dtype=torch.int32)
    seq_lens = torch.tensor([h + n for h, n in zip(histories, rows)], dtype=torch.int32)
    qkv = torch.randn((total, heads + 2 * kv_heads, dim), generator=g)
    qkv[:, heads:, ::16] *= 20.0
    qkv = qkv.to(torch.bfloat16)
    angles = torch.rand((64, half), generator=g) * 6.0
    cos, sin = angles.cos(), angles.sin()
    at = torch.cat([torch.arange(h, h + n) for h, n in zip(histories, rows)])
    turned = qkv[:, :heads + kv_heads, :2 * half].float()
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    c, s = cos[at][:, None], sin[at][:, None]
    both = (a * c - b * s, b * c + a * s)
    turned = torch.stack(both, -1).flatten(-2) if interleaved else torch.cat(both, -1)
    want = torch.cat([turned.to(torch.bfloat16), qkv[:, :heads + kv_heads, 2 * half:]], -1)
    blocks = 4 * 5
    table = torch.randperm(blocks, generator=g).view(4, 5).to(torch.int32)
    cache = (torch.randn((2, blocks, kv_heads, page, dim), generator=g) * 90).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.exp2(torch.randint(-9, -3, (2, blocks, kv_heads), generator=g).float())
    on_cache, on_scales = cache.to(device), scales.to(device)
    query, key, value = ops.rope_append(qkv.view(total, -1).to(device), cos.to(device), sin.to(device), on_cache, on_scales,
                                        starts.to(device), seq_lens.to(device), table.to(device), interleaved=interleaved)
    assert torch.equal(query.cpu(), want[:, :heads]) and torch.equal(key.cpu(), want[:, heads:])
    fp8_reference.write(want[:, heads:], qkv[:, heads + kv_heads:], cache, scales, starts, seq_lens, table)
    assert torch.equal(on_cache.view(torch.uint8).cpu(), cache.view(torch.uint8)) and torch.equal(on_scales.cpu(), scales)
    assert torch.equal(value.cpu(), qkv[:, heads + kv_heads:])
