"""8-bit projections, rotated appends and verification of drafts where offsets pass 31 and 32 bits."""

from __future__ import annotations

import pytest
import torch

from residualquant_amd import ops, step_ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _give_memory_back(device):
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def whole(shape, low, high, seed):
    return torch.randint(low, high + 1, shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def test_results_past_31_bits(device):
    """More than 2^31 results; whole numbers, whose sums (up to 72 x 24) FP32 holds exactly."""
    rows, out, features = 43000, 50257, 72
    x, values = whole((rows, features), -8, 8, 1), whole((out, features), -3, 3, 2)
    scales = torch.ones((-(-out // 128), 1), device=device)
    weight = step_ops.pack_weight_fp8(values.float().to(torch.float8_e4m3fn).to(device), scales)
    got = step_ops.linear_fp8(x.to(device), weight)
    assert got.numel() > 1 << 31
    at = torch.cat([torch.arange(40), torch.arange(21000, 21040), torch.arange(rows - 130, rows)])
    assert torch.equal(got[at.to(device)].cpu(), (x[at].float() @ values.float().t()).to(torch.bfloat16))


def test_weights_past_32_bits(device):
    """More than 2^32 codes, 0, 1 and 128: sums are whole numbers up to 2^21 x 2^2, exact in FP32 as in the products' sums of
    16 (128 x 8 has the smallest product, 1, within 2^-13)."""
    out, features = (1 << 21) + 70, 2048
    g = torch.Generator(device=device).manual_seed(3)
    codes = torch.randint(0, 3, (out, features), generator=g, device=device, dtype=torch.uint8)
    codes.mul_(0x38)
    assert codes.numel() > 1 << 32
    exponents = torch.randint(125, 130, (-(-out // 128), features // 128), generator=torch.Generator().manual_seed(4), dtype=torch.uint8)
    weight = step_ops.pack_weight_fp8(codes.view(torch.float8_e4m3fn), exponents.view(torch.float8_e8m0fnu).to(device))
    tails = [(0, 40), (1 << 20, (1 << 20) + 40), (out - 300, out)]
    held = []
    for begin, end in tails:
        scale = torch.exp2(exponents.double() - 127)[torch.arange(begin, end) // 128].repeat_interleave(128, 1)
        held.append(codes[begin:end].cpu().view(torch.float8_e4m3fn).double() * scale)
    del codes
    for rows in (3, 100, 600):
        print(f"rows={rows}", flush=True)
        x = whole((rows, features), -8, 8, rows)
        got = step_ops.linear_fp8(x.to(device), weight)
        for (begin, end), values in zip(tails, held):
            assert torch.equal(got[:, begin:end].cpu(), (x.double() @ values.t()).float().to(torch.bfloat16)), (rows, begin)


def test_cache_past_32_bits(device):
    """Blocks at the end of a cache of more than 2^32 bytes take what the same blocks of a small one take."""
    heads = kv_heads = 16
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn((23, 3 * heads * 128), generator=g).to(torch.bfloat16).to(device)
    angles = torch.rand((60, 64), generator=g) * 6.0
    cos, sin = angles.cos().to(device), angles.sin().to(device)
    starts = torch.tensor([0, 20, 23], dtype=torch.int32, device=device)
    seq_lens = torch.tensor([20 + 9, 3], dtype=torch.int32, device=device)
    blocks = 70000
    for eight in (True, False):
        dtype = torch.float8_e4m3fn if eight else torch.bfloat16
        small = torch.zeros((2, 4, kv_heads, 16, 128), dtype=dtype, device=device)
        large = torch.zeros((2, blocks, kv_heads, 16, 128), dtype=dtype, device=device)
        assert large.numel() > 1 << 32
        of_small = torch.ones((2, 4, kv_heads), device=device) if eight else None
        of_large = torch.ones((2, blocks, kv_heads), device=device) if eight else None
        few = torch.tensor([[3, 2], [1, 0]], dtype=torch.int32, device=device)
        where = torch.tensor([0, 40000, blocks - 2, blocks - 1], device=device)
        want = ops.rope_append(qkv, cos, sin, small, of_small, starts, seq_lens, few)
        got = ops.rope_append(qkv, cos, sin, large, of_large, starts, seq_lens, where[few.long()].to(torch.int32))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        as_words = torch.uint8 if eight else torch.int16
        assert torch.equal(large.view(as_words)[:, where], small.view(as_words))
        large.view(as_words)[:, where] = 0
        assert not bool(large.view(torch.int64).any())
        if eight:
            assert torch.equal(of_large[:, where], of_small)
        del large


def test_probabilities_past_31_bits(device):
    """17 rows of the largest vocabulary; the weights are quarters, whose sums are exact."""
    vocab, rows = 1 << 27, 17
    target = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=device)
    assert target.numel() > 1 << 31
    tokens = torch.tensor([(r * 9176533) % vocab for r in range(rows)], device=device)
    target[torch.arange(rows - 1, device=device), tokens[1:]] = 1.0
    places = torch.tensor([5, (1 << 26) + 3, vocab - 1], device=device)
    starts = torch.tensor([0, rows], dtype=torch.int32, device=device)
    for last in (rows - 1, 8):
        target[last, places] = 0.25
        if last < rows - 1:
            target[last, tokens[last + 1]] = 0.5  # (its draft, which was certain, is refused by 0.7)
        for u, place in ((0.1, 0), (0.5, 1), (0.9, 2)):
            uniforms = torch.full((rows,), 0.7, device=device)
            uniforms[-1] = u
            verified = step_ops.verify_drafts(target, tokens, uniforms, starts)
            assert verified.accepted.tolist() == [last]
            want = tokens[1:last + 1].tolist() + [int(places[place])] + [-1] * (rows - 1 - last)
            assert verified.tokens.tolist() == want, (last, u)
