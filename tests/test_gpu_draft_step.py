"""8-bit projections, rotated appends, attention and draft verification run together, as a speculative step uses them."""

from __future__ import annotations

import pytest
import torch

from residualquant_amd import ops, step_ops
from residualquant_amd.looped_decode import LoopedConfig, LoopedDecoder

from . import fp8_reference as reference
from .test_gpu_linear_fp8 import check as check_linear, make_weight
from .test_gpu_rope_append import rotated, tables
from .test_gpu_verify_drafts import reference as verify_reference

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, PAGE, VOCAB, HIDDEN = 4, 2, 96, 16, 1003, 384
BATCH, DRAFTS = 3, 4


class _Layer:
    """One attention layer and a vocabulary projection with E4M3 weights over an 8-bit cache."""

    def __init__(self, device, pages):
        g = torch.Generator().manual_seed(1)
        self.device = device
        self.parts = {name: make_weight(out, HIDDEN, kind, seed, device) for seed, (name, out, kind) in enumerate(
            (("qkv", (HEADS + 2 * KV_HEADS) * DIM, "exponents"), ("o", HIDDEN, "float"), ("head", VOCAB, "exponents")))}
        blocks = BATCH * pages + 2
        self.cos, self.sin = tables(pages * PAGE, DIM, device)
        self.cache = torch.zeros((2, blocks, KV_HEADS, PAGE, DIM), dtype=torch.float8_e4m3fn, device=device)
        self.scales = torch.ones((2, blocks, KV_HEADS), device=device)
        self.table = torch.randperm(blocks, generator=g)[:BATCH * pages].view(BATCH, pages).to(torch.int32).to(device)

    def step(self, x, starts, seq_lens, tokens, uniforms, draft, out):
        """One call over rows x: the tensors of every stage."""
        qkv = step_ops.linear_fp8(x, self.parts["qkv"][0])
        q, k, v = ops.rope_append(qkv, self.cos, self.sin, self.cache, self.scales, starts, seq_lens, self.table)
        ops.paged_attention_fp8(q, k, v, self.cache, self.scales, out, starts, seq_lens, self.table)
        hidden = step_ops.linear_fp8(out.flatten(1), self.parts["o"][0])
        logits = step_ops.linear_fp8(hidden, self.parts["head"][0])
        target = torch.softmax(logits.float() / (logits.float().std(dim=1, keepdim=True) + 1e-20), dim=1)
        verified = step_ops.verify_drafts(target, tokens, uniforms, starts, draft=draft)
        return {"qkv": qkv, "q": q, "k": k, "v": v, "out": out, "hidden": hidden, "logits": logits, "target": target,
                "verified": verified}


def _drafts(rows, g):
    return torch.softmax(torch.randn((rows, VOCAB), generator=g), dim=1)


def test_prompts_then_drafts(device):
    """Ragged prompts, then drafts of which some are taken: every stage against its reference on the stage's own inputs.
    What a refused draft left in the cache is written again by the tokens that follow."""
    layer = _Layer(device, pages=6)
    g = torch.Generator().manual_seed(2)
    cache, scales = layer.cache.cpu(), layer.scales.cpu()
    cos, sin = layer.cos.cpu(), layer.sin.cpu()
    lengths = torch.zeros(BATCH, dtype=torch.int64)
    taken = 0
    for call, rows in enumerate(([17, 1, 30], [0, 16, 5], [1, 5, 3], [5, 5, 5], [2, 0, 1], [5, 4, 5], [1, 1, 1], [5, 5, 5])):
        starts = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
        seq_lens = (lengths + torch.tensor(rows)).to(torch.int32)
        total = sum(rows)
        x = torch.randn((total, HIDDEN), generator=g).to(torch.bfloat16)
        tokens, uniforms = torch.randint(0, VOCAB, (total,), generator=g), torch.rand(total, generator=g)
        draft = None if call % 3 == 0 else _drafts(total, g)
        if call % 2:
            uniforms[::2] = 0.0  # (taken wherever the target has them at all)
        out = torch.zeros((total, HEADS, DIM), dtype=torch.bfloat16, device=device)
        s = layer.step(x.to(device), starts.to(device), seq_lens.to(device), tokens.to(device), uniforms.to(device),
                       None if draft is None else draft.to(device), out)
        check_linear(s["qkv"], x, layer.parts["qkv"][1])
        places = torch.cat([torch.arange(int(h), int(h) + n) for h, n in zip(lengths, rows)])
        parts = s["qkv"].cpu().view(total, HEADS + 2 * KV_HEADS, DIM)
        assert torch.equal(s["q"].cpu(), rotated(parts[:, :HEADS], cos[places], sin[places], False))
        assert torch.equal(s["k"].cpu(), rotated(parts[:, HEADS:HEADS + KV_HEADS], cos[places], sin[places], False))
        q, k, v = (s[n].cpu().contiguous() for n in ("q", "k", "v"))
        reference.write(k, v, cache, scales, starts, seq_lens, layer.table.cpu())
        assert torch.equal(layer.cache.cpu().view(torch.uint8), cache.view(torch.uint8)), rows
        assert torch.equal(layer.scales.cpu(), scales)
        want, bound = reference.attend(q, k, v, cache, scales, starts, seq_lens, layer.table.cpu(), DIM ** -0.5)
        assert bool(((s["out"].cpu().double() - want).abs() <= bound).all()), rows
        check_linear(s["hidden"], s["out"].flatten(1).cpu(), layer.parts["o"][1])
        check_linear(s["logits"], s["hidden"].cpu(), layer.parts["head"][1])
        accepted, following = verify_reference(s["target"].cpu(), tokens, uniforms, starts.tolist(), draft)
        assert s["verified"].accepted.tolist() == accepted and s["verified"].tokens.tolist() == following
        # The first call's rows are prompts; of the others the tokens behind the refused draft are given up.
        prompt = call < 2
        lengths = lengths + torch.tensor([n if prompt else min(n, 1 + a) for n, a in zip(rows, accepted)])
        taken += 0 if prompt else sum(accepted)
    assert taken > 0


def test_captured_steps_match_eager_steps(device):
    """A speculative step captured into a graph, its lengths advanced by what was taken, with eager steps of a twin between."""
    first, second = _Layer(device, pages=6), _Layer(device, pages=6)
    g = torch.Generator().manual_seed(3)
    total = BATCH * (DRAFTS + 1)
    starts = torch.arange(0, total + 1, DRAFTS + 1, dtype=torch.int32, device=device)
    lengths = [torch.full((BATCH,), 12 + DRAFTS + 1, dtype=torch.int32, device=device) for _ in range(2)]
    x = torch.randn((total, HIDDEN), generator=g).to(torch.bfloat16).to(device)
    tokens = torch.randint(0, VOCAB, (total,), generator=g).to(device)
    uniforms, draft = torch.rand(total, generator=g).to(device), _drafts(total, g).to(device)
    outs = [torch.zeros((total, HEADS, DIM), dtype=torch.bfloat16, device=device) for _ in range(2)]

    def run(layer, k):
        s = layer.step(x, starts, lengths[k], tokens, uniforms, draft, outs[k])
        lengths[k].add_(1 + s["verified"].accepted)
        return s

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(first, 0)
    torch.cuda.current_stream().wait_stream(stream)
    run(second, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(first, 0)
    for step in range(4):
        x.copy_(torch.randn((total, HIDDEN), generator=g).to(torch.bfloat16))
        uniforms.copy_(torch.rand(total, generator=g))
        draft.copy_(_drafts(total, g))
        tokens.copy_(torch.randint(0, VOCAB, (total,), generator=g))
        graph.replay()
        eager = run(second, 1)
        torch.cuda.synchronize()
        assert torch.equal(first.cache.view(torch.uint8), second.cache.view(torch.uint8)), step
        assert torch.equal(first.scales, second.scales) and torch.equal(outs[0], outs[1])
        assert torch.equal(captured["logits"], eager["logits"]) and torch.equal(lengths[0], lengths[1])
        assert all(torch.equal(a, b) for a, b in zip(captured["verified"], eager["verified"]))


def _small_config(**other):
    return LoopedConfig(layers=2, hidden=512, heads=4, head_dim=128, intermediate=768, vocab=1000, **other)


@pytest.mark.parametrize("batch", [1, 5, 70])
def test_looped_decoder_with_8_bit_projections(device, batch):
    """Captured and replayed, it gives what an eager twin gives; its logits are the head's product of its hidden rows."""
    first, second = (LoopedDecoder(_small_config(projection_bits=8, projection_format="e4m3"), batch, 30, 8, device,
                                   seed=4, top_logprobs=2) for _ in range(2))
    for decoder in (first, second):
        assert isinstance(decoder.lm_head, step_ops.Fp8Weight) and isinstance(decoder.qkv[0], step_ops.Fp8Weight)
        decoder.build_history(seed=5)
    second.taps = {(0, 0)}
    first.capture()
    for _ in range(3):
        got, want = first.replay(), second.step()
        torch.cuda.synchronize()
        assert bool(want.isfinite().all())
        assert torch.equal(got, want) and torch.equal(first.tokens, second.tokens)
        hidden = second.tapped[("h", second.config.loops - 1)]
        check_linear(want, hidden.cpu(), second.lm_head.dequantize().cpu().double())
    with pytest.raises(ValueError, match="16 or 4 bits"):
        LoopedDecoder(_small_config(projection_bits=8), 1, 20, 4, device)
    with pytest.raises(ValueError, match="e4m3"):
        LoopedDecoder(_small_config(projection_format="e4m3"), 1, 20, 4, device)
