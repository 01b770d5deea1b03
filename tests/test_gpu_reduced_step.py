"""The 8-bit cache, 4-bit projections and log probabilities run together, as a decode step uses them."""

from __future__ import annotations

import pytest
import torch

from residualquant_amd import ops, step_ops
from residualquant_amd.looped_decode import LoopedConfig, LoopedDecoder, _project

from . import fp8_reference as reference
from .test_gpu_linear_int4 import _reference as linear_reference
from .test_gpu_logprobs import _check as check_logprobs

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, PAGE, VOCAB, HIDDEN = 4, 2, 96, 16, 1003, 384
BATCH = 3


class _Layer:
    """One attention layer and a vocabulary projection with 4-bit weights over an 8-bit cache."""

    def __init__(self, device, pages):
        g = torch.Generator().manual_seed(1)
        self.device = device
        self.parts = {}
        for name, out, group in (("qkv", (HEADS + 2 * KV_HEADS) * DIM, 32), ("o", HIDDEN, 64), ("head", VOCAB, 128)):
            codes = torch.randint(-8, 8, (out, HIDDEN), generator=g, dtype=torch.int8)
            scales = (torch.rand((out, HIDDEN // group), generator=g) * 0.01 + 0.005).to(torch.bfloat16)
            self.parts[name] = (codes, scales, step_ops.pack_weight_int4(codes.to(device), scales.to(device)))
        blocks = BATCH * pages + 2
        self.cache = torch.zeros((2, blocks, KV_HEADS, PAGE, DIM), dtype=torch.float8_e4m3fn, device=device)
        self.scales = torch.ones((2, blocks, KV_HEADS), device=device)
        self.table = torch.randperm(blocks, generator=g)[:BATCH * pages].view(BATCH, pages).to(torch.int32).to(device)

    def step(self, x, starts, seq_lens, tokens, out):
        """One call over rows x: the tensors of every stage."""
        qkv = step_ops.linear_rows_int4(x, self.parts["qkv"][2])
        q = qkv[:, :HEADS * DIM].unflatten(1, (HEADS, DIM))
        k = qkv[:, HEADS * DIM:(HEADS + KV_HEADS) * DIM].unflatten(1, (KV_HEADS, DIM))
        v = qkv[:, (HEADS + KV_HEADS) * DIM:].unflatten(1, (KV_HEADS, DIM))
        ops.paged_attention_fp8(q, k, v, self.cache, self.scales, out, starts, seq_lens, self.table)
        ops.quantize_fp8(k, v, self.cache, self.scales, starts, seq_lens, self.table)
        hidden = step_ops.linear_rows_int4(out.flatten(1), self.parts["o"][2])
        logits = step_ops.linear_rows_int4(hidden, self.parts["head"][2])
        return {"qkv": qkv, "q": q, "k": k, "v": v, "out": out, "hidden": hidden, "logits": logits,
                "logprobs": step_ops.token_logprobs(logits, tokens, top=6)}


def _check_linear(layer, name, x, got):
    codes, scales, _ = layer.parts[name]
    want, bound = linear_reference(x.cpu(), codes, scales)
    assert bool(((got.cpu().double() - want).abs() <= bound).all()), name


def test_prompts_then_tokens(device):
    """Ragged prompts, then single tokens: every stage against its reference on the stage's own inputs."""
    layer = _Layer(device, pages=5)
    g = torch.Generator().manual_seed(2)
    seq_lens = torch.zeros(BATCH, dtype=torch.int32)
    cache, scales = layer.cache.cpu(), layer.scales.cpu()
    for rows in ([17, 1, 30], [0, 16, 5], [1, 1, 1], [1, 1, 1], [3, 0, 1], [1, 1, 1]):
        starts = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
        seq_lens = seq_lens + torch.tensor(rows, dtype=torch.int32)
        total = sum(rows)
        x = torch.randn((total, HIDDEN), generator=g).to(torch.bfloat16)
        tokens = torch.randint(0, VOCAB, (total,), generator=g)
        out = torch.zeros((total, HEADS, DIM), dtype=torch.bfloat16, device=device)
        s = layer.step(x.to(device), starts.to(device), seq_lens.to(device), tokens.to(device), out)
        _check_linear(layer, "qkv", x, s["qkv"])
        q, k, v = (s[n].cpu() for n in ("q", "k", "v"))
        want, bound = reference.attend(q, k, v, cache, scales, starts, seq_lens, layer.table.cpu(), DIM ** -0.5)
        assert bool(((s["out"].cpu().double() - want).abs() <= bound).all()), rows
        reference.write(k, v, cache, scales, starts, seq_lens, layer.table.cpu())
        assert torch.equal(layer.cache.cpu().view(torch.uint8), cache.view(torch.uint8)), rows
        assert torch.equal(layer.scales.cpu(), scales)
        _check_linear(layer, "o", s["out"].flatten(1), s["hidden"])
        _check_linear(layer, "head", s["hidden"], s["logits"])
        check_logprobs(s["logits"].cpu(), tokens, 6, device, got=s["logprobs"])


def test_captured_steps_match_eager_steps(device):
    """A step captured into a graph and replayed on a growing cache, with eager steps of a twin between."""
    first, second = _Layer(device, pages=4), _Layer(device, pages=4)
    g = torch.Generator().manual_seed(3)
    starts = torch.arange(BATCH + 1, dtype=torch.int32, device=device)
    seq_lens = torch.full((BATCH,), 15, dtype=torch.int32, device=device)
    x = torch.randn((BATCH, HIDDEN), generator=g).to(torch.bfloat16).to(device)
    tokens = torch.randint(0, VOCAB, (BATCH,), generator=g).to(device)
    outs = [torch.zeros((BATCH, HEADS, DIM), dtype=torch.bfloat16, device=device) for _ in range(2)]
    first.step(x, starts, seq_lens, tokens, outs[0])  # pages are written before the capture
    second.step(x, starts, seq_lens, tokens, outs[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seq_lens.add_(1)
        captured = first.step(x, starts, seq_lens, tokens, outs[0])
    for step in range(4):
        x.copy_(torch.randn((BATCH, HIDDEN), generator=g).to(torch.bfloat16))
        graph.replay()
        eager = second.step(x, starts, seq_lens, tokens, outs[1])
        torch.cuda.synchronize()
        assert torch.equal(first.cache.view(torch.uint8), second.cache.view(torch.uint8)), step
        assert torch.equal(first.scales, second.scales) and torch.equal(outs[0], outs[1])
        assert torch.equal(captured["logits"], eager["logits"])
        assert all(torch.equal(a, b) for a, b in zip(captured["logprobs"], eager["logprobs"]))


def _small_config(**other):
    return LoopedConfig(layers=2, hidden=512, heads=4, head_dim=128, intermediate=768, vocab=1000, **other)


@pytest.mark.parametrize("batch", [1, 5])
def test_looped_decoder_with_4_bit_projections(device, batch):
    """Against the same decoder with the restored weights in BF16 (equal where the scales are
    powers of two); only the order of float32 sums differs between the two."""
    narrow = LoopedDecoder(_small_config(projection_bits=4, projection_group=64), batch, 40, 8, device, seed=4,
                           top_logprobs=3)
    wide = LoopedDecoder(_small_config(), batch, 40, 8, device, seed=4)
    g = torch.Generator(device=device).manual_seed(9)
    for name in ("qkv", "o", "gate_up", "down", "lm_head"):
        held = getattr(narrow, name)
        weights = []
        for old in held if isinstance(held, list) else [held]:
            assert isinstance(old, step_ops.Int4Weight) and old.group == 64
            out, features = old.shape
            codes = torch.randint(-7, 8, (out, features), generator=g, device=device, dtype=torch.int8)
            scales = torch.full((out, features // 64), 2.0 ** -7, dtype=torch.bfloat16, device=device)
            weights.append(step_ops.pack_weight_int4(codes, scales))
        restored = [w.dequantize() for w in weights]
        setattr(narrow, name, weights if isinstance(held, list) else weights[0])
        setattr(wide, name, restored if isinstance(held, list) else restored[0])
    for decoder in (narrow, wide):
        decoder.build_history(seed=5)
        decoder.tokens.copy_(torch.arange(batch, device=device) * 7)
    got, want = narrow.step(), wide.step()
    # BF16 activations round differently where two sums fall on either side of a midpoint; the
    # model's logits amplify that over its eight layer passes.
    assert (got.float() - want.float()).norm() <= 0.03 * want.float().norm()
    assert torch.equal(narrow.tokens, got.argmax(dim=-1))
    check_logprobs(got.cpu(), narrow.tokens.cpu(), 3, device, got=narrow.logprobs)
    narrow.capture()
    for _ in range(3):
        logits = narrow.replay()
        torch.cuda.synchronize()
        check_logprobs(logits.cpu(), narrow.tokens.cpu(), 3, device, got=narrow.logprobs)


def test_looped_decoder_of_many_rows_and_refusals(device):
    decoder = LoopedDecoder(_small_config(projection_bits=4), 70, 20, 4, device, seed=6)
    decoder.build_history(seed=5)
    assert bool(decoder.step().isfinite().all())
    assert decoder.logprobs is None
    with pytest.raises(ValueError, match="16 or 4 bits"):
        LoopedDecoder(_small_config(projection_bits=8), 1, 20, 4, device)
    with pytest.raises(ValueError, match="alternatives"):
        LoopedDecoder(_small_config(), 1, 20, 4, device, top_logprobs=33)


def test_looped_decoder_logprobs_of_the_last_step_however_it_ran(device):
    """Captured and eager steps in turn: ``logprobs`` is the last step's, also where the graph itself is replayed."""
    decoder = LoopedDecoder(_small_config(), 3, 40, 9, device, seed=7, top_logprobs=4)
    decoder.build_history(seed=5)
    graph = decoder.capture()
    for run in (decoder.replay, decoder.step, decoder.replay, decoder.step, decoder.step, graph.replay):
        logits = run()
        torch.cuda.synchronize()
        logits = decoder.logits if logits is None else logits
        check_logprobs(logits.cpu(), decoder.tokens.cpu(), 4, device, got=decoder.logprobs)
    decoder.capture()
    logits = decoder.replay()
    torch.cuda.synchronize()
    check_logprobs(logits.cpu(), decoder.tokens.cpu(), 4, device, got=decoder.logprobs)


@pytest.mark.parametrize("rows", [64, 65, 70, 130, 257])
@pytest.mark.parametrize("out,features,group", [(1000, 512, 32), (512, 768, 64), (37, 5632, 128)])
def test_projection_of_many_rows(device, rows, out, features, group):
    """The decoder's projection at any number of rows: the weight itself is not rounded."""
    g = torch.Generator().manual_seed(rows + out)
    codes = torch.randint(-8, 8, (out, features), generator=g, dtype=torch.int8)
    scales = (torch.rand((out, features // group), generator=g) * 0.02 + 0.001).to(torch.bfloat16)
    x = torch.randn((rows, features), generator=g).to(torch.bfloat16)
    got = _project(x.to(device), step_ops.pack_weight_int4(codes.to(device), scales.to(device))).cpu().double()
    want, bound = linear_reference(x, codes, scales)
    assert got.shape == want.shape
    assert bool(((got - want).abs() <= bound).all()), ((got - want).abs() / bound).max()


def test_looped_decoder_of_many_rows_repeats_its_replays(device):
    """A step of 70 rows: captured and replayed, it gives what an eager twin gives."""
    first, second = (LoopedDecoder(_small_config(projection_bits=4), 70, 20, 6, device, seed=8) for _ in range(2))
    for decoder in (first, second):
        decoder.build_history(seed=5)
    first.capture()
    for _ in range(3):
        got, want = first.replay(), second.step()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(first.tokens, second.tokens)
