"""Fused elementwise ops around the packed attention in one looped-decoder layer.

One Ouro layer (plugins/looped_transformers/src/looped_transformers/ouro.py:101-157)
brackets its attention with vLLM's fused add + RMSNorm, the rotary embedding
of Q and K, and Qwen2MLP's SiLU(gate) * up.  Beside them stand the projections at a few rows,
with BF16 and with 4-bit weights, and the log probabilities of a step's
tokens.  Each op here is a HIP launch through ``librq_hip.so`` (rq_rms_norm,
rq_rope_qkv, rq_silu_mul, rq_linear_rows, rq_linear_rows_int4,
rq_token_logprobs); there is no CPU or torch fallback.  Work is enqueued on the current HIP stream of the
input's device.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .ops import _on_device


def _require(condition: bool, message: str) -> None:
    if not condition:
        raise RuntimeError(message)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _rows(tensor: torch.Tensor, name: str) -> None:
    _require(tensor.is_cuda and tensor.dtype == torch.bfloat16 and tensor.dim() == 2 and tensor.stride(1) == 1,
             f"{name} must be BF16 [rows, channels] on a HIP device with unit channel stride")


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
             out: Optional[torch.Tensor] = None, pre_weight: Optional[torch.Tensor] = None):
    """RMSNorm of ``x`` (vLLM RMSNorm.forward); with ``residual``, the fused form.

    Without a residual returns ``y = bf16(bf16(x * rsqrt(mean(x^2) + eps)) * weight)``.
    With one, ``residual`` is updated in place to ``bf16(x + residual)`` and
    ``(y, residual)`` is returned, y normalizing the updated residual
    (vLLM's fused_add_rms_norm contract).  With ``pre_weight``, ``x`` is
    first replaced by ``rms_norm(x, pre_weight, eps)`` in the same launch.
    """
    _rows(x, "x")
    rows, hidden = x.shape
    for w in (weight, pre_weight):
        if w is not None:
            _require(w.is_cuda and w.dtype == torch.bfloat16 and w.shape == (hidden,) and w.is_contiguous(),
                     "RMSNorm weight must be a contiguous BF16 [hidden] vector")
    if residual is not None:
        _rows(residual, "residual")
        _require(residual.shape == x.shape and residual.device == x.device, "residual must match x")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    _rows(out, "out")
    _require(out.shape == x.shape and out.device == x.device, "out must match x")
    with torch.cuda.device(x.device):
        status = _lib.lib().rq_rms_norm(
            x.data_ptr(), x.stride(0), pre_weight.data_ptr() if pre_weight is not None else None,
            residual.data_ptr() if residual is not None else None,
            residual.stride(0) if residual is not None else 0,
            residual.data_ptr() if residual is not None else None,
            residual.stride(0) if residual is not None else 0, weight.data_ptr(), out.data_ptr(), out.stride(0),
            rows, hidden, float(eps), _stream(x.device))
    _lib.check(status)
    return out if residual is None else (out, residual)


def rope_qkv(qkv: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, heads: int,
             head_dim: int, key_stage: Optional[torch.Tensor] = None,
             value_stage: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rotate-half rotary embedding of the Q and K parts of fused ``[q | k | v]`` rows.

    ``cos``/``sin`` are FP32 ``[max_position, head_dim / 2]`` tables
    (get_rope with rotary_dim = head_dim); positions int64 ``[rows]`` (clamped
    to the tables).  Returns rotated ``(q, k)`` as ``[rows, heads, head_dim]``;
    when ``key_stage``/``value_stage`` are given (``[rows, heads, head_dim]``,
    sharing one row stride) the rotated K and the raw V are also copied there.
    """
    _rows(qkv, "qkv")
    rows = qkv.size(0)
    _require(qkv.size(1) == 3 * heads * head_dim, "qkv rows must hold [q | k | v] of heads * head_dim each")
    _require(positions.is_cuda and positions.dtype == torch.int64 and positions.is_contiguous()
             and positions.numel() == rows, "Contiguous INT64 positions, one per row, required")
    for table in (cos, sin):
        _require(table.is_cuda and table.dtype == torch.float32 and table.is_contiguous() and table.dim() == 2
                 and table.size(1) == head_dim // 2 and table.shape == cos.shape,
                 "Contiguous FP32 [positions, head_dim / 2] cos/sin tables required")
    query = torch.empty((rows, heads, head_dim), dtype=qkv.dtype, device=qkv.device)
    key = torch.empty_like(query)
    stage_stride = 0
    for stage in (key_stage, value_stage):
        if stage is not None:
            _require(stage.is_cuda and stage.dtype == torch.bfloat16 and stage.shape == (rows, heads, head_dim)
                     and stage.stride(2) == 1 and stage.stride(1) == head_dim,
                     "K/V staging must be BF16 [rows, heads, head_dim] with packed trailing strides")
            _require(stage_stride in (0, stage.stride(0)), "K and V staging must share one row stride")
            stage_stride = stage.stride(0)
    with torch.cuda.device(qkv.device):
        status = _lib.lib().rq_rope_qkv(
            qkv.data_ptr(), qkv.stride(0), positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.size(0), heads,
            head_dim, rows, query.data_ptr(), query.stride(0), key.data_ptr(), key.stride(0),
            key_stage.data_ptr() if key_stage is not None else None,
            value_stage.data_ptr() if value_stage is not None else None, stage_stride, _stream(qkv.device))
    _lib.check(status)
    return query, key


def silu_mul(gate_up: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``bf16(silu(gate) * up)`` of ``[rows, 2 * width]`` rows (vLLM SiluAndMul)."""
    _rows(gate_up, "gate_up")
    rows, double = gate_up.shape
    _require(double % 4 == 0, "gate_up rows must hold two halves of an even width")
    width = double // 2
    if out is None:
        out = torch.empty((rows, width), dtype=gate_up.dtype, device=gate_up.device)
    _rows(out, "out")
    _require(out.shape == (rows, width) and out.device == gate_up.device, "out must be [rows, width]")
    with torch.cuda.device(gate_up.device):
        status = _lib.lib().rq_silu_mul(gate_up.data_ptr(), gate_up.stride(0), out.data_ptr(), out.stride(0), rows,
                                        width, _stream(gate_up.device))
    _lib.check(status)
    return out


LINEAR_MAX_ROWS = 8


def linear_rows(x: torch.Tensor, weight: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``bf16(x @ weight.T)`` for 1-8 BF16 rows (rq_linear_rows), FP32 accumulation.

    ``weight`` is a contiguous BF16 ``[out_features, in_features]`` linear
    weight; ``in_features`` a multiple of 8 up to 6144.  The projections of a
    decode step at small batch, streamed as matrix-vector products."""
    _rows(x, "x")
    rows, in_features = x.shape
    _require(weight.is_cuda and weight.dtype == torch.bfloat16 and weight.dim() == 2 and weight.is_contiguous()
             and weight.size(1) == in_features and weight.device == x.device,
             "weight must be a contiguous BF16 [out_features, in_features] tensor on x's device")
    if out is None:
        out = torch.empty((rows, weight.size(0)), dtype=torch.bfloat16, device=x.device)
    _rows(out, "out")
    _require(out.shape == (rows, weight.size(0)) and out.device == x.device, "out must be [rows, out_features]")
    with torch.cuda.device(x.device):
        status = _lib.lib().rq_linear_rows(x.data_ptr(), x.stride(0), weight.data_ptr(), out.data_ptr(), out.stride(0),
                                          rows, weight.size(0), in_features, _stream(x.device))
    _lib.check(status)
    return out


LINEAR_INT4_MAX_ROWS = 64


class Int4Weight:
    """A linear weight ``[out_features, in_features]`` in 4 bits, laid out for ``linear_rows_int4``.

    Codes in -8..7 with one BF16 scale per output row and ``group`` inputs;
    made by ``quantize_weight_int4`` or ``pack_weight_int4``.
    """

    def __init__(self, data: torch.Tensor, out_features: int, in_features: int, group: int):
        self.data, self.out_features, self.in_features, self.group = data, out_features, in_features, group
        self.device = data.device

    @property
    def shape(self) -> Tuple[int, int]:
        return self.out_features, self.in_features

    def dequantize(self) -> torch.Tensor:
        """The BF16 weight ``[out_features, in_features]``: ``bf16(code * scale)``."""
        weight = torch.empty(self.shape, dtype=torch.bfloat16, device=self.device)
        with _on_device(self.data.get_device()):
            status = _lib.lib().rq_dequantize_weight_int4(self.data.data_ptr(), self.data.numel(), self.out_features,
                                                          self.in_features, self.group, weight.data_ptr(),
                                                          _stream(self.device))
        _lib.check(status)
        return weight


def _int4_weight(out_features: int, in_features: int, group: int, device: torch.device) -> Int4Weight:
    needed = _lib.lib().rq_int4_weight_bytes(out_features, in_features, group)
    if needed == 0:
        raise RuntimeError(_lib.lib().rq_last_error().decode(errors="replace"))
    return Int4Weight(torch.empty(needed, dtype=torch.uint8, device=device), out_features, in_features, group)


def quantize_weight_int4(weight: torch.Tensor, group: int = 32) -> Int4Weight:
    """A contiguous BF16 weight ``[out_features, in_features]`` in 4 bits.

    Per output row and ``group`` (32, 64 or 128) inputs: scale = bf16(largest
    |w| / 7), code = w / scale to nearest, ties to even.
    """
    _require(weight.is_cuda and weight.dtype == torch.bfloat16 and weight.dim() == 2 and weight.is_contiguous(),
             "weight must be a contiguous BF16 [out_features, in_features] tensor on a HIP device")
    packed = _int4_weight(weight.size(0), weight.size(1), group, weight.device)
    with _on_device(weight.get_device()):
        status = _lib.lib().rq_quantize_weight_int4(weight.data_ptr(), packed.out_features, packed.in_features, group,
                                                    packed.data.data_ptr(), packed.data.numel(), _stream(weight.device))
    _lib.check(status)
    return packed


def pack_weight_int4(codes: torch.Tensor, scales: torch.Tensor) -> Int4Weight:
    """A weight given as INT8 ``codes`` ``[out_features, in_features]`` (limited
    to -8..7) and BF16 ``scales`` ``[out_features, in_features / group]``, both contiguous."""
    _require(codes.is_cuda and codes.dtype == torch.int8 and codes.dim() == 2 and codes.is_contiguous(),
             "codes must be a contiguous INT8 [out_features, in_features] tensor on a HIP device")
    _require(scales.device == codes.device and scales.dtype == torch.bfloat16 and scales.dim() == 2
             and scales.is_contiguous() and scales.size(0) == codes.size(0) and scales.size(1) > 0
             and codes.size(1) % scales.size(1) == 0,
             "scales must be a contiguous BF16 [out_features, in_features / group] tensor on the codes' device")
    packed = _int4_weight(codes.size(0), codes.size(1), codes.size(1) // scales.size(1), codes.device)
    with _on_device(codes.get_device()):
        status = _lib.lib().rq_pack_weight_int4(codes.data_ptr(), scales.data_ptr(), packed.out_features,
                                                packed.in_features, packed.group, packed.data.data_ptr(),
                                                packed.data.numel(), _stream(codes.device))
    _lib.check(status)
    return packed


def linear_rows_int4(x: torch.Tensor, weight: Int4Weight, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``bf16(x @ weight.T)`` for 1-64 BF16 rows and a 4-bit weight (rq_linear_rows_int4), FP32 accumulation.

    The codes are exact in the products and the scales multiply each group's
    sum; the weight itself is never rounded to BF16.  ``x`` rows are 16-byte aligned.
    """
    # (A step makes hundreds of these calls: shapes and strides are read once.)
    shape, strides = x.shape, x.stride()
    if not (len(shape) == 2 and strides[1] == 1 and x.is_cuda and x.dtype is torch.bfloat16):
        _rows(x, "x")
    rows, in_features = shape
    out_features, data, device = weight.out_features, weight.data, x.get_device()
    if in_features != weight.in_features or data.get_device() != device:
        raise RuntimeError("x must have the weight's in_features and device")
    out_stride = out_features
    if out is None:
        out = x.new_empty((rows, out_features))
    else:
        _rows(out, "out")
        if out.shape != (rows, out_features) or out.get_device() != device:
            raise RuntimeError("out must be [rows, out_features]")
        if rows > 1:
            out_stride = out.stride(0)
    with _on_device(device):
        status = _lib.lib().rq_linear_rows_int4(
            x.data_ptr(), strides[0] if rows > 1 else in_features, data.data_ptr(), data.numel(), out.data_ptr(),
            out_stride, rows, out_features, in_features, weight.group, torch._C._cuda_getCurrentRawStream(device))
    _lib.check(status)
    return out


LOGPROBS_MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    """Log probabilities (natural logarithm) of a call's tokens and their rows' distributions."""

    logprob: torch.Tensor       # FP32 [rows]
    entropy: torch.Tensor       # FP32 [rows]
    top_logprobs: torch.Tensor  # FP32 [rows, top], largest first
    top_tokens: torch.Tensor    # INT64 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Log probability of ``tokens[i]`` under ``logits[i]``, the row's entropy and its ``top`` alternatives.

    ``logits`` is BF16 or FP32 ``[rows, vocab]`` with unit column stride,
    ``tokens`` INT64 ``[rows]`` (a token outside the vocabulary gives NaN),
    ``top`` 0 to 32.  Logits of -inf (ruled-out tokens) have probability 0 and
    add nothing to the entropy; a row of -inf alone, or with a NaN or +inf,
    gives NaN.  Equal logits rank by the lower token.
    """
    shape, strides, dtype = logits.shape, logits.stride(), logits.dtype
    if not (logits.is_cuda and len(shape) == 2 and (strides[1] == 1 or shape[1] == 1)
            and (dtype is torch.bfloat16 or dtype is torch.float32)):
        raise RuntimeError("logits must be BF16 or FP32 [rows, vocab] on a HIP device with unit column stride")
    rows, vocab = shape
    device = logits.get_device()
    if not (tokens.get_device() == device and tokens.dtype is torch.int64 and tokens.dim() == 1
            and tokens.is_contiguous() and tokens.numel() == rows):
        raise RuntimeError("Contiguous INT64 tokens, one per row, on the logits' device required")
    top = int(top)
    if not 0 <= top <= min(LOGPROBS_MAX_TOP, vocab):
        raise RuntimeError(f"0 to {LOGPROBS_MAX_TOP} alternatives, at most the vocabulary, required")
    logprob = torch.empty(rows, dtype=torch.float32, device=logits.device)
    entropy = torch.empty_like(logprob)
    top_logprobs = logprob.new_empty((rows, top))
    top_tokens = tokens.new_empty((rows, top))
    with _on_device(device):
        status = _lib.lib().rq_token_logprobs(
            logits.data_ptr(), strides[0] if rows > 1 else vocab, 0 if dtype is torch.bfloat16 else 1, rows, vocab,
            tokens.data_ptr(), logprob.data_ptr(), entropy.data_ptr(), top, top_logprobs.data_ptr(),
            top_tokens.data_ptr(), torch._C._cuda_getCurrentRawStream(device))
    _lib.check(status)
    return TokenLogprobs(logprob, entropy, top_logprobs, top_tokens)
