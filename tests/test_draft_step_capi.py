"""Refusals of the 8-bit projection, rotated append and draft verification entry points (CPU).

Every call below fails its checks on the host: the fake addresses never reach a kernel."""

from __future__ import annotations

import os

import pytest
import torch

from residualquant_amd import _lib, ops, step_ops

FAKE = 0x10000


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        _lib.build()
    return _lib.lib()


def test_weight_bytes(lib):
    # Codes in whole tiles of 64 x 128, scales in fours of blocks.
    assert lib.rq_fp8_weight_bytes(1, 1, 0) == 64 * 128 + 4
    assert lib.rq_fp8_weight_bytes(1, 1, 1) == 64 * 128 + 16
    assert lib.rq_fp8_weight_bytes(2048, 5632, 0) == 2048 * 5632 + 16 * 44
    assert lib.rq_fp8_weight_bytes(130, 129, 1) == 192 * 256 + 2 * 16
    for wrong in ((0, 128, 0), (16, 0, 0), (16, 128, 2), (16, 128, -1), ((1 << 24) + 1, 128, 0), (16, (1 << 20) + 1, 0),
                  (1 << 24, 1 << 20, 0)):
        assert lib.rq_fp8_weight_bytes(*wrong) == 0, wrong
        assert lib.rq_last_error()


def _linear(lib, *, x=FAKE, x_stride=256, packed=FAKE, packed_bytes=1 << 40, scale_type=0, y=FAKE, y_stride=40, rows=200,
            out=40, features=256, workspace=FAKE, workspace_bytes=1 << 40):
    return lib.rq_linear_fp8(x, x_stride, packed, packed_bytes, scale_type, y, y_stride, rows, out, features, workspace,
                             workspace_bytes, None)


def test_projection_refusals(lib):
    needed = lib.rq_linear_fp8_workspace_bytes(200, 256)
    for wrong, code, words in (
            (dict(rows=-1), _lib.RQ_ENOKERNEL, b"No compiled 8-bit projection"),
            (dict(rows=(1 << 20) + 1), _lib.RQ_ENOKERNEL, b"No compiled 8-bit projection"),
            (dict(scale_type=2), _lib.RQ_EINVAL, b"Scales"),
            (dict(out=0), _lib.RQ_EINVAL, b"8-bit weights need"),
            (dict(features=0), _lib.RQ_EINVAL, b"8-bit weights need"),
            (dict(packed=None), _lib.RQ_EINVAL, b"packed weight"),
            (dict(packed=FAKE + 8), _lib.RQ_EINVAL, b"packed weight"),
            (dict(packed_bytes=64 * 256 + 3), _lib.RQ_EINVAL, b"packed weight"),
            (dict(x_stride=255), _lib.RQ_EINVAL, b"x rows"),
            (dict(y_stride=39), _lib.RQ_EINVAL, b"y rows"),
            (dict(x=None), _lib.RQ_EINVAL, b"BF16 x"),
            (dict(x=FAKE + 1), _lib.RQ_EINVAL, b"BF16 x"),
            (dict(y=FAKE + 1), _lib.RQ_EINVAL, b"BF16 output"),
            (dict(workspace=None), _lib.RQ_ENOSPACE, b"workspace of"),
            (dict(workspace_bytes=needed - 1), _lib.RQ_ENOSPACE, b"workspace of"),
            (dict(rows=1 << 20, features=1 << 20, x_stride=1 << 20), _lib.RQ_EINVAL, b"Too many rows")):
        assert _linear(lib, **wrong) == code, wrong
        assert words in lib.rq_last_error(), (wrong, lib.rq_last_error())
    assert _linear(lib, rows=0) == _lib.RQ_OK
    assert lib.rq_linear_fp8_workspace_bytes(1, 2048) == 0  # (rounded by every workgroup)


def test_packing_refusals(lib):
    for codes, scales, kind, out, features, packed, size in (
            (None, FAKE, 0, 16, 128, FAKE, 1 << 30), (FAKE, None, 0, 16, 128, FAKE, 1 << 30),
            (FAKE, FAKE + 2, 1, 16, 128, FAKE, 1 << 30), (FAKE, FAKE, 3, 16, 128, FAKE, 1 << 30),
            (FAKE, FAKE, 0, 16, 128, FAKE + 1, 1 << 30), (FAKE, FAKE, 0, 16, 128, FAKE, 2048), (FAKE, FAKE, 0, -1, 128, FAKE, 1 << 30)):
        assert lib.rq_pack_weight_fp8(codes, scales, kind, out, features, packed, size, None) == _lib.RQ_EINVAL
    assert lib.rq_quantize_weight_fp8(None, 16, 128, FAKE, 1 << 30, None) == _lib.RQ_EINVAL
    assert lib.rq_dequantize_weight_fp8(FAKE, 1 << 30, 0, 16, 128, None, None) == _lib.RQ_EINVAL


def _append(lib, *, qkv=FAKE, stride=8 * 128, rows=2, heads=4, kv_heads=2, dim=128, rotary=128, cos=FAKE, sin=FAKE,
            positions_in_table=64, positions=None, query=0x200000, query_stride=4 * 128, key=0x400000, key_stride=2 * 128,
            cache=FAKE, scales=FAKE, page=16, starts=FAKE, requests=2, table=FAKE, table_stride=4, max_pages=4):
    return lib.rq_rope_append(qkv, stride, rows, heads, kv_heads, dim, rotary, 0, cos, sin, positions_in_table, positions,
                              query, query_stride, key, key_stride, cache, scales, 8, page, starts, FAKE, requests, table,
                              table_stride, max_pages, None)


def test_append_refusals(lib):
    for wrong, code, words in (
            (dict(dim=64), _lib.RQ_ENOKERNEL, b"No compiled"),
            (dict(page=8), _lib.RQ_ENOKERNEL, b"No compiled"),
            (dict(heads=0), _lib.RQ_EINVAL, b"query heads"),
            (dict(heads=65536), _lib.RQ_EINVAL, b"query heads"),
            (dict(kv_heads=0), _lib.RQ_EINVAL, b"heads required"),
            (dict(rotary=0), _lib.RQ_EINVAL, b"multiple of 16"),
            (dict(rotary=24), _lib.RQ_EINVAL, b"multiple of 16"),
            (dict(rotary=144), _lib.RQ_EINVAL, b"multiple of 16"),
            (dict(cos=None), _lib.RQ_EINVAL, b"cos/sin"),
            (dict(sin=FAKE + 8), _lib.RQ_EINVAL, b"cos/sin"),
            (dict(positions_in_table=0), _lib.RQ_EINVAL, b"cos/sin"),
            (dict(positions=FAKE + 4), _lib.RQ_EINVAL, b"positions"),
            (dict(qkv=None), _lib.RQ_EINVAL, b"8-byte aligned"),
            (dict(query=0x200002), _lib.RQ_EINVAL, b"8-byte aligned"),
            (dict(key=0x400004), _lib.RQ_EINVAL, b"8-byte aligned"),
            (dict(stride=8 * 128 - 4), _lib.RQ_EINVAL, b"packed trailing strides"),
            (dict(query_stride=4 * 128 + 2), _lib.RQ_EINVAL, b"packed trailing strides"),
            (dict(key_stride=128), _lib.RQ_EINVAL, b"packed trailing strides"),
            (dict(cache=None), _lib.RQ_EINVAL, b"cache"),
            (dict(cache=None, scales=None), _lib.RQ_EINVAL, b"cache"),
            (dict(cache=FAKE + 8, scales=None), _lib.RQ_EINVAL, b"cache"),
            (dict(scales=FAKE + 2), _lib.RQ_EINVAL, b"cache"),
            (dict(starts=None), _lib.RQ_EINVAL, b"query starts"),
            (dict(table=None), _lib.RQ_EINVAL, b"page table"),
            (dict(max_pages=1 << 28, table_stride=1 << 28), _lib.RQ_EINVAL, b"page table"),
            (dict(query=FAKE), _lib.RQ_EINVAL, b"overlap"),
            (dict(query=FAKE + 2 * 8 * 128 * 2 - 8), _lib.RQ_EINVAL, b"overlap"),
            (dict(key=FAKE + 8), _lib.RQ_EINVAL, b"overlap"),
            (dict(key=0x200000 + 1024), _lib.RQ_EINVAL, b"overlap"),
            (dict(requests=1 << 24), _lib.RQ_EINVAL, b"Too many rows")):
        assert _append(lib, **wrong) == code, wrong
        assert words in lib.rq_last_error(), (wrong, lib.rq_last_error())
    assert _append(lib, rows=0) == _lib.RQ_OK
    assert _append(lib, requests=0) == _lib.RQ_OK


def _verify(lib, *, target=FAKE, target_stride=100, draft=FAKE, draft_stride=100, dtype=1, rows=4, vocab=100, tokens=FAKE,
            uniforms=FAKE, starts=FAKE, requests=2, accepted=FAKE, out=FAKE, workspace=FAKE, workspace_bytes=1 << 40):
    return lib.rq_verify_drafts(target, target_stride, draft, draft_stride, dtype, rows, vocab, tokens, uniforms, starts,
                                requests, accepted, out, workspace, workspace_bytes, None)


def test_verification_refusals(lib):
    needed = lib.rq_verify_drafts_workspace_bytes(2, 100)
    for wrong, code, words in (
            (dict(dtype=2), _lib.RQ_EINVAL, b"BF16 or FP32"),
            (dict(rows=-1), _lib.RQ_EINVAL, b"Probabilities [rows, vocab]"),
            (dict(vocab=0), _lib.RQ_EINVAL, b"Probabilities [rows, vocab]"),
            (dict(vocab=1 << 31), _lib.RQ_EINVAL, b"Probabilities [rows, vocab]"),
            (dict(target_stride=99), _lib.RQ_EINVAL, b"Probabilities [rows, vocab]"),
            (dict(draft_stride=99), _lib.RQ_EINVAL, b"Probabilities [rows, vocab]"),
            (dict(requests=-1), _lib.RQ_EINVAL, b"query starts"),
            (dict(starts=None), _lib.RQ_EINVAL, b"query starts"),
            (dict(accepted=None), _lib.RQ_EINVAL, b"query starts"),
            (dict(target=None), _lib.RQ_EINVAL, b"random numbers"),
            (dict(target=FAKE + 2), _lib.RQ_EINVAL, b"random numbers"),
            (dict(draft=FAKE + 1, dtype=0), _lib.RQ_EINVAL, b"random numbers"),
            (dict(tokens=None), _lib.RQ_EINVAL, b"random numbers"),
            (dict(uniforms=None), _lib.RQ_EINVAL, b"random numbers"),
            (dict(out=None), _lib.RQ_EINVAL, b"random numbers"),
            (dict(workspace=None), _lib.RQ_ENOSPACE, b"workspace of"),
            (dict(workspace_bytes=needed - 1), _lib.RQ_ENOSPACE, b"workspace of"),
            (dict(requests=1 << 28), _lib.RQ_EINVAL, b"Too many requests")):
        assert _verify(lib, **wrong) == code, wrong
        assert words in lib.rq_last_error(), (wrong, lib.rq_last_error())
    assert _verify(lib, requests=0) == _lib.RQ_OK


def test_tensors_on_the_host_are_refused():
    x, codes = torch.zeros((2, 128), dtype=torch.bfloat16), torch.zeros((16, 128), dtype=torch.float8_e4m3fn)
    weight = step_ops.Fp8Weight(torch.zeros(4096, dtype=torch.uint8), 16, 128, True)
    for call in (lambda: step_ops.linear_fp8(x, weight), lambda: step_ops.quantize_weight_fp8(x),
                 lambda: step_ops.pack_weight_fp8(codes, torch.ones((1, 1))),
                 lambda: step_ops.verify_drafts(torch.zeros((2, 9)), torch.zeros(2, dtype=torch.int64), torch.zeros(2),
                                                torch.zeros(2, dtype=torch.int32)),
                 lambda: ops.rope_append(torch.zeros((2, 8 * 128), dtype=torch.bfloat16), torch.zeros((9, 64)),
                                         torch.zeros((9, 64)), torch.zeros((2, 4, 2, 16, 128), dtype=torch.bfloat16), None,
                                         torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                                         torch.zeros((1, 4), dtype=torch.int32))):
        with pytest.raises(RuntimeError):
            call()


def test_results_over_their_inputs_are_refused(lib):
    # A few rows take no workspace; a results' row is 40 wide, an input's 256.
    for wrong in (dict(y=FAKE), dict(y=FAKE + 2 * 255), dict(y=FAKE + 2 * (3 * 256 + 255)), dict(x=FAKE + 2 * (3 * 40 + 39), y=FAKE),
                  dict(y=FAKE + 2 * 300, x_stride=512, y_stride=512, out=257), dict(y=FAKE, x=FAKE + 2 * 39, x_stride=512, y_stride=512),
                  dict(y=FAKE + 2 * 260, x_stride=512, y_stride=500)):
        assert _linear(lib, **{**dict(rows=4, workspace=None), **wrong}) == _lib.RQ_EINVAL, wrong
        assert b"overlap" in lib.rq_last_error(), wrong
    for out in (FAKE, FAKE + 8 * 3, FAKE - 8 * 3):
        assert _verify(lib, target=1 << 30, draft=None, tokens=FAKE, out=out) == _lib.RQ_EINVAL
        assert b"overlap" in lib.rq_last_error()
    # Rotated rows side by side in rows of one stride pass (here as far as the next check, of the sizes of a grid).
    side = dict(query=0x200000, key=0x200000 + 2 * 512, query_stride=768, key_stride=768, requests=1 << 24)
    assert _append(lib, **side) == _lib.RQ_EINVAL and b"Too many rows" in lib.rq_last_error()
    for wrong in (dict(key=0x200000 + 2 * 508), dict(query=0x200000 + 2 * 252, key=0x200000), dict(key=0x200000 + 2 * 516)):
        assert _append(lib, **{**side, **wrong}) == _lib.RQ_EINVAL and b"overlap" in lib.rq_last_error(), wrong
