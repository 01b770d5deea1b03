"""Refusals of the 8-bit cache, 4-bit weight and log probability entry points (CPU).

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


def _write(lib, *, key=FAKE, stride=4 * 128, rows=2, heads=4, dim=128, cache=FAKE, scales=FAKE, page=16, requests=2,
           starts=FAKE, table=FAKE, table_stride=4, max_pages=4):
    return lib.rq_quantize_fp8(key, stride, FAKE, 4 * 128, rows, heads, dim, cache, scales, 8, page, starts, FAKE,
                               requests, table, table_stride, max_pages, None)


def test_write_refusals(lib):
    for wrong, code, words in (
            (dict(dim=64), _lib.RQ_ENOKERNEL, b"No compiled 8-bit paged kernel"),
            (dict(page=64), _lib.RQ_ENOKERNEL, b"No compiled 8-bit paged kernel"),
            (dict(heads=0), _lib.RQ_EINVAL, b"heads required"),
            (dict(rows=-1), _lib.RQ_EINVAL, b"heads required"),
            (dict(cache=None), _lib.RQ_EINVAL, b"8-bit cache"),
            (dict(cache=FAKE + 8), _lib.RQ_EINVAL, b"8-bit cache"),
            (dict(scales=None), _lib.RQ_EINVAL, b"8-bit cache"),
            (dict(key=None), _lib.RQ_EINVAL, b"8-byte aligned"),
            (dict(key=FAKE + 4), _lib.RQ_EINVAL, b"8-byte aligned"),
            (dict(stride=4 * 128 - 4), _lib.RQ_EINVAL, b"packed trailing strides"),
            (dict(stride=4 * 128 + 2), _lib.RQ_EINVAL, b"packed trailing strides"),
            (dict(starts=None), _lib.RQ_EINVAL, b"query starts"),
            (dict(table=None), _lib.RQ_EINVAL, b"page table"),
            (dict(table_stride=3), _lib.RQ_EINVAL, b"page table"),
            (dict(max_pages=1 << 28, table_stride=1 << 28), _lib.RQ_EINVAL, b"page table")):
        assert _write(lib, **wrong) == code, wrong
        assert words in lib.rq_last_error(), (wrong, lib.rq_last_error())
    assert _write(lib, rows=0) == _lib.RQ_OK
    assert _write(lib, requests=0) == _lib.RQ_OK


def _attend(lib, *, query=FAKE, query_stride=8 * 128, key_stride=4 * 128, output=FAKE, rows=2, heads=8, kv_heads=4,
            dim=128, page=16, scale=0.1, workspace=FAKE, workspace_bytes=1 << 40, max_pages=4):
    return lib.rq_paged_attention_fp8(query, query_stride, FAKE, key_stride, FAKE, 4 * 128, output, 8 * 128, rows,
                                      heads, kv_heads, dim, FAKE, FAKE, 8, page, FAKE, FAKE, 2, FAKE, max_pages,
                                      max_pages, scale, workspace, workspace_bytes, None)


def test_attention_refusals(lib):
    for wrong, code, words in (
            (dict(dim=80), _lib.RQ_ENOKERNEL, b"No compiled 8-bit paged kernel"),
            (dict(heads=6), _lib.RQ_EINVAL, b"multiple of key/value heads"),
            (dict(heads=0), _lib.RQ_EINVAL, b"multiple of key/value heads"),
            (dict(scale=0.0), _lib.RQ_EINVAL, b"softmax_scale"),
            (dict(scale=float("nan")), _lib.RQ_EINVAL, b"softmax_scale"),
            (dict(scale=float("inf")), _lib.RQ_EINVAL, b"softmax_scale"),
            (dict(query=FAKE + 2), _lib.RQ_EINVAL, b"8-byte aligned"),
            (dict(output=FAKE + 4), _lib.RQ_EINVAL, b"8-byte aligned"),
            (dict(query_stride=8 * 128 - 4), _lib.RQ_EINVAL, b"packed trailing strides"),
            (dict(key_stride=4 * 128 + 1), _lib.RQ_EINVAL, b"packed trailing strides"),
            (dict(workspace=None), _lib.RQ_ENOSPACE, b"Attention workspace of"),
            (dict(workspace_bytes=16), _lib.RQ_ENOSPACE, b"Attention workspace of")):
        assert _attend(lib, **wrong) == code, wrong
        assert words in lib.rq_last_error(), (wrong, lib.rq_last_error())
    assert _attend(lib, rows=0) == _lib.RQ_OK


def test_page_tables_past_2_to_the_30_tokens_are_refused(lib):
    """The kernels count tokens in 31 bits, rounded up to steps and tiles ahead."""
    for page in (16, 32):
        pages = (1 << 30) // page + 1
        assert _write(lib, page=page, max_pages=pages, table_stride=pages) == _lib.RQ_EINVAL
        assert b"2^30 tokens" in lib.rq_last_error()
        assert _attend(lib, page=page, max_pages=pages) == _lib.RQ_EINVAL
        assert b"2^30 tokens" in lib.rq_last_error()


def test_attention_workspace_depends_on_shapes_only(lib):
    sizes = [lib.rq_paged_attention_fp8_workspace_bytes(rows, 16, 16, 128, 512, 16) for rows in (1, 32, 1024)]
    assert sizes == [lib.rq_paged_attention_fp8_workspace_bytes(rows, 16, 16, 128, 512, 16) for rows in (1, 32, 1024)]
    assert all(0 < size < 1 << 30 for size in sizes)
    assert lib.rq_paged_attention_fp8_workspace_bytes(0, 16, 16, 128, 512, 16) > 0


def test_int4_refusals(lib):
    assert lib.rq_int4_weight_bytes(128, 256, 48) == 0
    assert b"groups of 48" in lib.rq_last_error()
    assert lib.rq_int4_weight_bytes(128, 200, 32) == 0
    assert lib.rq_int4_weight_bytes(0, 256, 32) == 0
    assert lib.rq_int4_weight_bytes(1 << 24, 1 << 20, 32) == 0
    size = lib.rq_int4_weight_bytes(130, 256, 32)  # nine tiles of 16 rows: codes and scales
    assert size == 9 * (16 * 256 // 2 + 16 * 8 * 2)
    assert lib.rq_pack_weight_int4(FAKE, FAKE, 130, 256, 32, FAKE, size - 1, None) == _lib.RQ_EINVAL
    assert lib.rq_pack_weight_int4(None, FAKE, 130, 256, 32, FAKE, size, None) == _lib.RQ_EINVAL
    assert lib.rq_quantize_weight_int4(FAKE + 1, 130, 256, 32, FAKE, size, None) == _lib.RQ_EINVAL
    assert lib.rq_dequantize_weight_int4(FAKE + 8, size, 130, 256, 32, FAKE, None) == _lib.RQ_EINVAL

    def linear(rows=2, x=FAKE, x_stride=256, packed=FAKE, packed_bytes=size, y=FAKE, y_stride=130, group=32):
        return lib.rq_linear_rows_int4(x, x_stride, packed, packed_bytes, y, y_stride, rows, 130, 256, group, None)

    assert linear(rows=65) == _lib.RQ_ENOKERNEL
    assert b"at most 64" in lib.rq_last_error()
    for wrong in (dict(x=FAKE + 8), dict(x=None), dict(x_stride=248), dict(x_stride=260), dict(packed=None),
                  dict(packed_bytes=size - 1), dict(y=None), dict(y=FAKE + 1), dict(y_stride=129)):
        assert linear(**wrong) == _lib.RQ_EINVAL, wrong
    assert linear(group=16) == _lib.RQ_ENOKERNEL
    assert linear(rows=0) == _lib.RQ_OK


def test_logprob_refusals(lib):
    def call(logits=FAKE, stride=100, dtype=0, rows=2, vocab=100, tokens=FAKE, top=4, values=FAKE):
        return lib.rq_token_logprobs(logits, stride, dtype, rows, vocab, tokens, FAKE, FAKE, top, values, FAKE, None)

    for wrong in (dict(dtype=2), dict(rows=-1), dict(vocab=0), dict(stride=99), dict(top=33), dict(top=-1),
                  dict(vocab=3, stride=3), dict(logits=None), dict(logits=FAKE + 1), dict(logits=FAKE + 2, dtype=1),
                  dict(tokens=None), dict(values=None)):
        assert call(**wrong) == _lib.RQ_EINVAL, wrong
    assert call(rows=0) == _lib.RQ_OK


def test_python_refusals():
    rows = torch.zeros((2, 4, 128), dtype=torch.bfloat16)
    cache = torch.zeros((2, 4, 4, 16, 128), dtype=torch.float8_e4m3fn)
    scales = torch.ones((2, 4, 4))
    starts, lens = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    table = torch.zeros((2, 2), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="BF16"):
        ops.quantize_fp8(rows, rows, cache, scales, starts, lens, table)
    with pytest.raises(RuntimeError, match="BF16"):
        ops.paged_attention_fp8(rows, rows, rows, cache, scales, rows, starts, lens, table)
    with pytest.raises(RuntimeError, match="on a HIP device"):
        step_ops.quantize_weight_int4(torch.zeros((64, 64), dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="on a HIP device"):
        step_ops.pack_weight_int4(torch.zeros((64, 64), dtype=torch.int8), torch.zeros((64, 2), dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="on a HIP device"):
        step_ops.token_logprobs(torch.zeros((2, 64)), torch.zeros(2, dtype=torch.int64))


def test_calls_past_a_launch_are_refused(lib):
    """The threads of one launch stay below 2^32: larger calls are refused before they are launched."""
    assert _write(lib, requests=1 << 23) == _lib.RQ_EINVAL
    assert b"Too many rows and requests" in lib.rq_last_error()
    for heads, kv_heads, rows in ((8, 4, (1 << 29) - 1), (64, 64, 1 << 26)):  # tiles of 256 columns, 512 threads
        assert _attend(lib, rows=rows, heads=heads, kv_heads=kv_heads, query_stride=64 * 128, key_stride=64 * 128) == _lib.RQ_EINVAL

    def decode(requests):  # one row each: tiles of 16 columns, 256 threads
        return lib.rq_paged_attention_fp8(FAKE, 64 * 128, FAKE, 64 * 128, FAKE, 64 * 128, FAKE, 64 * 128, requests, 64, 64,
                                          128, FAKE, FAKE, 8, 16, FAKE, FAKE, requests, FAKE, 1, 1, 0.1, FAKE, 1 << 40, None)

    assert decode(1 << 18) == _lib.RQ_EINVAL
    assert b"Too many rows, heads and requests" in lib.rq_last_error()
    assert lib.rq_int4_weight_bytes(1 << 24, 1 << 11, 128) == 0
    assert b"2^35 elements" in lib.rq_last_error()
    assert lib.rq_int4_weight_bytes((1 << 24) - 16, 1 << 11, 128) > 0
