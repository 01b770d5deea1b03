"""Projections with 4-bit weights (step_ops.linear_rows_int4) against float64, and the packing."""

from __future__ import annotations

import pytest
import torch

from residualquant_amd import step_ops

pytestmark = pytest.mark.gpu


def _weight(out, features, group, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (out, features), generator=g, dtype=torch.int8)
    scales = (torch.rand((out, features // group), generator=g) * 0.02 + 0.001).to(torch.bfloat16)
    return codes, scales


def _reference(x, codes, scales):
    """(y, bound) in float64.  The bound: one BF16 rounding (2^-8 of y); a group's sum in float32,
    of codes shifted by up to 24 (a term is at most 31 |x| and the shift 24 |x|), each of its
    additions off by 2^-24 of the terms' sum; and one addition per group and 16 more, of the groups' sums."""
    out, groups = scales.shape
    group = codes.size(1) // groups
    xg = x.double().view(-1, groups, group)
    cg = codes.double().view(out, groups, group)
    s = scales.double()
    sums = torch.einsum("mgk,ngk->mng", xg, cg) * s
    y = sums.sum(dim=2)
    shifted = torch.einsum("mg,ng->mn", xg.abs().sum(dim=2), s.abs())
    bound = 2.0 ** -8 * y.abs() + 2.0 ** -24 * (55 * group * shifted + (groups + 16) * sums.abs().sum(dim=2)) + 1e-37
    return y, bound


SHAPES = [
    (1, 16, 32, 32), (1, 1, 128, 128), (2, 17, 64, 64), (3, 100, 160, 32), (16, 48, 256, 64), (17, 33, 384, 128),
    (5, 2048, 2048, 32), (1, 6144, 2048, 32), (12, 2048, 5632, 128), (32, 512, 1024, 64), (33, 130, 96, 32),
    (64, 257, 896, 64), (49, 64, 8192, 128), (8, 31, 4128, 32), (31, 1000, 2240, 64), (4, 4096, 32, 32),
]


@pytest.mark.parametrize("rows,out,features,group", SHAPES)
def test_linear(device, rows, out, features, group):
    print(f"rows={rows} out={out} in={features} group={group}", flush=True)
    codes, scales = _weight(out, features, group, seed=rows + out + features)
    x = torch.randn((rows, features), generator=torch.Generator().manual_seed(rows)).to(torch.bfloat16)
    weight = step_ops.pack_weight_int4(codes.to(device), scales.to(device))
    assert weight.shape == (out, features) and weight.group == group
    got = step_ops.linear_rows_int4(x.to(device), weight).cpu().double()
    want, bound = _reference(x, codes, scales)
    over = (got - want).abs() / bound
    assert over.max() <= 1.0, f"{over.max():.2f} times the bound"


@pytest.mark.parametrize("rows", [1, 7, 16, 17, 40, 64])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_linear_is_exact_on_small_integers(device, rows, group):
    """Integer inputs and powers of two as scales: every sum is exact in float32, so only the output is rounded."""
    out, features = 83, 640
    codes, _ = _weight(out, features, group, seed=rows + group)
    g = torch.Generator().manual_seed(rows)
    scales = torch.exp2(torch.randint(-2, 3, (out, features // group), generator=g).float()).to(torch.bfloat16)
    x = torch.randint(-4, 5, (rows, features), generator=g).to(torch.bfloat16)
    got = step_ops.linear_rows_int4(x.to(device), step_ops.pack_weight_int4(codes.to(device), scales.to(device)))
    want = x.double() @ (codes.double() * scales.double().repeat_interleave(group, dim=1)).t()
    assert torch.equal(got.cpu(), want.to(torch.bfloat16))


@pytest.mark.parametrize("rows,group", [(1, 32), (9, 64), (16, 128), (30, 64), (48, 32), (49, 128), (64, 64)])
@pytest.mark.parametrize("out,features", [(16643, 1152), (5000, 2048), (1037, 6400), (24, 6400)])
def test_wide_and_deep_weights_are_exact_on_small_integers(device, rows, group, out, features):
    """Many outputs or inputs, where x passes through shared memory, whole and in chunks."""
    codes, _ = _weight(out, features, group, seed=rows + out)
    g = torch.Generator().manual_seed(rows)
    scales = torch.exp2(torch.randint(-2, 3, (out, features // group), generator=g).float()).to(torch.bfloat16)
    x = torch.randint(-4, 5, (rows, features), generator=g).to(torch.bfloat16)
    got = step_ops.linear_rows_int4(x.to(device), step_ops.pack_weight_int4(codes.to(device), scales.to(device)))
    # (Below 2^24 in quarters: exact in float32 too, in any order.)
    want = x.float() @ (codes.float() * scales.float().repeat_interleave(group, dim=1)).t()
    assert torch.equal(got.cpu(), want.to(torch.bfloat16))


@pytest.mark.parametrize("rows,features", [(3, 256), (40, 256), (3, 1152), (16, 1152)])
def test_wide_weight_nan_and_infinity(device, rows, features):
    """As the narrow ones: on the row of the NaN or infinity only, the others as without it."""
    out = 16643
    codes, scales = _weight(out, features, 64, seed=8)
    codes[codes == 0] = 1
    weight = step_ops.pack_weight_int4(codes.to(device), scales.to(device))
    x = torch.randn((rows, features), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    plain = step_ops.linear_rows_int4(x.to(device), weight).cpu()
    for value in (torch.inf, torch.nan, 3.3e38):
        y = x.clone()
        y[1, 100] = value
        got = step_ops.linear_rows_int4(y.to(device), weight).cpu()
        want = (y[1].double() @ (codes.double() * scales.double().repeat_interleave(64, dim=1)).t()).to(torch.bfloat16)
        assert torch.equal(got[1].isnan(), want.isnan()) and torch.equal(got[1].isinf(), want.isinf())
        rest = [m for m in range(rows) if m != 1]
        assert torch.allclose(got[rest].double(), plain[rest].double(), rtol=2.0 ** -6, atol=2.0 ** -8)


def test_rows_far_apart(device):
    """Rows 2^24 and more elements apart."""
    codes, scales = _weight(70, 256, 64, seed=5)
    store = torch.zeros(2 * (1 << 24) + 256, dtype=torch.bfloat16, device=device)
    x = store.as_strided((3, 256), (1 << 24, 1))
    x.copy_(torch.randn((3, 256), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16))
    got = step_ops.linear_rows_int4(x, step_ops.pack_weight_int4(codes.to(device), scales.to(device))).cpu().double()
    want, bound = _reference(x.cpu(), codes, scales)
    assert ((got - want).abs() / bound).max() <= 1.0


def test_every_code_at_every_place(device):
    """One-hot inputs read the weight back: code x scale, exact in BF16."""
    out, features = 48, 256
    codes = ((torch.arange(out)[:, None] * 7 + torch.arange(features)[None] * 3) % 16 - 8).to(torch.int8)
    scales = torch.full((out, features // 32), 0.25, dtype=torch.bfloat16)
    weight = step_ops.pack_weight_int4(codes.to(device), scales.to(device))
    assert torch.equal(weight.dequantize().cpu().float(), codes.float() * 0.25)
    eye = torch.eye(features, dtype=torch.bfloat16, device=device)
    rows = torch.cat([step_ops.linear_rows_int4(eye[k:k + 64].contiguous(), weight) for k in range(0, features, 64)])
    assert torch.equal(rows.t().cpu().float(), codes.float() * 0.25)


@pytest.mark.parametrize("rows", [1, 20])
def test_linear_nan_and_infinity(device, rows):
    """A NaN or an infinity in x or in a scale acts as in the sum itself, and on its own row or output only."""
    codes, scales = _weight(40, 256, 32, seed=3)
    codes[codes == 0] = 1
    x = torch.randn((rows, 256), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    last = rows - 1
    for place, value in ((5, torch.inf), (200, -torch.inf), (77, torch.nan), (255, 3.3e38)):
        y = x.clone()
        y[last, place] = value
        got = step_ops.linear_rows_int4(y.to(device), step_ops.pack_weight_int4(codes.to(device), scales.to(device)))
        want = y.double() @ (codes.double() * scales.double().repeat_interleave(32, dim=1)).t()
        got, want = got.cpu().double(), want.to(torch.bfloat16).double()
        assert torch.equal(got.isnan(), want.isnan()), value
        assert torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf()), value
    scales[7, 2], scales[9, 0] = torch.nan, torch.inf
    got = step_ops.linear_rows_int4(x.to(device), step_ops.pack_weight_int4(codes.to(device), scales.to(device))).cpu()
    assert bool(got[:, 7].isnan().all()) and bool((~got[:, 9].isfinite()).all())
    rest = [n for n in range(40) if n not in (7, 9)]
    assert bool(got[:, rest].isfinite().all())


@pytest.mark.parametrize("out,features,group", [(50, 256, 32), (16, 384, 128), (129, 64, 64)])
def test_quantize_weight(device, out, features, group):
    g = torch.Generator().manual_seed(out)
    weight = (torch.randn((out, features), generator=g) * 0.05).to(torch.bfloat16)
    weight[3, :group] = 0.0
    weight[5, 0] = 3.0
    packed = step_ops.quantize_weight_int4(weight.to(device), group)
    grouped = weight.float().view(out, -1, group)
    scales = (grouped.abs().amax(dim=2) / 7).to(torch.bfloat16)
    codes = torch.where(scales[..., None] > 0, torch.round(grouped / scales.float()[..., None]), 0.0).clamp(-8, 7)
    want = (codes * scales.float()[..., None]).view(out, features).to(torch.bfloat16)
    assert torch.equal(packed.dequantize().cpu(), want)
    again = step_ops.pack_weight_int4(codes.to(torch.int8).view(out, features).to(device), scales.to(device))
    assert torch.equal(again.data, packed.data)


def test_quantize_weight_not_finite(device):
    weight = torch.ones((16, 64), dtype=torch.bfloat16, device=device)
    weight[2, 3], weight[4, 40] = torch.nan, torch.inf
    restored = step_ops.quantize_weight_int4(weight, 32).dequantize()
    assert bool(restored[2, :32].isnan().all()) and bool(restored[4, 32:].isnan().all())
    assert bool((restored[2, 32:] == 1).all()) and bool((restored[4, :32] == 1).all())


def test_strides_outputs_and_streams(device):
    codes, scales = _weight(70, 256, 64, seed=9)
    weight = step_ops.pack_weight_int4(codes.to(device), scales.to(device))
    x = torch.randn((6, 256), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(device)
    want = step_ops.linear_rows_int4(x, weight)
    wide = torch.zeros((6, 300 + 4), dtype=torch.bfloat16, device=device)
    wide[:, :256] = x
    out = torch.full((6, 101), 5.0, dtype=torch.bfloat16, device=device)
    step_ops.linear_rows_int4(wide[:, :256], weight, out=out[:, 30:100])
    assert torch.equal(out[:, 30:100], want)
    assert bool((out[:, :30] == 5).all()) and bool((out[:, 100:] == 5).all())
    # A single row whose row stride says nothing.
    single = torch.empty(256, dtype=torch.bfloat16, device=device).copy_(x[2]).as_strided((1, 256), (1, 1))
    assert torch.equal(step_ops.linear_rows_int4(single, weight)[0], step_ops.linear_rows_int4(x[2:3], weight)[0])
    stream = torch.cuda.Stream(device=device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        other = step_ops.linear_rows_int4(x, weight)
    torch.cuda.current_stream(device).wait_stream(stream)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step_ops.linear_rows_int4(x, weight)
    for step in range(3):
        x.copy_(torch.randn((6, 256), generator=torch.Generator().manual_seed(step)).to(torch.bfloat16))
        graph.replay()
        eager = step_ops.linear_rows_int4(x, weight)
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)


def test_empty_and_refusals(device):
    codes, scales = _weight(32, 64, 32, seed=10)
    weight = step_ops.pack_weight_int4(codes.to(device), scales.to(device))
    assert step_ops.linear_rows_int4(torch.empty((0, 64), dtype=torch.bfloat16, device=device), weight).shape == (0, 32)
    with pytest.raises(RuntimeError, match="at most 64"):
        step_ops.linear_rows_int4(torch.zeros((65, 64), dtype=torch.bfloat16, device=device), weight)
    with pytest.raises(RuntimeError, match="in_features"):
        step_ops.linear_rows_int4(torch.zeros((2, 96), dtype=torch.bfloat16, device=device), weight)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        wide = torch.zeros((2, 72), dtype=torch.bfloat16, device=device)
        step_ops.linear_rows_int4(wide[:, 4:68], weight)
    with pytest.raises(RuntimeError, match="groups of 16"):
        step_ops.pack_weight_int4(codes.to(device), torch.ones((32, 4), dtype=torch.bfloat16, device=device))
    with pytest.raises(RuntimeError, match="out must be"):
        step_ops.linear_rows_int4(torch.zeros((2, 64), dtype=torch.bfloat16, device=device), weight,
                                  out=torch.zeros((2, 31), dtype=torch.bfloat16, device=device))


# Beside the codes and through shared memory, whole and in chunks, for one to four row tiles.
ROUTES = [(1, 40, 256, 32), (7, 130, 2048, 64), (16, 300, 5632, 128), (40, 70, 512, 32), (3, 24, 6400, 64),
          (20, 9000, 1152, 32), (33, 5000, 2048, 64), (64, 1037, 6400, 128), (16, 16643, 1152, 64)]


def _far(x):
    """The same rows 2^24 elements apart."""
    store = torch.zeros((x.size(0) - 1) * (1 << 24) + x.size(1), dtype=torch.bfloat16, device=x.device)
    return store.as_strided(x.shape, (1 << 24, 1)).copy_(x)


@pytest.mark.parametrize("rows,out,features,group", ROUTES)
def test_inputs_under_codes_of_zero_add_nothing(device, rows, out, features, group):
    """An input whose codes are all 0 may have any finite size: the outputs are those without it, bit for bit."""
    print(f"rows={rows} out={out} in={features} group={group}", flush=True)
    codes, scales = _weight(out, features, group, seed=rows + out)
    places = [3, features // 2 + 1, features - 1]
    codes[:, places] = 0
    scales[:, 0] = 16.0
    weight = step_ops.pack_weight_int4(codes.to(device), scales.to(device))
    x = torch.randn((rows, features), generator=torch.Generator().manual_seed(rows)).to(torch.bfloat16).to(device)
    x[:, places] = 0
    want = step_ops.linear_rows_int4(x, weight)
    wide = rows <= 3 and step_ops.linear_rows_int4(_far(x), weight)
    for value in (1e3, -1e5, 1e8, 1e20, -3.3e38):
        x[:, places] = value
        assert torch.equal(step_ops.linear_rows_int4(x, weight), want), value
        if rows <= 3:
            assert torch.equal(step_ops.linear_rows_int4(_far(x), weight), wide), value


@pytest.mark.parametrize("rows,out,features,group", ROUTES)
def test_linear_with_outliers(device, rows, out, features, group):
    """Channels of 10^4 times the others' size.  The bound: one BF16 rounding, and each addition of a group's products
    and of the groups' sums off by 2^-23 of the terms' own size (a product of a code and an input is exact)."""
    codes, scales = _weight(out, features, group, seed=rows + out + 1)
    codes[torch.rand(codes.shape, generator=torch.Generator().manual_seed(2)) < 0.3] = 0
    x = torch.randn((rows, features), generator=torch.Generator().manual_seed(rows)).to(torch.bfloat16)
    x[:, 5::97] *= 1e4
    held = scales.double().repeat_interleave(group, dim=1) * codes.double()
    want = x.double() @ held.t()
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -23 * (group + features // group + 16) * (x.double().abs() @ held.abs().t())
    got = step_ops.linear_rows_int4(x.to(device), step_ops.pack_weight_int4(codes.to(device), scales.to(device)))
    over = (got.cpu().double() - want).abs() / bound
    assert over.max() <= 1.0, f"{over.max():.2f} times the bound"


@pytest.mark.parametrize("rows,out,features,group", ROUTES)
def test_nan_and_infinity_leave_other_outputs_alone(device, rows, out, features, group):
    """A row or an output with NaN or infinities is what float64 makes of it, and every other one as without, bit for bit."""
    codes, scales = _weight(out, features, group, seed=rows + out + 2)
    x = torch.randn((rows, features), generator=torch.Generator().manual_seed(rows)).to(torch.bfloat16)
    weight = step_ops.pack_weight_int4(codes.to(device), scales.to(device))
    plain = step_ops.linear_rows_int4(x.to(device), weight).cpu()
    held = codes.double() * scales.double().repeat_interleave(group, dim=1)
    hit = rows // 2
    rest = [m for m in range(rows) if m != hit]
    for place, value in ((0, torch.inf), (features - 1, -torch.inf), (features // 3, torch.nan), (features // 2, 3.3e38)):
        y = x.clone()
        y[hit, place] = value
        got = step_ops.linear_rows_int4(y.to(device), weight).cpu()
        want = (y[hit].double() @ held.t()).to(torch.bfloat16)
        assert torch.equal(got[hit].isnan(), want.isnan()), value
        assert torch.equal(got[hit].isposinf(), want.isposinf()) and torch.equal(got[hit].isneginf(), want.isneginf()), value
        assert torch.equal(got[rest], plain[rest]), value
    scales[out // 2, -1], scales[out - 1, 0] = torch.nan, torch.inf
    codes[out - 1, 0], codes[out - 1, 1:group] = 1, 0  # (an infinite scale times one term: no NaN from codes of 0)
    x[:, 0] = x[:, 0].abs() + 1
    plain = step_ops.linear_rows_int4(x.to(device), weight).cpu()
    got = step_ops.linear_rows_int4(x.to(device), step_ops.pack_weight_int4(codes.to(device), scales.to(device))).cpu()
    assert bool(got[:, out // 2].isnan().all()) and bool(got[:, out - 1].isposinf().all())
    rest = [n for n in range(out - 1) if n != out // 2]
    assert torch.equal(got[:, rest], plain[:, rest])
