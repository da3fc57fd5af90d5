"""Tensors of the 8-bit products that are views of wider ones: scales that are a column are refused, not read as if they lay next to each other,
and rows without a named stride have their tensor's."""
import numpy as np
import pytest

from tests.test_gpu_int8_projection import _dev, _tokens, _weights, check, quantised

pytestmark = pytest.mark.gpu

TOKENS, ROWS, COLUMNS = 6, 40, 256


@pytest.fixture
def products(gpu_ctx):
    """(projection, x, weights, weight scales, numpy of the last three)."""
    import torch
    from tinytitan_amd.engine import Int8Projection
    r = np.random.default_rng(1)
    w, ws = _weights(r, ROWS, COLUMNS)
    x = _tokens(r, TOKENS, COLUMNS)
    made = Int8Projection(gpu_ctx), _dev(x), _dev(w), _dev(ws), x, w, ws
    torch.cuda.synchronize()
    return made


def _column(values):
    """`values` as a column of a wider tensor: [n, 1], two elements from one to the next."""
    import torch
    wide = torch.stack([values, torch.full_like(values, 7.0)], 1).contiguous()
    return wide[:, :1]


def test_scales_that_are_a_column(gpu_ctx, products):
    import torch
    projection, x, weights, weight_scales, nx, nw, nws = products
    y = torch.full((TOKENS, ROWS), 3.0, dtype=torch.float16, device="cuda")
    levels, scales = torch.full((TOKENS, COLUMNS), 9, dtype=torch.int8, device="cuda"), torch.full((TOKENS,), 9.0, device="cuda")
    torch.cuda.synchronize()
    for strided in (_column(weight_scales), _column(weight_scales)[:, 0]):
        with pytest.raises(TypeError):
            projection.encode(weights, strided, x, y, ROWS, COLUMNS, TOKENS)
        with pytest.raises(TypeError):
            projection.encode_levels(weights, strided, levels, scales, y, ROWS, COLUMNS, TOKENS)
    for strided in (_column(scales), _column(scales)[:, 0]):
        with pytest.raises(TypeError):
            projection.quantise(x, levels, strided, COLUMNS, TOKENS)
        with pytest.raises(TypeError):
            projection.encode_levels(weights, weight_scales, levels, strided, y, ROWS, COLUMNS, TOKENS)
        assert (strided == 9.0).all()
    gpu_ctx.synchronize()
    assert (y == 3.0).all() and (levels == 9).all() and (scales == 9.0).all()
    # a column by itself is a vector
    projection.quantise(x, levels, scales[:, None], COLUMNS, TOKENS)
    projection.encode_levels(weights, weight_scales[:, None], levels, scales[:, None], y, ROWS, COLUMNS, TOKENS)
    gpu_ctx.synchronize()
    exact_levels, exact_scales = quantised(nx)
    assert np.array_equal(scales.cpu().numpy(), exact_scales)
    check(y.cpu().numpy(), exact_levels, exact_scales, nw, nws)


def test_levels_that_are_a_column(gpu_ctx, products):
    import torch
    projection, x, weights, weight_scales, _, _, _ = products
    wide = torch.full((COLUMNS, 2), 9, dtype=torch.int8, device="cuda")
    y, scale = torch.full((1, ROWS), 3.0, dtype=torch.float16, device="cuda"), torch.full((1,), 9.0, device="cuda")
    torch.cuda.synchronize()
    for strided in (wide[:, :1], wide[:, 0], wide[:, :1].T):
        with pytest.raises(TypeError):
            projection.quantise(x[:1], strided, scale, COLUMNS, 1)
        with pytest.raises(TypeError):
            projection.encode_levels(weights, weight_scales, strided, scale, y, ROWS, COLUMNS, 1)
    gpu_ctx.synchronize()
    assert (wide == 9).all() and (y == 3.0).all() and (scale == 9.0).all()


def test_factors_of_one_head_in_a_wider_buffer(gpu_ctx):
    # (the factors of differential attention are rows of any stride, those of one head a column)
    import torch
    from tests.exact_maps import check as check_maps
    from tests.test_gpu_attn_diff import Layer, _randn
    from tinytitan_amd.engine import DifferentialHeads
    layer = Layer(gpu_ctx, 1, 1, 64, [40, 700, 90])
    wide = _dev(np.random.default_rng(1).random((3, 5)).astype(np.float32))
    heads = DifferentialHeads(wide[:, 2:3])
    q = _randn(5, 3, 1, 64)
    torch.cuda.synchronize()
    got = layer.decode(q, [40, 700, 90], heads)
    for i, length in enumerate((40, 700, 90)):
        check_maps(got[i:i + 1], layer.want(q[i:i + 1], i, [length - 1], heads, lambdas=wide[i, 2:3]), f"sequence {i}")
    layer.close()


@pytest.mark.parametrize("tokens", [1, 2, 6, 80])
def test_rows_of_wider_buffers_without_a_named_stride(gpu_ctx, tokens):
    import torch
    from tinytitan_amd.engine import Int8Projection
    r = np.random.default_rng(tokens)
    w, ws = _weights(r, ROWS, COLUMNS)
    nx = _tokens(r, tokens, COLUMNS)
    exact_levels, exact_scales = quantised(nx)
    projection, weights, weight_scales = Int8Projection(gpu_ctx), _dev(w), _dev(ws)
    wide = [torch.full((tokens, width), fill, dtype=kind, device="cuda") for width, fill, kind in (
        (COLUMNS + 24, float("nan"), torch.float16), (COLUMNS + 48, 9, torch.int8), (ROWS + 5, 3.0, torch.float16), (ROWS + 5, 3.0, torch.float16))]
    x, levels, first, second = wide[0][:, 8:8 + COLUMNS], wide[1][:, 16:16 + COLUMNS], wide[2][:, 3:3 + ROWS], wide[3][:, 3:3 + ROWS].unflatten(1, (8, 5))
    x.copy_(_dev(nx))
    scales = torch.full((tokens,), 9.0, device="cuda")
    torch.cuda.synchronize()
    projection.encode(weights, weight_scales, x, first, ROWS, COLUMNS, tokens)
    projection.quantise(x, levels, scales, COLUMNS, tokens)
    projection.encode_levels(weights, weight_scales, levels, scales, second, ROWS, COLUMNS, tokens)
    gpu_ctx.synchronize()
    assert np.array_equal(levels.cpu().numpy(), exact_levels) and np.array_equal(scales.cpu().numpy(), exact_scales)
    check(first.cpu().numpy(), exact_levels, exact_scales, w, ws)
    assert torch.equal(second.flatten(1), first)
    for buffer, at, width, fill in ((wide[1], 16, COLUMNS, 9), (wide[2], 3, ROWS, 3.0), (wide[3], 3, ROWS, 3.0)):
        assert (buffer[:, :at] == fill).all() and (buffer[:, at + width:] == fill).all()


def test_more_tokens_than_a_launch_has_workgroups_are_refused(gpu_ctx, products):
    from tinytitan_amd import capi
    projection, x, weights, weight_scales, _, _, _ = products
    import torch
    y, levels, scales = torch.zeros(TOKENS, ROWS, dtype=torch.float16, device="cuda"), torch.zeros(TOKENS, COLUMNS, dtype=torch.int8, device="cuda"), torch.zeros(TOKENS, device="cuda")
    lib, many = gpu_ctx._lib, 1 << 24
    assert lib.tt_hip_int8_quantise_rows(gpu_ctx.handle, x.data_ptr(), COLUMNS, many, COLUMNS, levels.data_ptr(), COLUMNS, scales.data_ptr()) == capi.ERR_SHAPE
    assert lib.tt_hip_int8_projection(gpu_ctx.handle, weights.data_ptr(), weight_scales.data_ptr(), x.data_ptr(), COLUMNS, y.data_ptr(), ROWS, COLUMNS, many,
                                      ROWS) == capi.ERR_SHAPE
    gpu_ctx.synchronize()
    assert not levels.any() and not y.any()
