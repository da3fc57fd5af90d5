"""The stride that an 8-bit product takes for its rows where none is named.  No GPU: the call's arguments are looked at."""
import pytest
import torch

from tinytitan_amd.engine import Int8Projection


class Context:
    handle = 1

    class _calls:
        @staticmethod
        def int8_projection(ctx, weights, weight_scales, x, x_stride, y, rows, columns, tokens, y_stride):
            Context.strides = x_stride, y_stride
            return 0

        @staticmethod
        def int8_quantise_rows(ctx, x, x_stride, tokens, columns, levels, levels_stride, scales):
            Context.strides = x_stride, levels_stride
            return 0

        @staticmethod
        def int8_projection_levels(ctx, weights, weight_scales, levels, levels_stride, scales, y, rows, columns, tokens, y_stride):
            Context.strides = levels_stride, y_stride
            return 0


def _strides(of, to, of_stride=None, to_stride=None, columns=32, rows=16, tokens=5):
    """What the three calls take for the rows `of` and `to`, the same where they have the same widths."""
    projection, found = Int8Projection(Context), []
    projection.encode(None, None, of, to, rows, columns, tokens, x_stride=of_stride, y_stride=to_stride)
    found.append(Context.strides)
    projection.encode_levels(None, None, of, None, to, rows, columns, tokens, levels_stride=of_stride, y_stride=to_stride)
    found.append(Context.strides)
    if rows == columns:
        projection.quantise(of, to, None, columns, tokens, x_stride=of_stride, levels_stride=to_stride)
        found.append(Context.strides)
    assert len(set(found)) == 1
    return found[0]


def test_strides_of_rows():
    wide = torch.zeros(5, 100)
    assert _strides(torch.zeros(5, 32), torch.zeros(5, 16)) == (32, 16)
    assert _strides(wide[:, 3:35], wide[:, :16]) == (100, 100)
    assert _strides(wide[:, 3:35], wide[:, :32], rows=32) == (100, 100)
    assert _strides(wide[:, 3:35], wide[:, :16], 48, 24) == (48, 24)  # (as named)
    assert _strides(wide[:, :16].unflatten(1, (4, 4)), wide[:, :16], columns=16) == (100, 100)
    assert _strides(wide[::2, :32], torch.zeros(3, 16), tokens=3) == (200, 16)
    # without gaps: wherever a row of the tensor ends
    assert _strides(torch.zeros(160), torch.zeros(2, 40)) == (32, 16)
    assert _strides(wide, wide[0]) == (32, 16)
    assert _strides(wide[:1, :32], wide[:1, :16], tokens=1) == (32, 16)
    assert _strides(None, None) == (32, 16)


def test_rows_that_are_none_are_refused():
    wide = torch.zeros(5, 100)
    good = torch.zeros(5, 32)
    for bad in (wide[:, :64:2], wide[:, :31], wide[:, :64], torch.zeros(32, 5).T, torch.zeros(200)[::2], wide[:, :64].unflatten(1, (2, 32))):
        with pytest.raises(TypeError):
            _strides(bad, good, rows=32)
        with pytest.raises(TypeError):
            _strides(good, bad, rows=32)
        assert _strides(bad, bad, 40, 48, rows=32) == (40, 48)
