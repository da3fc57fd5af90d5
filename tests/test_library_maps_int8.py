"""Host-side checks of differential attention and of the 8-bit products: null handles, shapes of the heads' factors.  No GPU."""
import ctypes
import os

import pytest
import torch

from tinytitan_amd import capi

pytestmark = pytest.mark.skipif(not os.path.exists(capi.LIB_PATH), reason="library not built")


def test_null_handles_are_errors_not_crashes():
    lib, bad = capi.lib(), capi.ERR_INVALID_ARGUMENT
    assert lib.tt_hip_attn_decode_diff(None, None, 0, 1, None, None, 0, 8, None, None, 1.0, None, 0, None, 0.0, 1.0, None) == bad
    assert lib.tt_hip_attn_verify_diff(None, None, 0, 1, None, None, 2, 0, 8, None, None, 1.0, None, 0, None, 0.0, 1.0, None) == bad
    assert lib.tt_hip_attn_prefill_diff(None, None, 0, 0, 0, 1, 1, 0, 8, None, 0, None, 0, 1.0, None, 0, None, 0.0, 1.0, None, 0) == bad
    assert lib.tt_hip_diff_lambda(None, None, None, None, None, 0, 1, 1, 0.8, None) == bad
    assert lib.tt_hip_int8_projection(None, None, None, None, 0, None, 1, 16, 1, 0) == bad
    assert lib.tt_hip_int8_quantise_rows(None, None, 0, 1, 16, None, 0, None) == bad
    assert lib.tt_hip_int8_projection_levels(None, None, None, None, 0, None, None, 1, 16, 1, 0) == bad


def test_per_step_calls_take_host_tensors_for_an_error():
    calls = capi.calls()
    half, single, level = torch.zeros(4, dtype=torch.float16), torch.zeros(4), torch.zeros(4, dtype=torch.int8)
    with pytest.raises(TypeError):
        calls.int8_projection(None, level, None, None, 16, None, 1, 16, 1, 1)
    with pytest.raises(TypeError):
        calls.int8_projection(None, None, single, None, 16, None, 1, 16, 1, 1)
    with pytest.raises(TypeError):
        calls.attn_decode_diff(None, None, 0, 0, 5, 0, 8, half, None, 1.0, None, 0, None, 0.0, 1.0, None)
    with pytest.raises(TypeError):
        calls.attn_decode_diff(None, None, 0, 0, 5, 0, 8, None, None, 1.0, single, 0, None, 0.0, 1.0, None)
    assert calls.attn_decode_diff(None, None, 0, [0, 1], [5], 0, 8, None, None, 1.0, None, 0, None, 0.0, 1.0, None) == capi.ERR_INVALID_ARGUMENT
    assert calls.attn_verify_diff(None, None, 0, [0], [5, 6], 2, 0, 8, None, None, 1.0, None, 0, None, 0.0, 1.0, None) == capi.ERR_INVALID_ARGUMENT


def test_rows_of_factors():
    from tinytitan_amd.engine import DifferentialHeads, TinyTitanHIPError
    wide = torch.zeros(5, 20)
    assert DifferentialHeads(torch.zeros(8)).stride(8, 5) == 0
    assert DifferentialHeads(torch.zeros(5, 8)).stride(8, 5) == 8
    assert DifferentialHeads(wide[:, 3:11]).stride(8, 5) == 20
    assert DifferentialHeads(torch.zeros(1, 8)).stride(8, 1) == 8
    for shape in ((7,), (8, 5), (4, 8), (1, 8), (5, 1, 8), ()):
        with pytest.raises(TinyTitanHIPError) as e:
            DifferentialHeads(torch.zeros(shape)).stride(8, 5)
        assert e.value.status == capi.ERR_SHAPE
    with pytest.raises(TinyTitanHIPError):
        DifferentialHeads(wide.expand(5, 20)[:1].expand(5, 20)[:, :8]).stride(8, 5)  # one row stood in for five is [heads], not a stride of 0
    DifferentialHeads(torch.zeros(8), torch.zeros(64, dtype=torch.bfloat16)).check(64)
    for norm in (torch.zeros(32, dtype=torch.bfloat16), torch.zeros(128, dtype=torch.bfloat16)[::2]):
        with pytest.raises(TinyTitanHIPError):
            DifferentialHeads(torch.zeros(8), norm).check(64)
    with pytest.raises(TinyTitanHIPError) as e:
        DifferentialHeads(torch.zeros(8), torch.zeros(64, dtype=torch.float16)).check(64)
    assert e.value.status == capi.ERR_INVALID_ARGUMENT


def test_signatures_match_the_header():
    for name in ("tt_hip_attn_decode_diff", "tt_hip_attn_verify_diff", "tt_hip_attn_prefill_diff", "tt_hip_diff_lambda", "tt_hip_int8_projection",
                 "tt_hip_int8_quantise_rows", "tt_hip_int8_projection_levels"):
        declared = open(capi.HEADER_PATH).read().split(name + "(")[-1].split(")")[0]
        assert len(capi._SIGNATURES[name][1]) == declared.count(",") + 1, name
    assert ctypes.sizeof(ctypes.c_float) == 4
