"""Operators on score rows: what can be checked without a GPU."""
import ctypes as C

import pytest
import torch

from coral_b200 import capi


def test_row_layout():
    lib = capi.load()
    for dim in (1, 15, 16, 17, 127, 128, 200, 511, 512, 513, 4096, 65536):
        cp, sp = lib.coral_fp8_code_pitch(dim), lib.coral_fp8_scale_pitch(dim)
        assert cp % 16 == 0 and dim <= cp < dim + 16
        assert sp % 4 == 0 and sp >= -(-dim // 128) and (sp - 4) * 128 < dim
    for dim in (0, -1, capi.FP8_MAX_DIM + 1):
        assert lib.coral_fp8_code_pitch(dim) == 0 and lib.coral_fp8_scale_pitch(dim) == 0


def test_a_null_handle_is_refused():
    lib = capi.load()
    n = C.c_int64(0)
    assert lib.coral_fp8_quantize(None, None, 0, 1, 4, 4, None, None, None) == capi.ERR_ARG
    assert lib.coral_fp8_scores(None, None, None, 1, None, None, 1, 4, 1.0, None, None, 0, 1, None) == capi.ERR_ARG
    assert lib.coral_adjust_scores(None, None, 0, 1, 1, 1, None, 0, None, None, None, 0, None, 0, None, 1, None) == capi.ERR_ARG
    assert lib.coral_topk_workspace(None, 1, 1, 1, C.byref(n)) == capi.ERR_ARG
    assert lib.coral_topk_scores(None, None, 0, 1, 1, 1, 1, 0, None, None, None, 0, None) == capi.ERR_ARG
    assert lib.coral_scores_check(None) == capi.ERR_ARG


def test_the_binding_refuses_before_it_calls():
    """CPU tensors, types and shapes are refused without a device."""
    ix = object.__new__(capi.Index)
    ix._lib, ix._h, ix.device, ix._topk_bytes = capi.load(), None, 0, {}
    x = torch.zeros(4, 64)
    for call in (lambda: ix.fp8_quantize(x), lambda: ix.fp8_scores((x, x), (x, x), 64), lambda: ix.fp8_scores((x, x), (x, x), 0),
                 lambda: ix.adjust_scores(x), lambda: ix.topk_scores(x, 3)):
        with pytest.raises(capi.CoralError) as e:
            call()
        assert e.value.code == capi.ERR_ARG
