"""Refusals of the score operators: sizes that no array has."""
import pytest
import torch

from coral_b200 import capi

pytestmark = pytest.mark.gpu


@pytest.fixture
def ix():
    with capi.Index(1, 4, 32, "ip") as h:
        yield h
        torch.cuda.synchronize()


def test_rows_that_reach_too_far(ix):
    """Strides whose last row's offset overflows, or nearly: refused, whatever the checks of overlap make of them."""
    lib, h = ix._lib, ix._h
    buf = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    d, far, L, OK = buf.data_ptr(), (1 << 31) - 1, capi.ERR_LIMIT, capi.OK
    e = d + (1 << 19)
    for rows, ld in ((far, far), (far, 1 << 16), (1 << 20, 1 << 29), (3, 1 << 61)):
        if ld <= far:
            assert lib.coral_fp8_quantize(h, d, 0, rows, 64, ld, e, e, 1) == L
            assert lib.coral_fp8_scores(h, d, d, rows, d, d, 1, 64, 1.0, None, e, 0, ld, 1) == L
            assert lib.coral_adjust_scores(h, d, 0, rows, 1, ld, None, 0, None, None, None, 0, None, 0, e, 1, 1) == L
            assert lib.coral_adjust_scores(h, d, 0, rows, 1, 1, None, 0, None, None, None, 0, None, 0, e, ld, 1) == L
            assert lib.coral_topk_scores(h, d, 0, rows, 1, ld, 1, 0, e, e, None, 0, 1) == L
        assert lib.coral_adjust_scores(h, d, 0, rows, 1, 1, None, 0, None, None, None, 0, d, ld, e, 1, 1) == L
    # rows of many columns that fill more than any memory: more CTAs than a grid has
    assert lib.coral_topk_scores(h, d, 0, far, far, far, 1, 0, e, e, e, 1 << 62, 1) == L
    # one row has no next one
    assert lib.coral_topk_scores(h, d, 0, 1, 16, far, 2, 0, e, e + 64, None, 0, 1) == OK
    assert lib.coral_adjust_scores(h, d, 0, 1, 16, far, None, 0, None, None, None, 0, d, 1 << 61, e, far, 1) == OK
    torch.cuda.synchronize()


def test_types_that_are_none(ix):
    """What is no type, and what is no tensor, is refused as every argument is."""
    x = torch.randn(4, 64, device="cuda")
    q = ix.fp8_quantize(x)
    for kw in ({"dtype": "float32"}, {"dtype": float}, {"dtype": torch.float64}, {"out": 5}, {"out": 5, "dtype": torch.float32},
               {"out": [[0.0] * 4] * 4, "dtype": torch.float32}):
        with pytest.raises(capi.CoralError) as e:
            ix.fp8_scores(q, q, 64, **kw)
        assert e.value.code == capi.ERR_ARG


def test_empty_rows_may_be_far_apart(ix):
    """No column, however many rows and whatever the distance between them: nothing to do, nothing to refuse."""
    lib, h, far, OK = ix._lib, ix._h, (1 << 31) - 1, capi.OK
    assert lib.coral_fp8_scores(h, None, None, far, None, None, 0, 64, 1.0, None, None, 0, far, 1) == OK
    assert lib.coral_adjust_scores(h, None, 0, far, 0, far, None, 0, None, None, None, 0, None, 0, None, far, 1) == OK
    assert lib.coral_fp8_quantize(h, None, 0, 0, 64, far, None, None, 1) == OK
    pad = torch.zeros(2, 3, 2, dtype=torch.int32, device="cuda")
    assert lib.coral_topk_scores(h, None, 0, 3, 0, far, 2, 0, pad[0].data_ptr(), pad[1].data_ptr(), None, 0, 1) == OK
    assert bool((pad[0] == -1).all()) and bool((pad[1].view(torch.float32) == -3.4028234663852886e38).all())
