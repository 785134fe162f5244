"""What the entry points over a paged cache refuse at their limits, before anything is launched.  No GPU needed."""

import ctypes

import pytest

from flash_colsum_b200 import _cabi
from test_paged_cpu import ADDRESS, append, attend, cache, rows, strides


@pytest.mark.parametrize("k", [2 ** 26 + 1, 2 ** 27, 2 ** 31 - 1])
def test_lists_that_the_attention_cannot_count_are_refused(k):
    assert attend(k=k) < 0
    assert "at most 67108864 pages" in _cabi.last_error()


@pytest.mark.parametrize("stride", [(0, 128), (1024, 0), (0, 0), (1024, 120), (1016, 128), (128, 128), (128, 632), (8, 1024)])
def test_results_whose_rows_overlap_are_refused(stride):
    """Five tokens of eight heads of 128."""
    assert append(r=rows(query_out_stride=stride)) < 0
    assert "query_out strides must keep its rows apart" in _cabi.last_error()
    assert attend(out_st=stride) < 0
    assert "out strides must keep its rows apart" in _cabi.last_error()


@pytest.mark.parametrize("tokens,heads,stride", [(5, 8, (1024, 128)), (5, 8, (128, 640)), (5, 8, (1024, 1 << 40)), (1, 8, (0, 128)), (5, 1, (128, 0)),
                                                 (1, 1, (0, 0))])
def test_results_whose_rows_do_not_are_checked_further(tokens, heads, stride):
    c = cache(tokens=tokens, kv_heads=1)
    assert attend(c, heads=heads, out_st=stride, k=0) < 0
    assert "chosen" in _cabi.last_error()


@pytest.mark.parametrize("changes,word", [(dict(status=None), "status"), (dict(limit=0.0), "limit_seconds"), (dict(limit=2.5), "limit_seconds")])
def test_the_selftests_of_the_waits_check_their_arguments(changes, word):
    limit, status = changes.get("limit", 0.05), changes.get("status", ADDRESS)
    lib, c = _cabi.load(), ctypes.byref(cache())
    assert lib.fcs_selftest_wait_expiry_select(c, ADDRESS, strides(1024, 128), 8, ADDRESS, 4, 1, 1, ADDRESS, ADDRESS, 1 << 40, status, limit, None) < 0
    assert word in _cabi.last_error()
    assert lib.fcs_selftest_wait_expiry_attend(c, ADDRESS, strides(1024, 128), 8, ADDRESS, 4, 0.1, ADDRESS, strides(1024, 128), None, status, limit,
                                               None) < 0
    assert word in _cabi.last_error()


def test_plans_of_calls_over_a_paged_cache():
    """Host arithmetic, of 148 SMs where there is no device."""
    c = cache(sequences=32, tokens=32, starts=None, kv_heads=8, table_width=512, table_stride=512)
    p = _cabi.paged_plan(c, 32, 32)
    assert (p["append_heads"], p["append_steps"]) == (8, 1)
    assert (p["select_tiles"], p["select_ctas"], p["select_launches"]) == (0, 2, 1)
    assert (p["attend_tokens"], p["attend_queries"], p["attend_ctas"]) == (1, 8, 1)
    c = cache(sequences=1, tokens=512, kv_heads=8, table_width=512, table_stride=512)
    p = _cabi.paged_plan(c, 32, 32)
    assert p["select_tiles"] == 1 and (p["attend_tokens"], p["attend_ctas"]) == (4, 1)
    assert _cabi.paged_plan(cache(sequences=1, tokens=16384, kv_heads=8), 32, 1)["append_steps"] == 4
    assert _cabi.paged_plan(cache(sequences=1, tokens=1000, kv_heads=8, table_width=8192, table_stride=8192), 32, 48)["select_launches"] == 3
    assert _cabi.paged_plan(c, 0, 1)["attend_ctas"] == 0
    for heads, k in ((7, 1), (-8, 1), (8, 0)):
        with pytest.raises(RuntimeError, match="rejected"):
            _cabi.paged_plan(c, heads, k)
    with pytest.raises(RuntimeError, match="page size"):
        _cabi.paged_plan(cache(page_size=8), 8, 1)


@pytest.mark.parametrize("stride", [(128, 128, 128), (0, 8192, 128), (16384, 0, 128), (16384, 8192, 0), (16384, 8192, 120), (16384, 8184, 128),
                                    (16376, 8192, 128), (16384, 128, 248), (128, 1280, 2552)])
def test_pools_whose_rows_overlap_are_not_written(stride):
    """Ten pages of two heads of 64 slots of 128 features."""
    for name in ("key", "value"):
        assert append(cache(**{name + "_stride": stride})) < 0
        assert f"{name}_pages strides must keep its rows apart" in _cabi.last_error()
