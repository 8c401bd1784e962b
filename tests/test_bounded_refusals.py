"""Calls of the window and eviction entries that are refused before anything is launched, without a GPU."""
import pytest

from test_bounded_host import EVICT, FAKE, INVALID, WORKSPACE, i32, i64, ptrs, run


@pytest.mark.parametrize("width,bad,status", [
    (3, {}, INVALID), (4, {}, WORKSPACE),                                             # budget 64, pages of 16 rows
    (1, dict(wrows=16), WORKSPACE), (1, dict(wrows=17), INVALID),                     # the weights hold fewer rows
    (1, dict(pages=1), WORKSPACE), (2, dict(strides=i64(2)), WORKSPACE), (1, dict(strides=i64(2)), INVALID),
    (7, dict(budgets=i32(1 << 30)), INVALID), (8, dict(budgets=i32(1 << 30)), WORKSPACE),
])
def test_evict_needs_a_place_for_every_kept_row(width, bad, status):
    assert run("abkv_evict_by_weight", EVICT, dict(dst=ptrs(FAKE + 4), dstrides=i64(width), **bad)) == status
