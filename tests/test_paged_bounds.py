"""The bounds of tests/paged_cases.py against results with a part planted out of
them: a token, a tile, a wave's or a workgroup's run, wherever it lies."""
import numpy as np
import pytest

from tests.paged_cases import CALLS, TILE, name

HALF_STEP = 2.0 ** -24


@pytest.mark.parametrize("call", CALLS, ids=name)
def test_a_lost_part_is_beyond_the_bound(call):
    set_, chunk, _ = call.line()
    share = -(-chunk // (call.waves // set_))
    for n in sorted(set(call.lens)):
        if n == 0:
            continue
        first = call.first(n)
        for head in sorted({0, call.hq - 1}):
            ref, lse = call.reference(n, head)
            bound, lse_bound = call.out_bound(ref, HALF_STEP), call.lse_bound(lse)
            for size in (1, TILE, share * TILE, chunk * TILE):
                for at in (first, (first + n) // 2 // TILE * TILE, max(first, n - size)):
                    if size == 1 and n - first > 2:                    # (a token of weight 1)
                        at += -at % 3 if at - at % 3 < first else -(at % 3)
                    lost = np.arange(at, min(at + size, n))
                    lost = lost[lost >= first]
                    got, got_lse = call.reference(n, head, lost)
                    weight_shows = abs(got_lse - lse) > lse_bound
                    assert weight_shows or size == 1, (n, head, size, at)
                    # (a request of one channel keeps its mean without some of its tokens)
                    assert (np.abs(got - ref) > bound).any() or (weight_shows and (ref > 0).sum() == 1), (n, head, size, at)


def test_the_calls_cover_both_joins_and_sets():
    for call in CALLS:
        assert call.joins_in_two_steps() == call.two_steps, name(call)
        assert (call.line()[0] > 1) == call.sets, name(call)
