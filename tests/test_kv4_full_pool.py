"""The model of growth on a full pool, by itself: no row that an entry may write is another's, whatever runs out."""
import numpy as np
import pytest

from kv4_cases import fork_model
from kv4_full_pool import resize_in_order, written_pages


def pool(n_seq, max_pages, n_page):
    return {"table": np.full((n_seq, max_pages), -1, np.int32), "len": np.zeros(n_seq, np.int32), "refs": np.zeros(n_page, np.int32)}


def test_two_that_share_and_nothing_free():
    a = pool(2, 2, 2)
    assert resize_in_order(a, 16, [0], [20]) == ([0], [])
    fork_model(a, 16, [1], [0])
    assert resize_in_order(a, 16, [1], [18]) == ([0], [])
    assert resize_in_order(a, 16, [0, 1], [21, 19]) == ([1, 1], [])
    assert list(a["len"]) == [20, 18] and list(a["refs"]) == [2, 2]
    assert resize_in_order(a, 16, [0, 1], [20, 16]) == ([0, 0], [])  # one leaves the page
    assert resize_in_order(a, 16, [0], [21]) == ([0], [])


@pytest.mark.parametrize("page", [4, 16])
def test_no_row_is_anothers(page):
    rng = np.random.default_rng(page)
    failed = shared = 0
    for life in range(150):
        a = pool(6, 5, int(rng.integers(6, 16)))
        for step in range(12):
            fork_model(a, page, None, [int(x) for x in np.where(rng.random(6) < 0.5, np.arange(6), rng.integers(-1, 6, 6))])
            seq = [int(x) for x in rng.permutation(6)]
            new = [int(x) for x in np.clip(a["len"][seq] + rng.integers(-page // 2, page, 6), 0, 5 * page)]
            before = a["len"].copy()
            status, _ = resize_in_order(a, page, seq, new)
            assert np.array_equal(np.bincount(a["table"][a["table"] >= 0], minlength=len(a["refs"])), a["refs"])
            for s, p in written_pages(a, page, seq, before, [st if L > before[s] else 1 for s, L, st in zip(seq, new, status)]):
                assert a["refs"][p] == 1
            failed += status.count(1)
            shared += int((a["refs"] > 1).sum())
    assert failed > 100 and shared > 100
