"""The cases of attention over the 4-bit cache reach every kernel that takes a block by itself. Those need no workspace, shares of
all tiles do, so which of both a call takes shows without a device."""
import pytest

import malkin_amd as mk_
from kv4_paths import CASES, path, path_of
from test_kv4_refusals import attention, cache, refused


def shares(H, KV, d, n, most, run):
    kv = cache(n_head_kv=KV, head_dim=d, max_pages=1 << 10)
    rc = attention(n=n, H=H, qs=H * d, os=H * d, kv=kv, most=most, run=run, ws=None, wsb=0)
    text = mk_.load().mk_last_error().decode()
    assert rc == mk_.MK_ERR_INVALID and ("workspace" in text or "null context" in text), text
    return "workspace" in text


def test_all_are_reached():
    reached = {path_of(c) for c in CASES + [(4, 2, 64, 16, [1, 1], [1, 2])]}
    assert {p for p in reached if p[0] == "whole"} == {("whole", d, s, w) for d in (64, 128) for s in (1, 2) for w in (4, 8)}


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:4] + path_of(c)))
def test_the_rule_is_the_librarys(case):
    H, KV, d, page, new, rows = case
    for most in {max(rows), 1, 1024, 1025, 3200, 3201}:
        for run in (1, 2, max(new), 1000):
            args = (H, KV, d, sum(new), most, run)
            assert shares(*args) == (path(*args)[0] == "share"), args


def test_drafts_count_by_their_blocks():
    """8 users with 8 drafts each are 64 blocks, not 512: their documents are shared out past 1024 keys."""
    for n, run in ((64, 8), (64, 4), (120, 5)):
        assert shares(32, 8, 128, n, 3000, run) and not shares(32, 8, 128, n, 1000, run)
    assert not shares(32, 8, 128, 64, 3000, 1) and not shares(32, 8, 128, 512, 3000, 8)
    refused(attention(ws=None, most=0), mk_.MK_ERR_INVALID, "null context")
