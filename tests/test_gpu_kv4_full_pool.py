"""The 4-bit cache where its pool runs out: who grows, and that nobody's rows change by what others write."""
import numpy as np
import pytest

import malkin_amd as mk_
import test_gpu_pages
from kv4_cases import copied, in4, packed
from kv4_full_pool import resize_in_order, written_pages
from test_gpu_kv4 import write_call

pytestmark = pytest.mark.gpu


class Pool(test_gpu_pages.Pool):
    def resize(self, seq, new_len):
        """Statuses, and that pages written from now on are one sequence's."""
        n, before = len(new_len), self.a["len"].copy()
        L, (w, need) = mk_.load(), self.work(mk_.load().mk_kv4_resize_workspace(n, self.n_page))
        status = self.mk.to_device(np.full(n + 1, 77, np.int32))
        mk_.check(L.mk_kv4_resize(self.mk.h, self.c.ref, self.up(seq), self.up(new_len), n, status.ptr, w.ptr, need))
        got = [int(x) for x in status.download(np.int32)]
        want, moves = resize_in_order(self.a, self.page, seq, [int(x) for x in new_len])
        assert got == want + [77]
        copied(self.a, moves, self.page)
        self.check()
        assert (w.download(np.uint8)[need:] == 0xA5).all()
        order = range(n) if seq is None else seq
        grew = [0 if st == 0 and L > before[s] else 1 for s, L, st in zip(order, new_len, got)]
        for s, p in written_pages(self.a, self.page, seq, before, grew):
            assert self.a["refs"][p] == 1
        return want


@pytest.mark.parametrize("order", [[0, 1], [1, 0]])
def test_sharers_of_unequal_length(mk, order):
    """20 and 18 rows, one page in common that is not full: neither has a page for its copy."""
    p = Pool(mk, np.random.default_rng(1), 2, 3, 16, 2, 128, 3, 2)
    p.resize([0, 2], [20, 5])
    p.fork([1], [0])
    p.resize([1], [18])
    want = {0: 21, 1: 19}
    print("full pool, unequal", order, flush=True)
    assert p.resize(order, [want[s] for s in order]) == [1, 1]
    assert p.resize([2], [0]) == [0]  # its page serves one of them, and the other keeps the old one
    assert p.resize(order, [want[s] for s in order]) == [0, 0]


def test_equal_lengths_in_turns(mk):
    """Sharers whose entries come in another order after a fork, twice on a full pool."""
    p = Pool(mk, np.random.default_rng(2), 1, 2, 16, 1, 64, 2, 2)
    p.resize([0], [20])
    p.fork(None, [0, 0])
    print("full pool, equal", flush=True)
    assert p.resize([0, 1], [21, 21]) == [1, 1]
    p.fork(None, [1, 0])
    assert p.resize([1, 0], [21, 21]) == [1, 1]


def test_one_between(mk):
    """An entry that finds no page between two that share: whoever shares has a page, so the last may keep the old one; and one
    that grows past its page's end, after one of its own that does not fit."""
    p = Pool(mk, np.random.default_rng(3), 1, 4, 16, 1, 64, 4, 4)
    p.resize([0, 3], [20, 16])
    p.fork([1], [0])
    print("full pool, between", flush=True)
    assert p.resize([0, 3, 1], [21, 40, 22]) == [0, 1, 0]
    p.resize([0, 1, 3], [0, 0, 0])
    p.resize([0, 3], [20, 16])
    p.fork([1, 2], [0, 0])
    assert p.resize([0, 1, 2], [21, 21, 33]) == [0, 1, 1]
    assert p.resize([3, 2], [0, 0]) == [0, 0]
    assert p.resize([1], [33]) == [0]


@pytest.mark.parametrize("n_seq,n_page,page", [(6, 9, 16), (40, 70, 32), (1500, 2500, 16)])
def test_lives_on_a_small_pool(mk, n_seq, n_page, page):
    rng = np.random.default_rng(n_seq)
    p = Pool(mk, rng, 1, n_page, page, 1, 64, n_seq, 4)
    failed = 0
    for step in range(14):
        print("full pool, life", n_seq, step, flush=True)
        p.fork(None, [int(x) for x in np.where(rng.random(n_seq) < 0.5, np.arange(n_seq), rng.integers(-1, n_seq, n_seq))])
        seq = [int(x) for x in rng.permutation(n_seq)]
        new = [int(x) for x in np.clip(p.a["len"][seq] + rng.integers(-page // 2, page, n_seq), 0, 4 * page)]
        failed += p.resize(seq, new).count(1)
    assert failed


@pytest.mark.parametrize("d,layout,rope_dim,in_place", [(128, mk_.ROPE_HALVES, 128, True), (64, mk_.ROPE_PAIRS, 22, False)])
def test_writes_of_who_found_no_room(mk, d, layout, rope_dim, in_place):
    """Rows past a sequence's end, in a page that it shares and in one of its own: nothing is written, q stays as it was. The others
    of the batch are written, and without lengths all are."""
    rng = np.random.default_rng(d)
    H, KV, page, n_pos = 4, 2, 16, 40
    p = Pool(mk, rng, 2, 5, page, KV, d, 4, 3)
    p.resize([0, 2], [20, 35])
    p.fork([1], [0])
    p.resize([1], [18])
    assert p.resize([1, 0, 2], [19, 20, 36]) == [1, 0, 0]
    seq, row = [1, 2, 0, 1, 2], [18, 35, 19, 21, 36]
    cos, sin = (rng.standard_normal((n_pos, rope_dim // 2)).astype(np.float32) for _ in range(2))
    for lengths in (True, False):
        x = rng.standard_normal((len(seq), (H + 2 * KV) * d)).astype(np.float32)
        before = {k: p.c.get(k) for k in test_gpu_pages.DATA}
        length = p.c.c.len
        p.c.c.len = length if lengths else None
        print("full pool, writes", d, lengths, flush=True)
        q = write_call(mk, p.c, x, H, None, layout, rope_dim, cos, sin, [3, 1, 4, 1, 5], seq, row, 1, in_place)
        p.c.c.len = length
        live = [1, 2] if lengths else range(5)
        after = {k: p.c.get(k) for k in test_gpu_pages.DATA}
        for t in range(5):
            same = np.array_equal(q[t, :H * d], x[t, :H * d] if in_place else np.full(H * d, 3.0, np.float32))
            assert same == (t not in live)
        for t in live:
            pg, r = p.a["table"][seq[t], row[t] // page], row[t] % page
            num, s = in4(x[t, (H + KV) * d:].reshape(KV, d))
            assert np.array_equal(after["v"][pg, 1, :, r], packed(num))
            assert np.array_equal(after["v_scale"][pg, 1, :, :, r], s)
            assert not np.array_equal(after["k"][pg, 1, :, r], before["k"][pg, 1, :, r])
            for k in test_gpu_pages.DATA:
                at = (pg, 1, slice(None), slice(None), r) if k == "v_scale" else (pg, 1, slice(None), r)
                before[k][at] = after[k][at]
        for k in test_gpu_pages.DATA:
            assert np.array_equal(after[k].view(np.uint8), before[k].view(np.uint8)), k
