"""Forking, resizing and compacting the 4-bit cache's pages against a model that takes one entry after the other."""
import ctypes

import numpy as np
import pytest

import malkin_amd as mk_
from kv4_cases import Cache, compact_model, copied, fork_model, resize_model

pytestmark = pytest.mark.gpu
META = ("table", "len", "refs")
DATA = ("k", "v", "k_scale", "v_scale")


class Pool:
    """A cache on the device and the model's arrays beside it."""

    def __init__(self, mk, rng, n_layer, n_page, page, kv, d, n_seq, max_pages):
        self.mk, self.page = mk, page
        self.c = Cache(rng, n_layer, n_page, page, kv, d, n_seq, max_pages)
        self.n_seq, self.n_page, self.max_pages = n_seq, n_page, max_pages
        self.c.put(mk)
        self.a = self.c.a
        self.keep = []

    def up(self, v):
        if v is None:
            return None
        self.keep.append(self.mk.to_device(np.asarray(v, np.int32)))
        return self.keep[-1].ptr

    def work(self, need):
        self.keep.append(self.mk.to_device(np.full(need + 64, 0xA5, np.uint8)))
        return self.keep[-1], need

    def check(self, data=True):
        for x in META + (DATA if data else ()):
            got = self.c.get(x)
            assert np.array_equal(got.view(np.uint8), self.a[x].view(np.uint8)), x
        counts = np.bincount(self.a["table"][self.a["table"] >= 0], minlength=self.n_page)
        assert np.array_equal(counts, self.a["refs"])  # the model's own

    def fork(self, dst, src, data=True):
        L, (w, need) = mk_.load(), self.work(mk_.load().mk_kv4_fork_workspace(len(src), self.max_pages))
        mk_.check(L.mk_kv4_fork(self.mk.h, self.c.ref, self.up(dst), self.up(src), len(src), w.ptr, need))
        fork_model(self.a, self.page, dst, src)
        self.check(data)
        assert (w.download(np.uint8)[need:] == 0xA5).all()

    def resize(self, seq, new_len):
        n = len(new_len)
        L, (w, need) = mk_.load(), self.work(mk_.load().mk_kv4_resize_workspace(n, self.n_page))
        status = self.mk.to_device(np.full(n + 1, 77, np.int32))
        mk_.check(L.mk_kv4_resize(self.mk.h, self.c.ref, self.up(seq), self.up(new_len), n, status.ptr, w.ptr, need))
        want, moves = resize_model(self.a, self.page, seq, [int(x) for x in new_len])
        copied(self.a, moves, self.page)
        assert list(status.download(np.int32)) == want + [77]
        self.check()
        assert (w.download(np.uint8)[need:] == 0xA5).all()
        return want, moves

    def compact(self):
        L, (w, need) = mk_.load(), self.work(mk_.load().mk_kv4_compact_workspace(self.n_page))
        live = self.mk.to_device(np.zeros(1, np.int32))
        mk_.check(L.mk_kv4_compact(self.mk.h, self.c.ref, live.ptr, w.ptr, need))
        n, moves = compact_model(self.a)
        copied(self.a, moves, self.page)
        assert live.download(np.int32)[0] == n
        self.check()
        assert (w.download(np.uint8)[need:] == 0xA5).all()
        return moves


@pytest.mark.parametrize("d,page,kv,n_layer", [(128, 16, 2, 3), (64, 32, 3, 1), (128, 128, 1, 2)])
def test_life_of_a_pool(mk, d, page, kv, n_layer):
    """Prompts, beams that go on from each other, drafts taken back, users who leave, a pool that runs out, compaction."""
    rng = np.random.default_rng(d + page)
    p = Pool(mk, rng, n_layer, 60, page, kv, d, 12, 9)
    print("pages: prompts", flush=True)
    p.resize([3, 0, 7], [2 * page + 5, page, 1])
    print("pages: beams", flush=True)
    p.fork([1, 2, 4, 5], [0, 0, 3, 3])
    _, moves = p.resize([0, 1, 2, 3, 4, 5], [page + 1] * 3 + [2 * page + 6] * 3)
    assert len(moves) == 2  # of three holders of the page that is not full the last keeps it
    p.fork(None, [1, 0, 0, 4, 3, 4, 7, -1, 99, 2, 3, 11])  # all at once; 7 and 8 let go
    _, moves = p.resize([5, 3, 10], [2 * page + 7, 2 * page + 9, 3 * page])
    assert moves
    print("pages: shorter ends", flush=True)
    p.resize([0, 10, 9, 6], [page, 5, 0, 0])
    for step in range(12):
        src = [int(x) for x in rng.integers(-1, 13, 12)]
        p.fork(None, src)
        new = [int(x) for x in np.clip(p.a["len"] + rng.integers(-page, 2 * page, 12), 0, 9 * page)]
        p.resize([int(x) for x in rng.permutation(12)], new)
        if step % 4 == 3:
            p.compact()
            p.compact()  # nothing left to move


def test_entries_without_effect(mk):
    """Places outside, the same sequence twice, ends outside: left out; the others as if they were alone."""
    rng = np.random.default_rng(4)
    p = Pool(mk, rng, 1, 40, 16, 1, 64, 6, 8)
    p.resize(None, [20, 40, 0, 3, 128, 16])
    st, _ = p.resize([0, 9, 1, 0, -1, 2, 3], [50, 5, 129, 17, 5, -1, 60])
    assert st == [-1, -1, -1, 0, -1, -1, 0]
    p.fork([0, 7, 1, 0, -1, 2], [4, 1, 5, 3, 2, 2])
    p.fork([5], [5])
    p.fork([3, 4], [4, 3])  # swapped
    st, _ = p.resize(None, [1] * 9)  # more entries than sequences
    assert st == [0] * 6 + [-1] * 3


def test_pool_runs_out(mk):
    rng = np.random.default_rng(5)
    p = Pool(mk, rng, 2, 10, 16, 1, 64, 8, 12)
    p.resize([0, 1], [33, 40])  # 3 + 3 of 10
    p.fork([2, 3], [0, 0])
    # 2 wants a copy and a page (2 of 4 free), 4 three pages (not there), 5 none of its own, 3 a copy that no longer fits in order.
    st, moves = p.resize([2, 4, 5, 3, 6], [49, 40, 0, 34, 16])
    assert st == [0, 1, 0, 1, 1] and len(moves) == 1
    st, _ = p.resize([1, 4], [0, 40])  # what is let go serves the same call
    assert st == [0, 0]
    st, _ = p.resize([5], [192])
    assert st == [1]
    p.compact()


@pytest.mark.parametrize("n_page,n_seq,max_pages", [(70000, 500, 40), (20000, 3, 15000)])
def test_large_pools(mk, n_page, n_seq, max_pages):
    """More pages than one step of the walk over the pool, long tables, hundreds of entries."""
    rng = np.random.default_rng(6)
    p = Pool(mk, rng, 1, n_page, 16, 1, 64, n_seq, max_pages)
    most = 16 * max_pages
    first = [int(x) for x in rng.integers(0, min(most, 16 * n_page // n_seq), n_seq)]
    print("pages: large pool", n_page, n_seq, flush=True)
    p.resize(None, first)
    p.fork(None, [int(x) for x in rng.integers(-1, n_seq, n_seq)])
    p.resize(None, [int(x) for x in np.clip(p.a["len"] + rng.integers(-30, 40, n_seq), 0, most)])
    p.fork(None, [int(x) if rng.random() < 0.7 else -1 for x in range(n_seq)])
    moves = p.compact()
    assert moves


def test_many_entries_on_one_page(mk):
    """As many beams of one page as a resize takes."""
    rng = np.random.default_rng(7)
    p = Pool(mk, rng, 1, 5000, 16, 1, 64, 4096, 2)
    p.resize([17], [9])
    p.fork(None, [17] * 4096)
    print("pages: 4096 beams", flush=True)
    st, moves = p.resize(None, [10] * 4096)
    assert st == [0] * 4096 and len(moves) == 4095
    p.compact()


def test_captured(mk):
    """Fork, resize and compact in one graph, replayed from the same state, with eager runs between."""
    hip = ctypes.CDLL("libamdhip64.so")
    rng, L = np.random.default_rng(8), mk_.load()
    p = Pool(mk, rng, 2, 64, 16, 2, 128, 8, 8)
    p.resize([0, 4], [100, 37])
    p.fork(None, [0, 0, 0, 0, 4, 4, 4, 4])
    start = {x: p.c.get(x) for x in META + DATA}
    src, new, status, live = (mk.to_device(np.zeros(8, np.int32)) for _ in range(4))
    ws = [mk.alloc(n) for n in (L.mk_kv4_fork_workspace(8, 8), L.mk_kv4_resize_workspace(8, 64), L.mk_kv4_compact_workspace(64))]

    def step():
        mk_.check(L.mk_kv4_fork(mk.h, p.c.ref, None, src.ptr, 8, ws[0].ptr, ws[0].nbytes))
        mk_.check(L.mk_kv4_resize(mk.h, p.c.ref, None, new.ptr, 8, status.ptr, ws[1].ptr, ws[1].nbytes))
        mk_.check(L.mk_kv4_compact(mk.h, p.c.ref, live.ptr, ws[2].ptr, ws[2].nbytes))

    def reset():
        for x, v in start.items():
            p.c.b[x].upload(v)

    step()
    mk.sync()
    stream, graph, run = ctypes.c_void_p(L.mk_stream(mk.h)), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    step()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
    for i in range(4):
        parents = [int(x) for x in rng.integers(0, 4, 4)] + [4 + int(x) for x in rng.integers(0, 4, 4)]
        ends = [101 + i, 101, 101, 90, 38, 38, 60, 0]
        src.upload(np.asarray(parents, np.int32))
        new.upload(np.asarray(ends, np.int32))
        a = {x: v.copy() for x, v in start.items()}
        fork_model(a, 16, None, parents)
        _, moves = resize_model(a, 16, None, ends)
        copied(a, moves, 16)
        _, moves = compact_model(a)
        copied(a, moves, 16)
        for go in (lambda: hip.hipGraphLaunch(run, stream), lambda: step() or 0):
            reset()
            print("pages: replay", i, flush=True)
            assert go() == 0
            for x in META + DATA:
                assert np.array_equal(p.c.get(x).view(np.uint8), a[x].view(np.uint8)), x
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
