"""The beam search of the documentation on a pool that runs out, with beams that end: who finds no page writes nothing, the rows of
all others (a parked chat's among them, which shares the prompt's last page and goes on further there) stay as they were, and
the beams that go on follow their formulas. Eager and as one graph."""
import ctypes

import numpy as np
import pytest

import malkin_amd as mk_
from kv4_cases import Cache, attention64, beams64, copied, fork_model, in4, packed
from kv4_full_pool import resize_in_order
from test_gpu_beam import check as check_beams
from test_gpu_beam_step import BEAMS, D, DATA, E, GROUPS, KV, LAYERS, MOST, N, PAGE, PROMPTS, ROWS, H, Search, V, same
from test_gpu_kv4 import check as check_attention

pytestmark = pytest.mark.gpu

PARKED, STEPS = N, 5
FREE = 4  # pages beside those of the prompts


class Small(Search):
    def __init__(self, mk, synth, seed):
        super().__init__(mk, synth, seed)
        rng = np.random.default_rng(seed)
        n_page = sum(-(-p // PAGE) for p in PROMPTS) + FREE
        self.c = Cache(rng, LAYERS, n_page, PAGE, KV, D, N + 1, -(-MOST // PAGE)).put(mk)
        self.start = {x: v.copy() for x, v in self.c.a.items()}
        self.works[2] = mk.alloc(self.L.mk_kv4_resize_workspace(N, n_page))
        every = np.arange(V, dtype=np.int32)
        for name, v in (("every", every), ("is_eos", every * 0), ("done", every[:N] * 0), ("word", every[:N])):
            self.d[name] = mk.to_device(v)
            self.p[name] = self.d[name].ptr
        self.eos = 0

    def prompt(self):
        super().prompt()
        # The second group's prompt is a chat's that went on: it holds five rows more on the same last page.
        first, L = BEAMS, self.L
        for seq, rows in ((first, PROMPTS[1] + 5), (None, None), (first, PROMPTS[1])):
            if seq is None:
                up = [self.mk.to_device(np.array([x], np.int32)) for x in (PARKED, first)]
                mk_.check(L.mk_kv4_fork(self.mk.h, self.c.ref, up[0].ptr, up[1].ptr, 1, *self.work(1)))
                self.mk.sync()
            else:
                self.put(first=np.array([seq, seq], np.int32), plen=np.array([rows, rows], np.int32))
                mk_.check(L.mk_kv4_resize(self.mk.h, self.c.ref, self.p["first"], self.p["plen"], 1, self.p["status"], *self.work(2)))
        self.put(done=np.zeros(N, np.int32), word=np.zeros(N, np.int32))

    def step(self):
        L, p, c, h = self.L, self.p, mk_.check, self.mk.h
        c(L.mk_beam_select(h, p["logits"], V, GROUPS, BEAMS, V, p["scores"], p["done"], self.eos, BEAMS, p["best"], p["src"],
                           p["tokens"], *self.work(0)))
        c(L.mk_move_ids(h, p["scores"], None, p["best"], None, N))
        c(L.mk_move_ids(h, p["done"], None, p["is_eos"], p["tokens"], N))
        c(L.mk_move_ids(h, p["word"], None, p["every"], p["tokens"], N))
        c(L.mk_kv4_fork(h, self.c.ref, None, p["src"], N, *self.work(1)))
        c(L.mk_kv4_resize(h, self.c.ref, None, p["len"], N, p["status"], *self.work(2)))
        self.layers(p["word"], N, p["pos"], p["seq"], p["len"], 1)
        c(L.mk_matmul(h, ctypes.byref(self.head[1]), p["aq"], N, p["logits"], V, 0))

    def drop(self):
        """What the host does between two steps: beams without room take no further part."""
        status = self.get("status", N, dtype=np.int32)
        self.put(scores=np.where(status != 0, -np.inf, self.get("scores", N)).astype(np.float32))

    def ids(self, name):
        return self.get(name, N, dtype=np.int32)


def test_search_on_a_full_pool(mk, synth_lib):
    hip = ctypes.CDLL("libamdhip64.so")
    s = Small(mk, synth_lib, 11)
    print("full pool, prompts", flush=True)
    s.prompt()
    assert list(s.c.get("refs")[s.c.get("table")[PARKED][:10]]) == [2] * 10 and s.c.get("len")[PARKED] == 155
    # The first group's second best token ends its beam.
    s.eos = beams64(s.get("logits", N, V), s.get("scores", N), None, 0, BEAMS, BEAMS)[0][0][1][2]
    s.put(is_eos=(np.arange(V) == s.eos).astype(np.int32))
    states, lost, ended = [], 0, 0
    for i in range(STEPS):
        print("full pool, step", i, flush=True)
        logits, scores, done = s.get("logits", N, V), s.get("scores", N), s.ids("done")
        model = {x: v.copy() for x, v in zip(DATA, s.c.get(*DATA))}
        s.ready(i)
        s.step()
        states.append(s.state() + [s.ids("done"), s.ids("word"), s.get("scores", N)])
        best, src, tokens, status = s.get("best", GROUPS, BEAMS), s.ids("src"), s.ids("tokens"), s.ids("status")
        with np.errstate(invalid="ignore"):
            want = beams64(logits, scores, done, s.eos, BEAMS, BEAMS)[0]
        check_beams((best, src.reshape(GROUPS, -1), tokens.reshape(GROUPS, -1)), want)
        live = src >= 0
        assert np.array_equal(s.ids("done")[live], (tokens == s.eos)[live]) and np.array_equal(s.ids("word")[live], tokens[live])
        assert np.array_equal(s.get("scores", N), best.reshape(-1))
        fork_model(model, PAGE, None, src)
        rows = np.repeat(PROMPTS, BEAMS) + i
        st, moves = resize_in_order(model, PAGE, None, [int(x) + 1 for x in rows])
        copied(model, moves, PAGE)
        assert list(status) == st
        # Everything but the rows that beams with room wrote.
        now = dict(zip(DATA, s.c.get(*DATA)))
        for t in np.flatnonzero(status == 0):
            p, r = model["table"][t, rows[t] // PAGE], rows[t] % PAGE
            for x in ("k", "v", "k_scale"):
                model[x][p, :, :, r] = now[x][p, :, :, r]
            model["v_scale"][p, :, :, :, r] = now["v_scale"][p, :, :, :, r]
        for x in DATA:
            assert np.array_equal(now[x].view(np.uint8), model[x].view(np.uint8)), x
        # What was written, and the attention of beams that go on.
        s.c.a = now
        going = np.flatnonzero((status == 0) & live)
        for layer in range(LAYERS):
            qkv = s.get(f"qkv{layer}", N, ROWS)
            num, scale = in4(qkv[:, E + KV * D:].reshape(N, KV, D))
            for t in going:
                p, r = now["table"][t, rows[t] // PAGE], rows[t] % PAGE
                assert np.array_equal(now["v"][p, layer, :, r], packed(num[t]))
                assert np.array_equal(now["v_scale"][p, layer, :, :, r], scale[t])
            want = attention64(s.c, layer, qkv[:, :E], H, np.where(np.isin(np.arange(N), going), np.arange(N), -1), rows + 1)
            check_attention(s.get(f"att{layer}", N, E), want, rows=going)
        lost, ended = lost + int((status != 0).sum()), ended + int(done.sum())
        s.drop()
    assert lost and ended and len(going)

    stream = ctypes.c_void_p(s.L.mk_stream(mk.h))
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    mk.sync()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    s.step()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
    for again in range(2):
        s.prompt()
        for i in range(STEPS):
            print("full pool, replay", again, i, flush=True)
            s.ready(i)
            assert hip.hipGraphLaunch(run, stream) == 0
            same(s.state() + [s.ids("done"), s.ids("word"), s.get("scores", N)], states[i])
            s.drop()
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
