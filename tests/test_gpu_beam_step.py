"""Beam search over the 4-bit cache as a server runs it: prompts into pages, then per token the selection, the fork of the beams'
pages, room for a row more, two layers of q|k|v projection, rotation with the write of keys and values, attention, and the LM head.
Every operator is checked against a 64-bit form on the values that it was given, one graph of the step gives the eager search's
bits, and two contexts at work at the same time do not change each other's results."""
import ctypes

import numpy as np
import pytest

import malkin_amd as mk_
from kv4_cases import Cache, attention64, beams64, copied, fork_model, in4, packed, resize_model, rotated64, unpacked
from test_gpu_beam import check as check_beams
from test_gpu_kv4 import check as check_attention
from test_gpu_serving_step import packed as weight

pytestmark = pytest.mark.gpu

H, KV, D, V, LAYERS, PAGE = 8, 2, 64, 4096, 2, 16
E, ROWS, HALF = H * D, (H + 2 * KV) * D, D // 2
BEAMS, PROMPTS, STEPS = 4, [37, 150], 7
GROUPS = len(PROMPTS)
N = GROUPS * BEAMS
MOST = max(PROMPTS) + STEPS + 1
DATA = ("k", "v", "k_scale", "v_scale", "table", "len", "refs")


class Search:
    def __init__(self, mk, synth, seed):
        rng = np.random.default_rng(seed)
        self.mk, self.L = mk, mk_.load()
        up = lambda x: mk.to_device(np.ascontiguousarray(x))  # noqa: E731
        # Room for the prompts and for a page or two of each beam's own.
        self.c = Cache(rng, LAYERS, sum(-(-p // PAGE) for p in PROMPTS) + 2 * N + 1, PAGE, KV, D, N, -(-MOST // PAGE)).put(mk)
        self.start = {x: v.copy() for x, v in self.c.a.items()}
        self.wq = [weight(mk, synth, rng, ROWS, E) for _ in range(LAYERS)]
        self.head = weight(mk, synth, rng, V, E)
        rope = mk_.MkRope(D, mk_.ROPE_NTK, 1e4, 2.0, 0, 0.0, 0.0, 0.0)
        self.words = [rng.integers(0, V, p).astype(np.int32) for p in PROMPTS]
        big = sum(PROMPTS)
        f32 = lambda *s: mk.alloc(4 * int(np.prod(s)))  # noqa: E731
        self.d = dict(embed=up(rng.standard_normal((V, E)).astype(np.float32)), norm=up(1 + 0.1 * rng.standard_normal(E).astype(np.float32)),
                      cos=f32(MOST, HALF), sin=f32(MOST, HALF), xq=mk.alloc(big * E // 32 * 40), aq=mk.alloc(big * E // 32 * 40),
                      logits=f32(N, V), scores=f32(N), best=f32(N), src=f32(N), tokens=f32(N), status=f32(N), len=f32(N), pos=f32(N),
                      seq=f32(N), ptok=f32(big), pseq=f32(big), ppos=f32(big), pkeys=f32(big), first=f32(GROUPS), plen=f32(GROUPS))
        for i in range(LAYERS):
            self.d[f"qkv{i}"], self.d[f"att{i}"] = f32(big, ROWS), f32(big, E)
        self.p = {k: b.ptr for k, b in self.d.items()}
        L = self.L
        self.works = [mk.alloc(x) for x in (L.mk_beam_workspace(GROUPS, BEAMS, V, BEAMS), L.mk_kv4_fork_workspace(N, -(-MOST // PAGE)),
                                            L.mk_kv4_resize_workspace(N, self.c.shape[1]),
                                            L.mk_attention_kv4_workspace(big, H, KV, D, MOST, max(PROMPTS)))]
        mk_.check(L.mk_rope_tables(mk.h, ctypes.byref(rope), None, 0, MOST, self.p["cos"], self.p["sin"]))

    def work(self, i):
        return self.works[i].ptr, self.works[i].nbytes

    def put(self, **arrays):
        for k, v in arrays.items():
            self.d[k].upload(np.asarray(v))

    def layers(self, tok, n, pos, seq, keys, run):
        """Rows `tok` of the embedding through both layers; the last one's outputs are left in aq."""
        L, p, c = self.L, self.p, mk_.check
        c(L.mk_rmsnorm_q8(self.mk.h, p["embed"], tok, p["norm"], n, E, 1e-6, p["xq"]))
        for i in range(LAYERS):
            at = self.d[f"qkv{i}"].offset
            c(L.mk_matmul(self.mk.h, ctypes.byref(self.wq[i][1]), p["aq" if i else "xq"], n, at(0), ROWS, 0))
            c(L.mk_rope_kv4(self.mk.h, at(0), at(4 * E), at(4 * (E + KV * D)), ROWS, n, H, None, None, 1e-6,
                            mk_.ROPE_PAIRS, D, p["cos"], p["sin"], MOST, pos, seq, pos, self.c.ref, i, at(0), ROWS))
            c(L.mk_attention_kv4(self.mk.h, at(0), ROWS, p[f"att{i}"], E, n, H, self.c.ref, i, seq, keys, MOST, run, p["aq"],
                                 *self.work(3)))

    def forward(self):
        """The beams' newest tokens, one each, and the logits after them."""
        self.layers(self.p["tokens"], N, self.p["pos"], self.p["seq"], self.p["len"], 1)
        mk_.check(self.L.mk_matmul(self.mk.h, ctypes.byref(self.head[1]), self.p["aq"], N, self.p["logits"], V, 0))

    def step(self):
        L, p, c = self.L, self.p, mk_.check
        c(L.mk_beam_select(self.mk.h, p["logits"], V, GROUPS, BEAMS, V, p["scores"], None, 0, BEAMS, p["best"], p["src"],
                           p["tokens"], *self.work(0)))
        c(L.mk_move_ids(self.mk.h, p["scores"], None, p["best"], None, N))
        c(L.mk_kv4_fork(self.mk.h, self.c.ref, None, p["src"], N, *self.work(1)))
        c(L.mk_kv4_resize(self.mk.h, self.c.ref, None, p["len"], N, p["status"], *self.work(2)))
        self.forward()

    def prompt(self):
        """All but the last word of each prompt into its group's first beam, then that word; the other beams are not there yet."""
        for x in DATA:
            self.c.b[x].upload(self.start[x])
        firsts, n = np.arange(GROUPS) * BEAMS, sum(PROMPTS) - GROUPS
        self.put(first=firsts.astype(np.int32), plen=np.array(PROMPTS, np.int32))
        mk_.check(self.L.mk_kv4_resize(self.mk.h, self.c.ref, self.p["first"], self.p["plen"], GROUPS, self.p["status"], *self.work(2)))
        pos = np.concatenate([np.arange(m - 1) for m in PROMPTS]).astype(np.int32)
        self.put(ptok=np.concatenate([w[:-1] for w in self.words]), ppos=pos, pkeys=pos + 1,
                 pseq=np.repeat(firsts, [m - 1 for m in PROMPTS]).astype(np.int32))
        self.layers(self.p["ptok"], n, self.p["ppos"], self.p["pseq"], self.p["pkeys"], max(PROMPTS) - 1)
        seq, tokens, scores = np.full(N, -1, np.int32), np.zeros(N, np.int32), np.full(N, -np.inf, np.float32)
        seq[firsts], tokens[firsts], scores[firsts] = firsts, [w[-1] for w in self.words], 0
        rows = np.repeat(PROMPTS, BEAMS).astype(np.int32)
        self.put(tokens=tokens, pos=rows - 1, len=rows, seq=seq, scores=scores)
        self.forward()
        self.put(seq=np.arange(N, dtype=np.int32))

    def ready(self, i):
        rows = np.repeat(PROMPTS, BEAMS).astype(np.int32) + i
        self.put(pos=rows, len=rows + 1)

    def get(self, name, *shape, dtype=np.float32):
        return self.d[name].download(dtype)[:int(np.prod(shape))].reshape(shape)

    def state(self):
        """Everything a step leaves."""
        ids = [self.get(x, N, dtype=np.int32) for x in ("src", "tokens", "status")]
        return [self.get("logits", N, V), self.get("best", N), *ids, *self.c.get(*DATA)]


def check_layers(s, seq, pos, n):
    """q, the rows of V and the attention of the forward that has just run, on what the device's arrays hold."""
    cos, sin = (s.get(x, MOST, HALF).astype(np.float64) for x in ("cos", "sin"))
    a = dict(zip(DATA, s.c.get(*DATA)))
    s.c.a = a
    live = np.flatnonzero(seq >= 0)
    for i in range(LAYERS):
        qkv = s.get(f"qkv{i}", n, ROWS)
        v = qkv[:, E + KV * D:].reshape(n, KV, D)
        num, scale = in4(v)
        for t in live:
            p, r = a["table"][seq[t], pos[t] // PAGE], pos[t] % PAGE
            assert np.array_equal(a["v"][p, i, :, r], packed(num[t]))
            assert np.array_equal(a["v_scale"][p, i, :, :, r], scale[t])
            # k as it was before the rotation: a number is off by half a step, and the range ends at 7 steps on one side
            k = rotated64(qkv[t, E:E + KV * D].reshape(KV, D).astype(np.float64), cos[pos[t]], sin[pos[t]], True)
            ks = a["k_scale"][p, i, :, r].astype(np.float64)
            got = (unpacked(a["k"][p, i, :, r]).astype(np.float64) - 8) * np.repeat(ks, 32, -1)
            assert (np.abs(got - k) <= np.repeat(np.abs(ks), 32, -1) * 1.07).all()
        want = attention64(s.c, i, qkv[:, :E], H, seq, np.where(seq >= 0, pos + 1, 0))
        check_attention(s.get(f"att{i}", n, E), want)


def same(a, b):
    for x, y in zip(a, b):
        assert np.array_equal(x.view(np.uint8), y.view(np.uint8))


def test_search(mk, synth_lib):
    hip = ctypes.CDLL("libamdhip64.so")
    s = Search(mk, synth_lib, 5)
    print("beam search, prompts", flush=True)
    s.prompt()
    seq = np.where(np.arange(N) % BEAMS == 0, np.arange(N), -1)
    check_layers(s, seq, np.repeat(PROMPTS, BEAMS) - 1, N)
    states = []
    for i in range(STEPS):
        print("beam search, step", i, flush=True)
        logits, scores = s.get("logits", N, V), s.get("scores", N)
        model = {x: v.copy() for x, v in zip(DATA, s.c.get(*DATA))}
        s.ready(i)
        s.step()
        states.append(s.state())
        best, src, tokens, status = s.get("best", GROUPS, BEAMS), *(s.get(x, N, dtype=np.int32) for x in ("src", "tokens", "status"))
        check_beams((best, src.reshape(GROUPS, -1), tokens.reshape(GROUPS, -1)), beams64(logits, scores, None, 0, BEAMS, BEAMS)[0])
        fork_model(model, PAGE, None, src)
        want, moves = resize_model(model, PAGE, None, [int(x) for x in np.repeat(PROMPTS, BEAMS) + i + 1])
        assert list(status) == want == [0] * N
        for x in ("table", "len", "refs"):
            assert np.array_equal(s.c.get(x), model[x]), x
        # Rows that the beams held before are those that they go on from.
        copied(model, moves, PAGE)
        now = s.c.get("k")
        for t in range(N):
            for r in range(0, int(np.repeat(PROMPTS, BEAMS)[t]) + i, 13):
                p = model["table"][t, r // PAGE]
                assert np.array_equal(now[p, :, :, r % PAGE], model["k"][p, :, :, r % PAGE])
        check_layers(s, np.arange(N), np.repeat(PROMPTS, BEAMS) + i, N)
    assert len({tuple(x) for x in states[-1][3].reshape(GROUPS, BEAMS)}) == GROUPS

    # The step in one graph: the search again, with the program's own work between replays, and a second time.
    s.prompt()
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
            print("beam search, replay", again, i, flush=True)
            s.ready(i)
            assert hip.hipGraphLaunch(run, stream) == 0
            same(s.state(), states[i])
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0


def test_two_contexts_at_once(mk, synth_lib):
    other = mk_.Context(0)
    jobs = [Search(m, synth_lib, seed) for seed, m in enumerate((mk, other))]
    alone = []
    for s in jobs:
        s.prompt()
        mine = []
        for i in range(STEPS):
            s.ready(i)
            s.step()
            mine.append(s.state())
        alone.append(mine)
    print("two contexts", flush=True)
    for s in jobs:
        s.prompt()
    for i in range(STEPS):
        for s in jobs:
            s.ready(i)
        for s in jobs:
            s.step()
        for s, mine in zip(jobs, alone):
            same(s.state(), mine[i])
    del jobs, s
    other.close()
