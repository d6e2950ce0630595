"""A speculative step of several users behind one shared prefix, each with an adapter of its own: q|k|v projection, adapters,
QK-norm + RoPE + KV write, attention over the prefix and the users' rows, LM head, verification of the drafts, whole
vocabulary and top-k. Every operator is checked against a 64-bit form on the values that it was given, and the whole chain
captured in one graph gives the eager run's bits. Two contexts at work at the same time, each call with a workspace of its
own, do not change each other's results."""
import ctypes

import numpy as np
import pytest

import malkin_amd as mk_
import test_gpu_attn_prefix as prefix
import test_gpu_lora as adapters
import test_gpu_verify as drafted
from operator_cases import EPS, attention64, cut64, lora64, make_cache, softmax64, verify64

pytestmark = pytest.mark.gpu

E, H, KV, D, V = 512, 8, 2, 128, 4096
P, CTX, ROWS = 333, 64, (H + 2 * KV) * D


def packed(mk, synth, rng, rows, cols):
    w = (0.05 * rng.standard_normal((rows, cols))).astype(np.float32)
    raw = mk.to_device(synth.quantize_rows(mk_.Q8_0, w))
    L = mk_.load()
    out = mk.alloc(L.mk_packed_bytes(mk_.Q8_0, rows, cols))
    mk_.check(L.mk_pack_weight(mk.h, mk_.Q8_0, raw.ptr, cols // 32 * 34, rows, cols, out.ptr))
    mk.sync()
    return out, mk_.MkWeight(mk_.Q8_0, 0, rows, cols, out.p)


def test_step(mk, synth_lib):
    hip, L, rng = ctypes.CDLL("libamdhip64.so"), mk_.load(), np.random.default_rng(3)
    counts, have, temps = [3, 0, 4, 1], [7, 0, 20, 31], [0.8, 1.0, 0.0, 1.2]  # drafts, rows so far, temperatures
    users, new = len(counts), [c + 1 for c in counts]
    n, n_draft = sum(new), sum(counts)
    seq = np.repeat(np.arange(users), new).astype(np.int32)
    own = np.concatenate([np.arange(m) + h for m, h in zip(new, have)]).astype(np.int32)
    keys = (P + own + 1).astype(np.int32)
    most = int(keys.max())

    wq_b, wq = packed(mk, synth_lib, rng, ROWS, E)
    head_b, head = packed(mk, synth_lib, rng, V, H * D)
    ranks, host = [8, 16, 4], []
    table, keep = np.zeros(3, mk_.LORA_ADAPTER), []
    for i, r in enumerate(ranks):
        a = (rng.standard_normal((r, E)) / 16).astype(np.float16)
        b = (0.2 * rng.standard_normal((ROWS, r))).astype(np.float16)
        da, db = mk.to_device(a), mk.to_device(b)
        keep += [da, db]
        table[i] = (da.p, db.p, 1.5, r)
        host.append((a.astype(np.float32), b.astype(np.float32), 1.5))
    ids = np.array([[0, -1, 2, 1][s] for s in seq], np.int32)

    kv = make_cache(rng, 1, users, KV, CTX, D)
    pre = make_cache(rng, 1, 2, KV, P, D)
    kv_b, pre_b = ([mk.to_device(x) for x in c] for c in (kv, pre))
    kvc = mk_.MkKvCache(*(b.p for b in kv_b), 1, users, KV, D, CTX)
    prec = mk_.MkKvCache(*(b.p for b in pre_b), 1, 2, KV, D, P)
    pos = np.arange(P + CTX)
    inv = 1e6 ** (-np.arange(D // 2) / (D // 2))
    cos, sin = (f(np.outer(pos, inv)).astype(np.float32) for f in (np.cos, np.sin))

    f32 = lambda *s: mk.alloc(4 * int(np.prod(s)))  # noqa: E731
    up = lambda x: mk.to_device(np.ascontiguousarray(x))  # noqa: E731
    x = rng.standard_normal((n, E)).astype(np.float32)
    d = dict(x=up(x), norm=up(1 + 0.1 * rng.standard_normal(E).astype(np.float32)), xn=f32(n, E),
             xq=mk.alloc(n * E // 32 * 40), base=f32(n, ROWS), qkv=f32(n, ROWS), qn=up(np.full(D, 1.5, np.float32)),
             kn=up(np.ones(D, np.float32)), cos=up(cos), sin=up(sin), rpos=up(keys - 1), seq=up(seq), row=up(own),
             keys=up(keys), ids=up(ids), table=up(table), att=f32(n, H * D), aq=mk.alloc(n * H * D // 32 * 40),
             logits=f32(n, V), tv=f32(n, 40), ti=f32(n, 40), u=up(rng.random(n_draft)), un=up(rng.random(users)))
    lanes = np.zeros(users, mk_.VERIFY_LANE)
    lanes["n_draft"], lanes["first"] = counts, np.cumsum(counts) - counts
    lanes["row"], lanes["temperature"] = np.cumsum(new) - new, temps
    lanes["min_p"], lanes["top_p"] = 0.02, 0.95
    d["lanes"] = up(lanes)
    drafts = rng.integers(0, V, n_draft).astype(np.int32)
    d["drafts"] = up(drafts)
    out = {k: [f32(users), f32(users, max(new)), f32(users, max(new))] for k in ("dense", "topk")}
    wa = mk.alloc(L.mk_attention_prefix_workspace(n, H, KV, D, P, most))
    wl = mk.alloc(L.mk_lora_workspace(n, 16, E))
    wv = mk.alloc(L.mk_verify_workspace(users, max(counts), V))
    p = {k: b.ptr for k, b in d.items()}
    at = d["qkv"].offset

    def step():
        c = mk_.check
        c(L.mk_rmsnorm(mk.h, p["x"], p["norm"], n, E, 1e-6, p["xn"]))
        c(L.mk_rmsnorm_q8(mk.h, p["x"], None, p["norm"], n, E, 1e-6, p["xq"]))
        c(L.mk_matmul(mk.h, ctypes.byref(wq), p["xq"], n, p["base"], ROWS, 0))
        c(L.mk_lora(mk.h, mk_.F16, p["table"], 3, 16, p["ids"], p["xn"], E, n, ROWS, E, p["base"], ROWS, p["qkv"], ROWS,
                    wl.ptr, wl.nbytes))
        c(L.mk_qk_norm_rope_kv(mk.h, p["qkv"], at(4 * H * D), at(4 * (H + KV) * D), ROWS, n, H, p["qn"], p["kn"], 1e-6,
                               p["cos"], p["sin"], p["rpos"], p["seq"], p["row"], ctypes.byref(kvc), 0))
        c(L.mk_attention_prefix(mk.h, p["qkv"], ROWS, p["att"], H * D, n, H, ctypes.byref(prec), 1, P,
                                ctypes.byref(kvc), 0, 0, p["seq"], p["keys"], most, p["aq"], wa.ptr, wa.nbytes))
        c(L.mk_matmul(mk.h, ctypes.byref(head), p["aq"], n, p["logits"], V, 0))
        c(L.mk_verify(mk.h, p["logits"], V, n, None, 0, n_draft, V, p["lanes"], users, max(counts), p["drafts"], p["u"],
                      p["un"], *(b.ptr for b in out["dense"]), wv.ptr, wv.nbytes))
        c(L.mk_topk(mk.h, p["logits"], V, None, n, V, 40, p["tv"], p["ti"]))
        c(L.mk_verify_topk(mk.h, p["tv"], p["ti"], 40, n, None, None, 0, n_draft, p["lanes"], users, max(counts),
                           p["drafts"], p["u"], p["un"], *(b.ptr for b in out["topk"])))

    def get(name, *shape, dtype=np.float32):
        return d[name].download(dtype).reshape(shape)

    def results():
        r = {k: get(k, n, -1) for k in ("base", "qkv", "att", "logits")}
        for k, bufs in out.items():
            r[k] = [b.download(t) for b, t in zip(bufs, (np.int32, np.int32, np.float32))]
        r["kv"] = [b.download(np.uint8) for b in kv_b]
        return r

    print("serving step, first run", flush=True)
    step()
    # Drafts that the target finds likely, so that some are accepted, in a second run.
    logits = get("logits", n, V)
    for i, l in enumerate(lanes):
        for j in range(l["n_draft"]):
            order = np.argsort(-logits[l["row"] + j])
            drafts[l["first"] + j] = order[0] if (i + j) % 3 else order[5]
    d["drafts"].upload(drafts)
    print("serving step, second run", flush=True)
    step()
    r = results()

    # Adapters: the q|k|v rows before the norm, from their value part (the norm and rotation leave v alone).
    want, tol = lora64(get("xn", n, E), host, ids, r["base"], ROWS)
    v0 = (H + KV) * D
    assert (np.abs(r["qkv"][:, v0:] - want[:, v0:]) <= tol[:, v0:]).all()
    # Attention, on the queries and the cache that the norm, rotation and KV write left.
    cache = [b.download(t).reshape(a.shape) for b, a, t in zip(kv_b, kv, (np.int8, np.int8, np.float32, np.float32))]
    want, tol = attention64(r["qkv"][:, :H * D], H, pre, 1, P, cache, 0, 0, seq, keys)
    assert (np.abs(r["att"] - want) <= tol).all()
    # Verification, on the logits; the cut's weights, their quotient and the result are each rounded to floats.
    order = np.arange(V)
    tv, ti = get("tv", n, 40), get("ti", n, 40, dtype=np.int32)
    u, un = d["u"].download(np.float64), d["un"].download(np.float64)
    accepted = 0
    for i, l in enumerate(lanes):
        dense = verify64(l, lambda j: (order, softmax64(r["logits"][l["row"] + j], l["temperature"])), None, drafts, u,
                         un[i], max(new))
        cut = verify64(l, lambda j: cut64(tv[l["row"] + j], ti[l["row"] + j], l, V), None, drafts, u, un[i], max(new))
        for name, w in (("dense", dense), ("topk", cut)):
            assert r[name][0][i] == w[0]
            assert list(r[name][1].reshape(users, -1)[i]) == w[1]
            assert np.allclose(r[name][2].reshape(users, -1)[i], w[2], rtol=4 * EPS, atol=1e-12)
        accepted += dense[0]
    assert accepted > 0

    # The chain in one graph: the same bits, again and again, with eager runs between.
    stream = ctypes.c_void_p(L.mk_stream(mk.h))
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    mk.sync()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    step()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
    for i in range(4):
        d["x"].upload(x if i % 2 else x[::-1])
        print("serving step, replay", i, flush=True)
        assert hip.hipGraphLaunch(run, stream) == 0
        a = results()
        step()
        b = results()
        for k in a:
            for y, z in zip(a[k], b[k]):
                assert np.array_equal(np.asarray(y).view(np.uint8), np.asarray(z).view(np.uint8)), k
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0


def test_two_contexts_at_once(mk):
    other, lib, jobs = mk_.Context(0), mk_.load(), []
    for i, m in enumerate((mk, other)):
        rng = np.random.default_rng(i)
        q, pre, kv, seq, keys = prefix.build(rng, 32, 8, 128, [1] * 8, 900, [60 + 9 * j for j in range(8)], 0)
        att = prefix.Call(m, q, 32, pre, 1, 900, kv, 0, 1, seq, keys, max(keys))
        ids, ranks = [0, 1, -1, 2] * 5, [16, 8, 32]
        x = rng.standard_normal((20, 512)).astype(np.float32)
        table = adapters.Set(m, rng, "f16", ranks, 1024, 512)
        _, lora, keep = adapters.call(m, "f16", table, 3, 32, ids, x, 1024, rng.standard_normal((20, 1024)).astype(np.float32))
        counts = [3, 1, 0, 2]
        lanes = drafted.lanes_of(counts, [0.7, 0.0, 1.0, 1.3])
        p, w, u, un = drafted.inputs(rng, counts, 20000)
        ver = drafted.Dense(m, p, w, lanes, drafted.sample_drafts(rng, w, lanes), u, un, 3)

        def run(att=att, lora=lora, ver=ver):
            att.run()
            mk_.check(lib.mk_lora(*lora))
            ver.run()

        def read(att=att, keep=keep, ver=ver, table=table):
            return [att.result(), keep[3].download(np.float32), *ver.read()]

        run()
        jobs.append((run, read, read()))
    print("two contexts", flush=True)
    for _ in range(50):
        for run, _, _ in jobs:
            run()
    for _, read, alone in jobs:
        for a, b in zip(alone, read()):
            assert np.array_equal(a, b)
    del jobs, att, keep, ver, table, run, read
    other.close()
