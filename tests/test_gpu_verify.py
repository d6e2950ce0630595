"""mk_verify and mk_verify_topk against a plain 64-bit walk: counts, tokens and probabilities for lanes of different
lengths, temperatures and proposers, vocabularies that no segment divides, masked, NaN and infinite logits, random numbers
at both ends, lanes that do not fit, the distribution of the drawn tokens, agreement with the host's mk_sampler_verify,
captured graphs."""
import ctypes

import numpy as np
import pytest

import malkin_amd as mk_
from operator_cases import EPS, cut64, cut_any64, softmax64, verify64

pytestmark = pytest.mark.gpu


def lanes_of(counts, temps, min_p=0.0, top_p=1.0):
    l = np.zeros(len(counts), mk_.VERIFY_LANE)
    c = np.asarray(counts)
    l["n_draft"], l["first"], l["row"] = c, np.cumsum(c) - c, np.cumsum(c + 1) - c - 1
    l["temperature"], l["min_p"], l["top_p"] = temps, min_p, top_p
    return l


class Dense:
    """One mk_verify call's buffers; run() and read()."""

    def __init__(self, mk, p, q, lanes, drafts, u, un, most, pads=(0, 0), probs=True):
        self.mk, self.n, self.most = mk, len(lanes), most
        V = p.shape[1]

        def wide(x, pad):
            w = np.full((max(1, len(x)), V + pad), 1e30, np.float32)
            w[:len(x), :V] = x
            return mk.to_device(w)

        self.p = wide(p, pads[0])
        self.q = wide(q, pads[1]) if q is not None else None
        self.lanes, self.d = mk.to_device(lanes), mk.to_device(np.asarray(list(drafts) + [0], np.int32))
        self.u, self.un = (mk.to_device(np.asarray(list(x) + [0.0], np.float64)) for x in (u, un))
        self.acc, self.tok = mk.to_device(np.full(self.n, 77, np.int32)), mk.to_device(
            np.full((self.n, most + 1), 77, np.int32))
        self.pr = mk.to_device(np.full((self.n, most + 1), 77, np.float32))
        need = mk_.load().mk_verify_workspace(self.n, most, V)
        self.need, self.work = need, mk.to_device(np.full(need + 64, 0xFF, np.uint8))
        self.args = (mk.h, self.p.ptr, V + pads[0], len(p), self.q.ptr if self.q else None, V + pads[1], len(drafts), V,
                     self.lanes.ptr, self.n, most, self.d.ptr, self.u.ptr, self.un.ptr, self.acc.ptr, self.tok.ptr,
                     self.pr.ptr if probs else None, self.work.ptr, need)

    def run(self):
        mk_.check(mk_.load().mk_verify(*self.args))
        return self

    def read(self):
        out = [b.download(t).reshape(s) for b, t, s in ((self.acc, np.int32, (self.n,)),
                                                       (self.tok, np.int32, (self.n, self.most + 1)),
                                                       (self.pr, np.float32, (self.n, self.most + 1)))]
        assert (self.work.download(np.uint8)[self.need:] == 0xFF).all()
        return out


def want_dense(p, q, lanes, drafts, u, un, most):
    order = np.arange(p.shape[1])
    out = []
    for i, l in enumerate(lanes):
        t = l["temperature"]
        out.append(verify64(l, lambda j: (order, softmax64(p[l["row"] + j], t)),
                            (lambda j: (order, softmax64(q[l["first"] + j], t))) if q is not None else None, drafts, u,
                            un[i], most + 1))
    return [np.array([o[k] for o in out]) for k in range(3)]


def check(got, want, rel=EPS):
    """Counts and tokens equal; a probability is rounded once (rel), after sums in 64 bits."""
    for a, b in zip(got[:2], want[:2]):
        assert np.array_equal(a, b), (np.argwhere(a != b)[:5], a[a != b][:5], b[a != b][:5])
    assert (np.abs(got[2] - want[2]) <= rel * want[2] + 1e-12).all()


def inputs(rng, counts, V, sharp=1.5, noise=0.5):
    n = int(sum(counts))
    p = (sharp * rng.standard_normal((n + len(counts), V))).astype(np.float32)
    hot = rng.integers(0, V, (len(p), 4))
    p[np.arange(len(p))[:, None], hot] += (8 + rng.standard_normal(hot.shape)).astype(np.float32)
    at = np.concatenate([np.arange(c) + o for c, o in zip(counts, np.cumsum(np.asarray(counts) + 1) -
                                                          np.asarray(counts) - 1)]).astype(int) if n else []
    q = (p[at] + noise * rng.standard_normal((n, V))).astype(np.float32)
    return p, q, rng.random(n), rng.random(len(counts))


def sample_drafts(rng, q, lanes):
    d = np.zeros(len(q), np.int32)
    for l in lanes:
        for j in range(l["first"], l["first"] + l["n_draft"]):
            d[j] = rng.choice(q.shape[1], p=softmax64(q[j], l["temperature"]))
    return d


CASES = [  # drafts per lane, vocabulary
    ([0], 1), ([1], 2), ([3], 17), ([2, 0, 5], 1000), ([4, 4, 1], 4096), ([1, 6], 4097), ([3, 8, 2, 1, 0, 7], 8191),
    ([2, 2], 151936), ([33], 5000), ([1] * 50, 300), ([1, 0, 2, 3] * 8, 35001), ([2, 1] * 16, 32768),
]


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("counts,V", CASES, ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)}x{max(v)}")
def test_dense_against_plain(mk, counts, V, certain):
    rng = np.random.default_rng(V + len(counts))
    lanes = lanes_of(counts, [[0.7, 0.0, 1.0, 1.3, 0.05][i % 5] for i in range(len(counts))])
    p, q, u, un = inputs(rng, counts, V)
    drafts = sample_drafts(rng, q, lanes)
    most = max(counts) + (2 if V == 1000 else 0)
    for pads in ((0, 0), (3, 1)):
        print("verify", counts, V, certain, pads, flush=True)
        c = Dense(mk, p, None if certain else q, lanes, drafts, u, un, most, pads)
        got = c.run().read()
        check(got, want_dense(p, None if certain else q, lanes, drafts, u, un, most))
        again = c.run().read()
        assert all(np.array_equal(a, b) for a, b in zip(got, again))
    c = Dense(mk, p, None if certain else q, lanes, drafts, u, un, most, probs=False).run().read()
    assert np.array_equal(c[0], got[0]) and np.array_equal(c[1], got[1]) and (c[2] == 77).all()


def test_dense_ends_and_masks(mk):
    """u of 0 and just below 1, logits of -inf, NaN, +inf and ties, rows of nothing, drafts that no row gives or that lie
    outside the vocabulary, equal distributions (nothing left over them)."""
    V, top = 5000, np.nextafter(1.0, 0.0)
    rng = np.random.default_rng(1)
    counts = [2] * 12
    lanes = lanes_of(counts, [1.0, 1.0, 0.0, 0.9, 1.0, 1.0, 0.0, 1.0, 1.0, 0.5, 1.0, 1.0])
    p, q, u, un = inputs(rng, counts, V)
    drafts = sample_drafts(rng, q, lanes)
    row, first = lanes["row"], lanes["first"]
    un[0], un[1] = 0.0, top
    u[first[0]], u[first[1]] = 0.0, top
    p[row[2]:row[2] + 3] = np.round(p[row[2]:row[2] + 3] / 4)       # ties: the first maximum
    p[row[3], rng.random(V) < 0.5] = -np.inf
    p[row[3], ::7], q[first[3], ::5] = np.nan, np.nan
    p[row[4]] = -np.inf                                             # refused, and no token
    p[row[5], [4, 900]] = np.inf                                    # the two share everything
    p[row[6]] = np.nan
    drafts[first[7]], drafts[first[8] + 1] = V, -1                  # outside the vocabulary
    u[first[8]] = 0.0
    q[first[9], drafts[first[9]]] = -np.inf                         # the draft model's own row excludes its draft
    q[first[10]] = p[row[10]]
    u[first[10]] = 0.5                                              # accepted: equal probabilities
    # Equal rows, a draft that neither gives: refused, and nothing is left over Q, so P itself.
    q[first[11]] = p[row[11]]
    p[row[11], 3] = q[first[11], 3] = -np.inf
    drafts[first[11]] = 3
    un[2:] = rng.random(10)
    print("verify, ends and masks", flush=True)
    got = Dense(mk, p, q, lanes, drafts, u, un, 2).run().read()
    want = want_dense(p, q, lanes, drafts, u, un, 2)
    check(got, want)
    assert got[0][4] == 0 and (got[1][4] == -1).all() and (got[1][6] == -1).all()
    assert got[0][7] == 0 and got[0][8] <= 1 and got[0][9] == 0 and got[0][10] >= 1 and got[0][11] == 0
    got = Dense(mk, p, None, lanes, drafts, u, un, 2).run().read()
    check(got, want_dense(p, None, lanes, drafts, u, un, 2))


def test_extreme_temperatures(mk):
    """From the smallest positive number, which is greedy but for ties, to infinity, which is uniform."""
    V, rng = 9000, np.random.default_rng(4)
    temps = [1e-45, 1e-30, 1e-3, 1e4, 3.4e38, np.inf]
    counts = [2] * len(temps)
    lanes = lanes_of(counts, temps)
    p, q, u, un = inputs(rng, counts, V)
    p[lanes["row"][0], [7, 70]] = p.max() + 1  # ties share
    drafts = sample_drafts(rng, q, lanes)
    print("verify, extreme temperatures", flush=True)
    for qq in (q, None):
        check(Dense(mk, p, qq, lanes, drafts, u, un, 2).run().read(), want_dense(p, qq, lanes, drafts, u, un, 2))


def test_lanes_that_do_not_fit(mk):
    rng = np.random.default_rng(2)
    counts, V = [2, 1, 3, 2], 600
    lanes = lanes_of(counts, 1.0)
    p, q, u, un = inputs(rng, counts, V)
    drafts = sample_drafts(rng, q, lanes)
    bad = np.concatenate([lanes, lanes[[0, 1, 2, 3, 0, 1]], lanes[:1]])
    bad["n_draft"][4], bad["row"][5], bad["first"][6] = 4, len(p) - 1, 6
    bad["row"][7], bad["first"][8], bad["n_draft"][9] = -1, -1, -1
    un = np.concatenate([un, rng.random(6), un[:1]])
    print("verify, lanes out of range", flush=True)
    got = Dense(mk, p, q, bad, drafts, u, un, 3).run().read()
    ok = [0, 1, 2, 3, 10]  # and lane 0 twice
    check([g[ok] for g in got], want_dense(p, q, bad[ok], drafts, u, un[ok], 3))
    no = [4, 5, 6, 7, 8, 9]
    assert (got[0][no] == -1).all() and (got[1][no] == -1).all() and (got[2][no] == 0).all()
    k = 20
    top = [np.argsort(-x, 1, kind="stable")[:, :k].astype(np.int32) for x in (p, q)]
    val = [np.take_along_axis(x, i, 1) for x, i in zip((p, q), top)]
    c = Topk(mk, val[0], top[0], val[1], top[1], bad, drafts, u, un, 3)
    got = c.run().read()
    check([g[ok] for g in got], want_topk(val[0], top[0], val[1], top[1], bad[ok], drafts, u, un[ok], 3), 4 * EPS)
    assert (got[0][no] == -1).all() and (got[1][no] == -1).all() and (got[2][no] == 0).all()


class Topk(Dense):
    def __init__(self, mk, pv, pi, qv, qi, lanes, drafts, u, un, most):
        self.mk, self.n, self.most, self.need = mk, len(lanes), most, 0
        self.bufs = [mk.to_device(x) if x is not None else None
                     for x in (pv, pi, qv, qi, lanes, np.asarray(list(drafts) + [0], np.int32),
                               np.asarray(list(u) + [0.0]), np.asarray(un, np.float64))]
        self.acc, self.tok = mk.to_device(np.full(self.n, 77, np.int32)), mk.to_device(
            np.full((self.n, most + 1), 77, np.int32))
        self.pr, self.work = mk.to_device(np.full((self.n, most + 1), 77, np.float32)), mk.to_device(
            np.full(64, 0xFF, np.uint8))
        b = [x.ptr if x is not None else None for x in self.bufs]
        self.args = (mk.h, b[0], b[1], pv.shape[1], len(pv), b[2], b[3], qv.shape[1] if qv is not None else 0,
                     len(drafts), b[4], self.n, most, b[5], b[6], b[7], self.acc.ptr, self.tok.ptr, self.pr.ptr)

    def run(self):
        mk_.check(mk_.load().mk_verify_topk(*self.args))
        return self


def want_topk(pv, pi, qv, qi, lanes, drafts, u, un, most):
    out = []
    for i, l in enumerate(lanes):
        out.append(verify64(l, lambda j: cut64(pv[l["row"] + j], pi[l["row"] + j], l, 0),
                            (lambda j: cut64(qv[l["first"] + j], qi[l["first"] + j], l, 0)) if qv is not None else None,
                            drafts, u, un[i], most + 1))
    return [np.array([o[k] for o in out]) for k in range(3)]


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("pk,qk", [(1, 1), (40, 40), (63, 64), (65, 20), (200, 300), (1024, 1024)])
def test_topk_against_plain(mk, pk, qk, certain):
    """Probabilities: the weight's float rounding (its exp may round the other way at a tie of the last bit), its sum's in
    64 bits and the quotient's, each half a step, against the same on the host."""
    rng = np.random.default_rng(pk + qk)
    counts, V = [4, 0, 8, 1, 3, 5, 2, 6], 3000
    lanes = lanes_of(counts, [0.7, 1.0, 0.0, 1.3, 0.9, 1.0, 2.0, 0.6], 0.05, 0.95)
    lanes["min_p"][3], lanes["top_p"][3] = 0.0, 1.0
    lanes["min_p"][5], lanes["top_p"][6] = 1.0, 0.0   # nothing but the first
    p, q, u, un = inputs(rng, counts, V, 1.0, 0.3)
    un[0], un[3] = 0.0, np.nextafter(1.0, 0.0)
    pi, qi = (np.argsort(-x, 1, kind="stable")[:, :k].astype(np.int32) for x, k in ((p, pk), (q, qk)))
    pv, qv = np.take_along_axis(p, pi, 1), np.take_along_axis(q, qi, 1)
    drafts = np.zeros(len(q), np.int32)
    for l in lanes:
        for j in range(l["first"], l["first"] + l["n_draft"]):
            ids, pr = cut64(qv[j], qi[j], l, V)
            drafts[j] = rng.choice(ids, p=pr.astype(np.float64) / pr.astype(np.float64).sum())
    drafts[1] = qi[1, -1]  # perhaps past the kept head
    if certain:
        qv = qi = None
    print("verify topk", pk, qk, certain, flush=True)
    c = Topk(mk, pv, pi, qv, qi, lanes, drafts, u, un, 8)
    got = c.run().read()
    check(got, want_topk(pv, pi, qv, qi, lanes, drafts, u, un, 8), 4 * EPS)
    again = c.run().read()
    assert all(np.array_equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("whole", [True, False])
def test_tokens_follow_the_target(mk, whole):
    """The point of the method: whatever the draft's distribution, the first token follows the target's. 60000 lanes over
    40 tokens, each count within 6 standard deviations."""
    rng = np.random.default_rng(7)
    V, n = 40, 60000
    p, q = rng.standard_normal((2, V)).astype(np.float32) * 1.5
    lanes = lanes_of([1] * n, 1.0)
    lanes["row"], drafts = 0, rng.choice(V, n, p=softmax64(q, 1.0)).astype(np.int32)
    rows = np.stack([p, p])
    u, un = rng.random(n), rng.random(n)
    print("verify, distribution", whole, flush=True)
    if whole:
        lanes["first"] = np.arange(n)
        # One draft row per draft is what the layout wants; a few thousand lanes at a time keep that small.
        counts = np.zeros(V)
        for a in range(0, n, 20000):
            l = lanes[a:a + 20000].copy()
            l["first"] -= a
            got = Dense(mk, rows, np.tile(q, (len(l), 1)), l, drafts[a:a + 20000], u[a:a + 20000], un[a:a + 20000],
                        1).run().read()
            counts += np.bincount(got[1][:, 0], minlength=V)
    else:
        pi, qi = (np.argsort(-x, kind="stable").astype(np.int32) for x in (p, q))
        lanes["first"], lanes["top_p"] = np.arange(n), 1.0
        got = Topk(mk, rows[:, pi], np.stack([pi, pi]), np.tile(q[qi], (n, 1)), np.tile(qi, (n, 1)), lanes, drafts, u, un,
                   1).run().read()
        counts = np.bincount(got[1][:, 0], minlength=V)
    want = softmax64(p, 1.0)
    assert (np.abs(counts - n * want) <= 6 * np.sqrt(n * want * (1 - want))).all(), (counts, n * want)


def test_topk_agrees_with_the_host_sampler(mk):
    """The same random numbers through mk_sampler_verify: accepted or not, and the token."""
    rng = np.random.default_rng(11)
    lane = dict(temperature=0.8, min_p=0.02, top_p=0.9)
    k, n = 30, 200
    pv, qv = (np.sort(2 * rng.standard_normal((n + 0, k)).astype(np.float32))[:, ::-1].copy() for _ in range(2))
    pi, qi = (np.stack([rng.permutation(60)[:k] for _ in range(n)]).astype(np.int32) for _ in range(2))
    dist = [(cut64(pv[i], pi[i], lane, 60), cut64(qv[i], qi[i], lane, 60)) for i in range(n)]
    drafts, u, un, want = [], [], [], []
    for i, (p, q) in enumerate(dist):
        drafts.append(int(rng.choice(q[0])))
        s = mk_.Sampler(seed=i + 1)
        tok, ok = s.verify([(float(a), int(b)) for b, a in zip(*p)], [(float(a), int(b)) for b, a in zip(*q)], drafts[-1])
        want.append((ok, tok))
        # The sampler's numbers: uniform() is the generator's next word over 2^64.
        a, b = mt64(i + 1)
        u.append(a)
        un.append(b)
    lanes = lanes_of([1] * n, lane["temperature"], lane["min_p"], lane["top_p"])
    rows = np.repeat(np.arange(n), 2)
    got = Topk(mk, pv[rows], pi[rows], qv, qi, lanes, drafts, u, un, 1).run().read()
    for i, (ok, tok) in enumerate(want):
        assert bool(got[0][i]) == ok and (ok or got[1][i, 0] == tok), (i, got[0][i], got[1][i], ok, tok)
    assert 10 <= sum(ok for ok, _ in want) <= n - 10  # both kinds occur


def mt64(seed):
    """The first two uniforms of a std::mt19937_64."""
    m = (1 << 64) - 1
    w = [seed]
    for i in range(1, 312):
        w.append((6364136223846793005 * (w[-1] ^ (w[-1] >> 62)) + i) & m)
    out = []
    for i in range(2):
        y = (w[i] & 0xFFFFFFFF80000000) | (w[i + 1] & 0x7FFFFFFF)
        z = w[i + 156] ^ (y >> 1) ^ (0xB5026F5AA96619E9 if y & 1 else 0)
        z ^= (z >> 29) & 0x5555555555555555
        z ^= (z << 17) & 0x71D67FFFEDA60000 & m
        z ^= (z << 37) & 0xFFF7EEE000000000 & m
        out.append((z ^ (z >> 43)) * 2.0 ** -64)
    return out


def test_captured_and_replayed(mk):
    hip = ctypes.CDLL("libamdhip64.so")
    rng = np.random.default_rng(12)
    counts, V = [3, 1, 4], 9000
    lanes = lanes_of(counts, [1.0, 0.0, 0.8])
    p, q, u, un = inputs(rng, counts, V)
    drafts = sample_drafts(rng, q, lanes)
    c = Dense(mk, p, q, lanes, drafts, u, un, 4)
    stream = ctypes.c_void_p(mk_.load().mk_stream(mk.h))
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    mk.sync()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    c.run()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
    for i in range(4):
        u, un = rng.random(len(u)), rng.random(len(un))
        c.u.upload(u)
        c.un.upload(un)
        print("replay", i, flush=True)
        assert hip.hipGraphLaunch(run, stream) == 0
        got = c.read()
        check(got, want_dense(p, q, lanes, drafts, u, un, 4))
        again = c.run().read()
        assert all(np.array_equal(a, b) for a, b in zip(got, again))
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0


def highest_first(z, k):
    """mk_topk's rows: values and ids by the order of their bits, NaN ahead of infinity, then by id."""
    u = z.view(np.uint32)
    key = np.where(u >> 31, ~u, u | np.uint32(1 << 31))
    ids = np.argsort(~key, 1, kind="stable")[:, :k].astype(np.int32)
    return np.take_along_axis(z, ids, 1), ids


@pytest.mark.parametrize("k", [40, 200])
def test_topk_infinities_and_nan(mk, k):
    """Candidates' logits by mk_verify's rules: NaN counts as -inf, which is no candidate, +inf as the largest float, a row
    of nothing but those has no token and refuses every draft, whatever the temperature and the cut."""
    rng = np.random.default_rng(31)
    temps = [1.0, 0.0, np.inf, 1e-45]
    kinds, V = 12, 500
    counts = [2] * (kinds * len(temps))
    lanes = lanes_of(counts, np.repeat(np.float32(temps), kinds), 0.05, 0.95)
    p, q, u, un = inputs(rng, counts, V)
    for i, l in enumerate(lanes):
        a, b, kind = l["row"], l["first"], i % kinds
        u[b:b + 2] = [0.0, 0.3]
        if kind == 0:                                      # one token has everything
            p[a, 17] = np.inf
        elif kind == 1:                                    # three share it
            p[a:a + 3, [9, 30, 77]] = np.inf
            q[b:b + 2, [30, 60]] = np.inf
        elif kind == 2:                                    # NaN ahead of the candidates, more of them than a wave's lanes
            p[a:a + 3, 40:40 + k // 2] = q[b, 11:20] = np.nan
        elif kind == 3:                                    # few candidates left
            p[a:a + 3, 5:] = q[b:b + 2, 7:] = -np.inf
        elif kind == 4:
            p[a] = -np.inf
        elif kind == 5:
            p[a] = np.nan
        elif kind == 6:                                    # nothing in the draft's row
            q[b] = -np.inf
        elif kind == 7:
            p[a, 3], q[b, 100:] = np.nan, np.nan
            lanes["min_p"][i] = 1.0
        elif kind == 8:
            p[a, 3] = q[b, 8] = np.nan
            lanes["top_p"][i] = 0.0
        elif kind == 9:                                    # the whole of the candidates, infinities of all kinds
            p[a:a + 3, ::3], p[a:a + 3, 1::3], p[a:a + 3, 4] = -np.inf, np.nan, np.inf
            lanes["min_p"][i], lanes["top_p"][i] = 0.0, 1.0
        elif kind == 10:                                   # negative NaN, the last of all
            p[a:a + 3, ::2] = np.uint32(0xFFC00000).view(np.float32)
        else:
            p[a + 1:a + 3] = -np.inf
    (pv, pi), (qv, qi) = highest_first(p, k), highest_first(q, k)
    drafts = qi[:, 0].copy()
    for i, l in enumerate(lanes):                          # drafts that the target likes, or its row's first entry
        drafts[l["first"]] = pi[l["row"], 0] if i % kinds in (3, 4, 5, 11) else drafts[l["first"]]

    def plain(cert):
        out = [verify64(l, lambda j: cut_any64(pv[l["row"] + j], pi[l["row"] + j], l),
                        None if cert else lambda j: cut_any64(qv[l["first"] + j], qi[l["first"] + j], l), drafts, u,
                        un[i], 3) for i, l in enumerate(lanes)]
        return [np.array([o[j] for o in out]) for j in range(3)]

    for cert in (False, True):
        print("verify topk, infinities and NaN", k, cert, flush=True)
        got = Topk(mk, pv, pi, None if cert else qv, None if cert else qi, lanes, drafts, u, un, 2).run().read()
        check(got, plain(cert), 4 * EPS)
        for i in range(len(lanes)):
            if i % kinds in (4, 5):
                assert got[0][i] == 0 and (got[1][i] == -1).all() and (got[2][i] == 0).all()


# Rows of several segments per workgroup (a span, from 4096 segments in all): 3 of 38, 5 of 9 whose rows no vector
# divides, the last span shorter; vocabularies whose blocks a wave's registers do not hold (past 163840).
SPANS = [([8] * 12, 151936, (0, 0)), ([8] * 12, 151936, (3, 1)), ([1, 0, 2, 3] * 80, 35001, (0, 0)),
         ([2, 1, 0, 3, 1, 2], 262144, (0, 0)), ([1, 2, 2], 200001, (0, 0)), ([3] * 12, 262144, (0, 0))]


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("counts,V,pads", SPANS, ids=lambda v: f"{len(v)}x{max(v)}" if isinstance(v, list) else str(v))
def test_dense_spans_of_segments(mk, counts, V, pads, certain):
    rng = np.random.default_rng(V + len(counts) + 5)
    lanes = lanes_of(counts, [[0.7, 0.0, 1.0, 1.3, 2.0][i % 5] for i in range(len(counts))])
    p, q, u, un = inputs(rng, counts, V, 1.0, 0.3)
    p[:, :16] -= 30.0  # no draw ends in the first tokens
    drafts = rng.integers(0, V, len(q)).astype(np.int32)
    drafts[::2] = q[::2].argmax(1)
    print("verify, spans", len(counts), V, pads, certain, flush=True)
    c = Dense(mk, p, None if certain else q, lanes, drafts, u, un, max(counts), pads)
    got = c.run().read()
    check(got, want_dense(p, None if certain else q, lanes, drafts, u, un, max(counts)))
    again = c.run().read()
    assert all(np.array_equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("V", [36864, 36866])
def test_dense_maxima_across_segments(mk, V):
    """Nine segments, in spans of several: maxima that each segment raises by more than its sums reach (346 T), or lowers,
    ties of a greedy row in a later segment of a span and in several, one finite logit in a row's end."""
    rng = np.random.default_rng(3)
    counts = [1] * 360  # 1080 rows: spans of four, without draft rows three
    temps = np.float32([1.0, 0.0, 0.3, 1.0, 0.0, 2.0])
    lanes = lanes_of(counts, np.tile(temps, 60))
    p, q, u, un = inputs(rng, counts, V, 1.0, 0.3)
    seg = np.arange(V) // 4096
    for i, l in enumerate(lanes):
        for row in (p[l["row"]], p[l["row"] + 1], q[l["first"]]):
            kind = i // 6 % 6
            step = np.float32(400.0) * max(l["temperature"], np.float32(1.0))
            if kind == 0:
                row += step * seg
            elif kind == 1:
                row -= step * seg
            elif kind == 2:                # up and down, the highest in the middle
                row += step * np.array([0, 3, 1, 4, 6, 2, 5, 6, 0, 0])[seg]
            elif kind == 3:                # ties, first in the third segment
                row[[2 * 4096 + 1500, 2 * 4096 + 1501, 3 * 4096 + 2, 7 * 4096]] = 60.0
            elif kind == 4:                # nothing but one token near the end
                row[:] = -np.inf
                row[V - 1 - i % 5] = -3.0
            else:                          # a high start in one thread's logits, masked segments behind it
                row[16:20] += step
                row[4096:5 * 4096] = -np.inf
    drafts = q.argmax(1).astype(np.int32)
    drafts[::7] = 5 * 4096 + 77
    for qq in (q, None):
        print("verify, maxima across segments", V, qq is None, flush=True)
        got, want = Dense(mk, p, qq, lanes, drafts, u, un, 1).run().read(), want_dense(p, qq, lanes, drafts, u, un, 1)
        assert np.array_equal(got[0], want[0])
        # Where the draft was refused although P and Q are equal up to rounding (a draft that neither gives, four ties
        # that share both), the next token is drawn by rounding. A weight's exponent d, in 64ths of a power of two, is a
        # difference times a quotient of three roundings, so off by 2^-51 |d|, |d| < 63000, which is 2^-51 63000 ln 2 / 64 =
        # 3.1e-13 of the weight; its series adds 4e-14: together less than 2^-41. A probability, its quotient by a sum of
        # such weights, is within 2^-40, P - Q within 2^-39 max(P, Q), and a positive part that sums to less than
        # 2^-39 (sum P + sum Q) = 2^-38 is not known at all. (Numpy's roundings are others, not fewer.) Any token may come
        # whose difference can be positive.
        same = np.ones(len(lanes), bool)
        for i in np.flatnonzero((got[1] != want[1]).any(1)):
            l, n = lanes[i], got[0][i]
            assert qq is not None and n < l["n_draft"] and np.array_equal(got[1][i, :n], want[1][i, :n])
            P, Q = (softmax64(x, l["temperature"]) for x in (p[l["row"] + n], q[l["first"] + n]))
            x = got[1][i, n]
            assert np.maximum(P - Q, 0.0).sum() < 2.0 ** -38 and P[x] >= (1 - 2.0 ** -39) * Q[x] and P[x] > 0
            same[i] = False
        check([g[same] for g in got], [w[same] for w in want])
        assert same.sum() >= len(lanes) - 60


@pytest.mark.parametrize("certain", [False, True])
def test_as_many_drafts_as_there_may_be(mk, certain):
    """256 drafts, all accepted, refused at the last, in the middle and at the first; whole rows and candidates."""
    rng = np.random.default_rng(6)
    counts, V, k = [256, 256, 255, 0, 256, 129, 256], 300, 40
    lanes = lanes_of(counts, [1.0, 0.8, 1.0, 1.0, 1.0, 1.2, 0.0])
    p, q, u, un = inputs(rng, counts, V, 1.0, 0.2)
    (pv, pi), (qv, qi) = highest_first(p, k), highest_first(q, k)
    drafts, first = np.zeros(len(q), np.int32), lanes["first"]
    for l in lanes:
        for j in range(l["n_draft"]):  # a token that both rows have among their first
            drafts[l["first"] + j] = pi[l["row"] + j, 0]
    u *= 1e-9
    for i, j in ((1, 255), (2, 254), (4, 100), (5, 0)):
        drafts[first[i] + j] = pi[lanes["row"][i] + j, -1]
        u[first[i] + j] = 1.0 - 1e-9
        q[first[i] + j, drafts[first[i] + j]] = 9.0
    qv, qi = highest_first(q, k)
    print("verify, 256 drafts", certain, flush=True)
    got = Dense(mk, p, None if certain else q, lanes, drafts, u, un, 256).run().read()
    check(got, want_dense(p, None if certain else q, lanes, drafts, u, un, 256))
    assert list(got[0][[1, 2, 3, 4, 5]]) == [255, 254, 0, 100, 0] and (got[0][0] == 256 or not certain)
    a = (None, None) if certain else (qv, qi)
    got = Topk(mk, pv, pi, *a, lanes, drafts, u, un, 256).run().read()
    check(got, want_topk(pv, pi, *a, lanes, drafts, u, un, 256), 4 * EPS)
    assert list(got[0][[1, 2, 3, 4, 5]]) == [255, 254, 0, 100, 0]
