"""mk_beam_select against sums and sorts in 64 bits: beams that have ended or are not there, masked and infinite logits, ties,
vocabularies of one token and of many segments, more candidates asked for than there are, strides, captured graphs."""
import ctypes

import numpy as np
import pytest

import malkin_amd as mk_
from kv4_cases import beams64

pytestmark = pytest.mark.gpu


class Call:
    def __init__(self, mk, logits, scores, done, eos, beams, k, pad=0):
        rows, V = logits.shape
        self.mk, self.groups, self.k = mk, rows // beams, k
        wide = np.full((rows, V + pad), 1e9, np.float32)
        wide[:, :V] = logits
        self.l, self.s = mk.to_device(wide), mk.to_device(scores.astype(np.float32))
        self.d = mk.to_device(done.astype(np.int32)) if done is not None else None
        self.out = [mk.to_device(np.full(self.groups * k + 3, 55, t)) for t in (np.float32, np.int32, np.int32)]
        self.need = mk_.load().mk_beam_workspace(self.groups, beams, V, k)
        self.work = mk.to_device(np.full(self.need + 64, 0xA5, np.uint8))
        self.args = (mk.h, self.l.ptr, V + pad, self.groups, beams, V, self.s.ptr, self.d.ptr if self.d else None, eos, k,
                     *(b.ptr for b in self.out), self.work.ptr, self.need)

    def run(self):
        mk_.check(mk_.load().mk_beam_select(*self.args))

    def read(self):
        s, q, t = (b.download(x) for b, x in zip(self.out, (np.float32, np.int32, np.int32)))
        n = self.groups * self.k
        assert (s[n:] == 55).all() and (q[n:] == 55).all() and (t[n:] == 55).all()
        assert (self.work.download(np.uint8)[self.need:] == 0xA5).all()
        return [x[:n].reshape(self.groups, self.k) for x in (s, q, t)]


def check(got, want):
    """Rows and tokens are equal; a score in 64 bits is off by less than 2^-40 of its parts, then rounded to 32."""
    s, q, t = got
    for g, best in enumerate(want):
        assert [(int(a), int(b)) for a, b in zip(q[g], t[g])] == [(b[1], b[2]) for b in best], g
        w = np.array([b[0] for b in best])
        fine = np.isfinite(w)
        assert (s[g][~fine] == -np.inf).all()
        assert (np.abs(s[g][fine] - w[fine]) <= 2.0 ** -24 * np.abs(w[fine]) + 2.0 ** -38 * 100).all()


def inputs(rng, groups, beams, V, peaks=True):
    z = (1.5 * rng.standard_normal((groups * beams, V))).astype(np.float32)
    if peaks:
        for r in z:
            r[rng.integers(0, V, min(12, V))] += 12
    return z, (-1 - 5 * rng.random(groups * beams)).astype(np.float32)


CASES = [  # groups, beams, vocabulary, k, pad
    (1, 1, 1, 1, 0), (2, 2, 3, 5, 1), (1, 4, 151936, 8, 0), (3, 4, 5000, 4, 3), (2, 8, 4096, 16, 0), (1, 3, 4097, 17, 5),
    (5, 32, 3203, 64, 0), (1, 64, 20011, 128, 0), (1, 64, 151936, 128, 0), (30, 5, 151936, 10, 2), (2, 1, 70000, 128, 0),
    (1, 2, 2097152, 3, 0), (300, 2, 100, 2, 0), (1, 16, 8192, 1, 0), (7, 4, 129, 128, 0),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_plain(mk, case):
    groups, beams, V, k, pad = case
    rng = np.random.default_rng(V + k)
    z, s = inputs(rng, groups, beams, V, V > 50)
    for done in (None, (rng.random(len(s)) < 0.3)):
        print("beams", case, done is not None, flush=True)
        c = Call(mk, z, s, done, V // 2, beams, k, pad)
        c.run()
        want, gap = beams64(z, s, done, V // 2, beams, k)
        assert gap > 1e-12
        got = c.read()
        check(got, want)
        c.run()
        for a, b in zip(got, c.read()):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("beams,k", [(4, 8), (32, 64), (3, 128)])
def test_masks_and_ends(mk, beams, k):
    """NaN and -inf are no candidates, +inf is the largest float, beams that are not there, ended beams, groups of nothing."""
    rng = np.random.default_rng(k)
    groups, V = 9, 9001
    z, s = inputs(rng, groups, beams, V)
    done = rng.random(len(s)) < 0.2
    z[:, rng.random(V) < 0.4] = -np.inf
    first = lambda g: g * beams  # noqa: E731
    z[first(1)] = np.nan
    z[first(1) + 1, 100] = np.inf
    z[first(2):first(3), :] = -np.inf
    z[first(3):first(4), 7:] = -np.inf  # seven tokens left, at most
    s[first(4):first(5)] = -np.inf
    s[first(5)], s[first(5) + 1], s[first(5) + 2] = np.nan, np.inf, -np.inf
    done[first(6):first(7)] = True
    done[first(2):first(3)] = False
    s[first(6)] = -np.inf
    z[first(7), :] = np.inf
    z[first(7) + 1, ::3] = np.finfo(np.float32).max
    print("beams, masks", beams, k, flush=True)
    c = Call(mk, z, s, done, 8, beams, k)
    c.run()
    with np.errstate(invalid="ignore", over="ignore"):
        want, _ = beams64(z, s, done, 8, beams, k)
    check(c.read(), want)


@pytest.mark.parametrize("V", [100, 4096, 30000])
@pytest.mark.parametrize("beams,k", [(1, 5), (4, 8), (8, 128), (64, 128), (64, 16)])
def test_ties(mk, V, beams, k):
    """Equal logits, equal beams: the lower beam, then the lower token; sorted logits; zeros of both signs."""
    rng = np.random.default_rng(V + k)
    flat = np.zeros((beams, V), np.float32)
    few = np.round(rng.standard_normal((beams, V))).astype(np.float32)
    few[:] = few[0]
    signs = np.where(rng.random((beams, V)) < 0.5, np.float32(0), np.float32(-0.0))
    up = np.tile(np.arange(V, dtype=np.float32) / 1024, (beams, 1))
    z = np.concatenate([flat, few, signs, up, up[:, ::-1]])
    s = np.full(len(z), -2.0, np.float32)
    print("beams, ties", V, beams, k, flush=True)
    c = Call(mk, z, s, None, 0, beams, k)
    c.run()
    got = c.read()
    # Equal rows have equal sums on the device too, so that ties between beams are ties there.
    check(got, beams64(z, s, None, 0, beams, k)[0])


def test_captured(mk):
    hip = ctypes.CDLL("libamdhip64.so")
    rng = np.random.default_rng(3)
    sets = [inputs(rng, 6, 4, 40000) for _ in range(2)]
    calls = [Call(mk, z, s, None, 0, 4, 8) for z, s in sets]
    stream, graph, run = ctypes.c_void_p(mk_.load().mk_stream(mk.h)), ctypes.c_void_p(), ctypes.c_void_p()
    mk.sync()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    for c in calls:
        c.run()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
    for i in range(4):
        for c, (z, s) in zip(calls, sets):
            s = np.roll(s, i)
            c.s.upload(s)
        print("beams, replay", i, flush=True)
        assert hip.hipGraphLaunch(run, stream) == 0
        for c, (z, s) in zip(calls, sets):
            got = c.read()
            check(got, beams64(z, np.roll(s, i), None, 0, 4, 8)[0])
            c.run()
            for a, b in zip(got, c.read()):
                assert np.array_equal(a, b)
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
