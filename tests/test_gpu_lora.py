"""mk_lora against plain 64-bit products: all three adapter types, ranks that no vector divides, tokens that share an
adapter across and inside tiles, tokens without one, ids and ranks outside the table, in place and out of place,
unaligned strides, column counts that no vector divides, captured graphs."""
import ctypes

import numpy as np
import pytest

import malkin_amd as mk_
from operator_cases import lora64, lora_norms64

pytestmark = pytest.mark.gpu

KINDS = {"f32": mk_.F32, "f16": mk_.F16, "bf16": mk_.BF16}


def encode(x, kind):
    """x rounded to the type: (its bytes as an array, the values they stand for)."""
    if kind == "f32":
        return x, x
    if kind == "f16":
        h = x.astype(np.float16)
        return h, h.astype(np.float32)
    u = (x.view(np.uint32) + 0x8000 & 0xFFFF0000).astype(np.uint32)
    return (u >> 16).astype(np.uint16), u.view(np.float32)


class Set:
    """Adapters on the device: ranks[i] (0: an entry that takes no part)."""

    def __init__(self, mk, rng, kind, ranks, rows, cols, off=0):
        self.host, self.bufs = [], []
        table = np.zeros(len(ranks), mk_.LORA_ADAPTER)
        for i, r in enumerate(ranks):
            m = max(abs(r), 1)
            a, av = encode((rng.standard_normal((m, cols)) / np.sqrt(cols)).astype(np.float32), kind)
            b, bv = encode(rng.standard_normal((rows, m)).astype(np.float32), kind)
            pad = np.zeros(off, a.dtype)  # off: values before the matrix, so that it is not 16-byte aligned
            ba, bb = (mk.to_device(np.concatenate([pad, x.ravel()])) for x in (a, b))
            self.bufs += [ba, bb]
            table[i] = (ba.p + pad.nbytes, bb.p + pad.nbytes, 0.5 + i, r)
            self.host.append((av, bv, 0.5 + i) if r > 0 else None)
        self.table = mk.to_device(table if len(table) else np.zeros(1, mk_.LORA_ADAPTER))


def call(mk, kind, s, n_adapters, max_rank, ids, x, rows, base, pads=(0, 0, 0), in_place=False):
    n, cols = x.shape
    px, pb, py = pads

    def wide(v, pad, fill):
        w = np.full((n, v.shape[1] + pad), fill, np.float32)
        w[:, :v.shape[1]] = v
        return mk.to_device(w)

    dx, dids = wide(x, px, np.nan), mk.to_device(np.asarray(ids, np.int32))
    db = wide(base, pb, 5.0) if base is not None else None
    dy = db if in_place else wide(np.full((n, rows), 9.0, np.float32), py, 4.0)
    need = mk_.load().mk_lora_workspace(n, max_rank, cols)
    work = mk.to_device(np.full(need + 64, 0xFF, np.uint8))  # NaN to whoever reads what was not written
    ys = rows + (pb if in_place else py)
    args = (mk.h, KINDS[kind], s.table.ptr, n_adapters, max_rank, dids.ptr, dx.ptr, cols + px, n, rows, cols,
            db.ptr if db is not None else None, rows + pb, dy.ptr, ys, work.ptr, need)
    mk_.check(mk_.load().mk_lora(*args))
    y = dy.download(np.float32).reshape(n, ys)
    assert (y[:, rows:] == (5.0 if in_place else 4.0)).all()
    assert (work.download(np.uint8)[need:] == 0xFF).all()
    return y[:, :rows], args, (dx, dids, db, dy, work)


def check(got, want, tol):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])


# ranks, rows, cols, ids
CASES = [
    ([8], 64, 32, [0]),
    ([16], 256, 256, [0, 0, 0]),
    ([1, 3, 16], 96, 96, [2, 0, 1, -1, 2, 0]),
    ([16, 32, 64, 8], 1024, 512, [t % 5 - 1 for t in range(33)]),
    ([5, 20, 33], 520, 288, [0, 1, 2, 7, -3, 1] * 6),
    ([64], 6144, 4096, [0] * 17),
    ([16, 16], 300, 1000, [0] * 40 + [1] * 40 + [-1] * 3),
    ([200, 512], 128, 128, [1, 0, 1]),
    ([4] * 30, 64, 2048, list(range(30)) + [3] * 5),
    ([7], 37, 45, [0, -1, 0]),                       # nothing that a vector divides
    ([16], 4096, 12288, [0] * 4),
    ([32, 8, 16], 640, 320, [0] * 200 + [1] * 7 + [2] * 90),
]


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[1]}-{c[2]}-n{len(c[3])}")
def test_against_plain(mk, case, kind):
    ranks, rows, cols, ids = case
    rng = np.random.default_rng(rows + cols)
    s = Set(mk, rng, kind, ranks, rows, cols)
    x = rng.standard_normal((len(ids), cols)).astype(np.float32)
    x[:, ::37] *= 30.0
    base = rng.standard_normal((len(ids), rows)).astype(np.float32)
    want, tol = lora64(x, s.host, ids, base, rows)
    print("lora", case[1:3], len(ids), kind, flush=True)
    got, args, keep = call(mk, kind, s, len(ranks), max(ranks), ids, x, rows, base)
    check(got, want, tol)
    mk_.check(mk_.load().mk_lora(*args))  # again on the same buffers: the same bits
    again = keep[3].download(np.float32).reshape(len(ids), rows)
    assert np.array_equal(got.view(np.uint32), again.view(np.uint32))
    # In place, and without a base.
    got, _, _ = call(mk, kind, s, len(ranks), max(ranks), ids, x, rows, base, in_place=True)
    check(got, want, tol)
    want, tol = lora64(x, s.host, ids, None, rows)
    got, _, _ = call(mk, kind, s, len(ranks), max(ranks), ids, x, rows, None)
    check(got, want, tol)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("off,pads", [(0, (1, 0, 0)), (0, (0, 3, 1)), (1, (0, 0, 0)), (3, (4, 4, 8)), (0, (4, 4, 8))])
def test_strides_and_alignment(mk, kind, off, pads):
    rng = np.random.default_rng(off)
    ranks, rows, cols, ids = [16, 12], 264, 288, [0, 1, -1, 0, 1] * 5
    s = Set(mk, rng, kind, ranks, rows, cols, off)
    x = rng.standard_normal((len(ids), cols)).astype(np.float32)
    base = rng.standard_normal((len(ids), rows)).astype(np.float32)
    want, tol = lora64(x, s.host, ids, base, rows)
    print("lora strides", kind, off, pads, flush=True)
    for in_place in (False, True):
        got, _, _ = call(mk, kind, s, 2, 16, ids, x, rows, base, pads, in_place)
        check(got, want, tol)


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_one_token_shows_nothing_of_another(mk, kind):
    """A token of NaN or infinities, beside others of the same adapter and of others, changes its own row alone."""
    rng = np.random.default_rng(11)
    ranks, rows, cols = [16, 40], 300, 544
    ids = [0, 1, 0, -1, 1, 0, 0] * 4
    s = Set(mk, rng, kind, ranks, rows, cols)
    x = rng.standard_normal((len(ids), cols)).astype(np.float32)
    base = rng.standard_normal((len(ids), rows)).astype(np.float32)
    want, tol = lora64(x, s.host, ids, base, rows)
    x[2, 5:], x[11], x[10, ::3], base[13, ::2] = np.nan, np.inf, np.nan, np.nan
    print("lora, one token of NaN", kind, flush=True)
    ok = [i for i in range(len(ids)) if i not in (2, 11, 13)]  # token 10 has no adapter
    for in_place in (False, True):
        got, _, _ = call(mk, kind, s, 2, 40, ids, x, rows, base, in_place=in_place)
        check(got[ok], want[ok], tol[ok])
        assert not np.isfinite(got[[2, 11]]).any() and np.isnan(got[13, ::2]).all()
        check(got[13, 1::2], want[13, 1::2], tol[13, 1::2])


def test_entries_that_take_no_part(mk):
    """Ranks of 0, negative or past max_rank, ids outside the table: the base as it is, its -0 and NaN included."""
    rng = np.random.default_rng(4)
    ranks, rows, cols = [16, 0, -2, 24], 128, 64
    s = Set(mk, rng, "f16", ranks, rows, cols)
    s.host[3] = None  # above max_rank
    ids = [0, 1, 2, 3, 4, -1, 2**31 - 1, -2**31, 0]
    x = rng.standard_normal((len(ids), cols)).astype(np.float32)
    x[1:8] = np.inf  # what no adapter reads reaches nothing, not even the tile's other tokens
    base = rng.standard_normal((len(ids), rows)).astype(np.float32)
    base[1, 0], base[2, 1] = -0.0, np.inf
    x0 = np.where(np.isfinite(x), x, 0.0).astype(np.float32)
    want, tol = lora64(x0, s.host, ids, base, rows)
    for in_place in (False, True):
        print("lora, entries out of range", in_place, flush=True)
        got, _, _ = call(mk, "f16", s, 4, 16, ids, x, rows, base, in_place=in_place)
        assert np.array_equal(got[1:8].view(np.uint32), base[1:8].view(np.uint32))
        check(got[[0, 8]], want[[0, 8]], tol[[0, 8]])
    got, _, _ = call(mk, "f16", s, 0, 16, ids, x, rows, None)  # an empty table
    assert (got == 0).all()


def test_captured_and_replayed(mk):
    """The adapters of the tokens change between replays of one graph."""
    hip = ctypes.CDLL("libamdhip64.so")
    rng = np.random.default_rng(6)
    ranks, rows, cols, n = [16, 8, 32], 512, 1024, 20
    s = Set(mk, rng, "bf16", ranks, rows, cols)
    x = rng.standard_normal((n, cols)).astype(np.float32)
    base = rng.standard_normal((n, rows)).astype(np.float32)
    _, args, keep = call(mk, "bf16", s, 3, 32, [0] * n, x, rows, base)
    stream = ctypes.c_void_p(mk_.load().mk_stream(mk.h))
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    mk.sync()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    mk_.check(mk_.load().mk_lora(*args))
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
    for i in range(4):
        ids = rng.integers(-1, 3, n).astype(np.int32)
        keep[1].upload(ids)
        print("replay", i, flush=True)
        assert hip.hipGraphLaunch(run, stream) == 0
        got = keep[3].download(np.float32).reshape(n, rows)
        want, tol = lora64(x, s.host, ids, base, rows)
        check(got, want, tol)
        mk_.check(mk_.load().mk_lora(*args))
        assert np.array_equal(got.view(np.uint32), keep[3].download(np.uint32).reshape(n, rows))
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("ranks", [[1], [8, 3], [16, 20]])
def test_infinite_x(mk, ranks, kind):
    """Infinities in a token give what the formula gives, infinities with their sign or NaN, at ranks that no tile of
    sixteen fills too; the other tokens of the adapter are as without them."""
    rng = np.random.default_rng(21)
    rows, cols, n = 272, 160, 40
    s = Set(mk, rng, kind, ranks, rows, cols)
    ids = [t % len(ranks) for t in range(n)]
    x = rng.standard_normal((n, cols)).astype(np.float32)
    base = rng.standard_normal((n, rows)).astype(np.float32)
    want, tol = lora64(x, s.host, ids, base, rows)
    for t, c in ((0, 0), (5, 7), (18, cols - 1), (39, 64)):
        x[t, c] = np.inf if t % 2 else -np.inf
        with np.errstate(invalid="ignore"):
            want[t], _ = lora64(x[t:t + 1], s.host, ids[t:t + 1], base[t:t + 1], rows)
    print("lora, infinite x", ranks, kind, flush=True)
    got, _, _ = call(mk, kind, s, len(ranks), max(ranks), ids, x, rows, base)
    odd = ~np.isfinite(want)
    assert odd[[0, 5, 18, 39]].all() and odd.sum() == 4 * rows and (ranks != [1] or np.isinf(want[odd]).all())
    assert np.array_equal(got[odd].astype(np.float64), want[odd], equal_nan=True)
    check(got[~odd], want[~odd], tol[~odd])


def test_any_bound_on_the_table(mk):
    """The number of adapters only bounds the ids: the largest int, a bound that the caller does not know better."""
    rng = np.random.default_rng(8)
    ranks, rows, cols, ids = [16, 8, 5], 128, 64, [0, 2, 1, -1, 1, 2, 0, -5] * 10
    s = Set(mk, rng, "f16", ranks, rows, cols)
    x = rng.standard_normal((len(ids), cols)).astype(np.float32)
    base = rng.standard_normal((len(ids), rows)).astype(np.float32)
    want, tol = lora64(x, s.host, ids, base, rows)
    bits = []
    for bound in (3, 13, 14, 15, 16, 2**31 - 1):
        print("lora, bound", bound, flush=True)
        got, _, _ = call(mk, "f16", s, bound, 16, ids, x, rows, base)
        check(got, want, tol)
        bits.append(got.view(np.uint32))
    assert all(np.array_equal(bits[0], b) for b in bits)


# Large ranks over several 16-token tiles and 64-token windows, more adapters than a window's few slots.
LARGE = [
    ([65], 272, 256, [0] * 17),
    ([200, 65], 260, 288, [0] * 30 + [1] * 34),
    ([512, 128], 320, 256, [0] * 40 + [1] * 40 + [0] * 20),
    ([128, 512], 200, 136, [t % 3 - 1 for t in range(100)]),
    ([100], 70, 45, [0] * 33),
    ([8 + 3 * i for i in range(20)], 264, 320, [(7 * t) % 21 - 1 for t in range(200)]),
    ([96] * 15, 256, 2048, [t % 15 for t in range(130)]),
]


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("case", CASES + LARGE, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[1]}-{c[2]}-n{len(c[3])}")
def test_close_as_a_whole(mk, case, kind):
    """Every element within its bound, and the error of every token's row as small as sums in fp32 leave it."""
    ranks, rows, cols, ids = case
    rng = np.random.default_rng(rows + cols + 1)
    s = Set(mk, rng, kind, ranks, rows, cols)
    x = rng.standard_normal((len(ids), cols)).astype(np.float32)
    base = rng.standard_normal((len(ids), rows)).astype(np.float32)
    print("lora as a whole", case[1:3], len(ids), kind, flush=True)
    want, tol = lora64(x, s.host, ids, base, rows)
    for in_place in (False, True):
        got, _, _ = call(mk, kind, s, len(ranks), max(ranks), ids, x, rows, base, in_place=in_place)
        check(got, want, tol)
    got, _, _ = call(mk, kind, s, len(ranks), max(ranks), ids, x, rows, None)
    want, tol = lora_norms64(x, s.host, ids, rows)
    off = np.sqrt(((got - want) ** 2).sum(-1))
    assert (off <= tol).all(), (off / np.maximum(tol, 1e-30)).max()
