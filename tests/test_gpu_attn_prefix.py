"""mk_attention_prefix against a plain 64-bit attention: decoding, chains of drafts and prompts behind a shared prefix,
prefixes and rows of one key and of lengths that no tile divides, tokens without keys or inside the prefix, values in
places that no token may see, strides, row offsets, a cache past 2^32 bytes, captured graphs."""
import ctypes

import numpy as np
import pytest

import malkin_amd as mk_
from operator_cases import attention64, attention_norms64, make_cache

pytestmark = pytest.mark.gpu


def to_cache(mk, c):
    k, v, ks, vs = c
    bufs = [mk.to_device(x) for x in (k, v, ks, vs)]
    return bufs, mk_.MkKvCache(*(b.p for b in bufs), k.shape[0], k.shape[1], k.shape[2], k.shape[4], k.shape[3])


class Call:
    """Inputs of one call on the device; run() queues it."""

    def __init__(self, mk, q, H, pre, pseq, P, kv, row0, layer, seq, keys, most, pad=0, q8=False, same=False):
        self.mk, self.n, self.H, self.d, KV = mk, len(seq), H, kv[0].shape[4], kv[0].shape[2]
        HD = H * self.d
        self.HD, self.stride = HD, HD + pad
        wide = np.full((self.n, self.stride), 7.0, np.float32)
        wide[:, :HD] = q
        self.kv_b, self.kv = to_cache(mk, kv)
        self.pre_b, self.pre = (self.kv_b, self.kv) if same else to_cache(mk, pre) if P else (None, None)
        self.q, self.out = mk.to_device(wide), mk.to_device(np.full((self.n, self.stride), 3.0, np.float32))
        self.seq, self.keys = (mk.to_device(np.asarray(x, np.int32)) for x in (seq, keys))
        self.xq = mk.to_device(np.zeros(self.n * HD // 32 * 40, np.uint8)) if q8 else None
        need = mk_.load().mk_attention_prefix_workspace(self.n, H, KV, self.d, P, most)
        self.work = mk.to_device(np.full(max(need, 16) + 64, 0xA5, np.uint8))
        self.need = need
        self.args = (mk.h, self.q.ptr, self.stride, self.out.ptr, self.stride, self.n, H,
                     ctypes.byref(self.pre) if self.pre is not None else None, pseq, P, ctypes.byref(self.kv), row0,
                     layer, self.seq.ptr, self.keys.ptr, most, self.xq.ptr if q8 else None, self.work.ptr, need)

    def run(self):
        mk_.check(mk_.load().mk_attention_prefix(*self.args))

    def result(self):
        o = self.out.download(np.float32).reshape(self.n, self.stride)
        assert (o[:, self.HD:] == 3.0).all()  # what lies between rows is left as it was
        assert (self.work.download(np.uint8)[max(self.need, 16):] == 0xA5).all()
        return o[:, :self.HD]


def check(got, want, tol):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])


# heads, KV heads, head_dim, tokens of each sequence, prefix, rows of its own the last token of each sees, row0
CASES = [
    (4, 2, 128, [1], 1, [1], 0),
    (4, 2, 64, [1, 1], 16, [1, 2], 0),
    (8, 8, 128, [1, 1, 1], 33, [5, 31, 64], 0),       # one query head per KV head
    (32, 8, 128, [1] * 8, 257, [1, 17, 64, 65, 127, 128, 129, 200], 0),
    (40, 8, 128, [5, 5, 1, 3], 130, [40, 7, 1, 64], 130),  # five heads per KV head, chains, absolute rows
    (8, 2, 64, [3, 1, 9], 100, [50, 2, 9], 11),
    (16, 1, 128, [2, 1], 65, [9, 3], 0),              # sixteen heads of one KV head
    (32, 1, 64, [1, 2], 40, [4, 6], 3),               # and thirty-two
    (4, 2, 128, [70, 33], 95, [90, 33], 0),           # prompts
    (32, 8, 128, [300], 64, [300], 0),
    (4, 2, 128, [1] * 40, 1000, list(range(1, 41)), 0),
    (16, 8, 128, [1, 1], 5000, [700, 1], 0),
    (6, 2, 128, [4, 4], 0, [40, 4], 0),               # no prefix
    (4, 4, 64, [1], 0, [1], 0),
    (8, 8, 64, [770], 3333, [770], 0),                # long chunks, two workgroups a CU
    (8, 2, 128, [5] * 10, 92, [300 + 13 * i for i in range(10)], 0),  # runs of drafts, their own rows split
]


def build(rng, H, KV, d, new, P, rows, row0, n_layer=2):
    n_seq = len(new) + 1
    slots = [(3 * i + 1) % n_seq if n_seq % 3 else i for i in range(len(new))]
    kv = make_cache(rng, n_layer, n_seq, KV, row0 + max(rows) + 3, d)
    pre = make_cache(rng, n_layer, 3, KV, P + 2, d) if P else None
    seq = [s for s, m in zip(slots, new) for _ in range(m)]
    keys = [P + r - m + j + 1 for r, m in zip(rows, new) for j in range(m)]
    q = (1.5 * rng.standard_normal((len(seq), H * d))).astype(np.float32)
    return q, pre, kv, seq, keys


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:3]) + f"-n{sum(c[3])}-p{c[4]}")
def test_against_plain(mk, case):
    H, KV, d, new, P, rows, row0 = case
    rng = np.random.default_rng(sum(new) + P)
    q, pre, kv, seq, keys = build(rng, H, KV, d, new, P, rows, row0)
    want, tol = attention64(q, H, pre, 1, P, kv, row0, 1, seq, keys)
    for pad, q8 in ((0, False), (5, True)):
        print("prefix attention", case, pad, q8, flush=True)
        c = Call(mk, q, H, pre, 1, P, kv, row0, 1, seq, keys, max(keys), pad, q8)
        c.run()
        got = c.result()
        check(got, want, tol)
        if q8:  # the BlockQ8 rows are those of the output
            ref = mk.alloc(c.n * c.HD // 32 * 40)
            dense = mk.to_device(got)
            mk_.check(mk_.load().mk_quantize_q8(mk.h, dense.ptr, c.n, c.HD, ref.ptr))
            assert np.array_equal(ref.download(np.uint8), c.xq.download(np.uint8))
        c.run()  # again on the same buffers: the same bits
        assert np.array_equal(got.view(np.uint32), c.result().view(np.uint32))


@pytest.mark.parametrize("d", [64, 128])
def test_rows_without_keys_and_inside_the_prefix(mk, d):
    """Padded rows get zeros, a token may end inside the prefix, a bound above every n_keys changes nothing but the
    split, one below cuts; scales and values that no token sees (infinities, NaN) reach nothing."""
    rng = np.random.default_rng(3)
    H, KV, P = 8, 2, 150
    q, pre, kv, _, _ = build(rng, H, KV, d, [1] * 9, P, [40] * 9, 0)
    seq = [0, 5, -1, 2, 99, 3, 3, 4, 1]
    keys = [0, 7, 20, 150, 160, 151, -4, 190, 171]
    hold = [0, 7, 0, 150, 0, 151, 0, 190, 171]
    # Rows past what anyone reads: sequence 4 is read to its row 39, sequence 1 to row 20, the others less.
    for x in (kv[2], kv[3]):
        x[1, 4, :, 40:] = np.nan
        x[1, 1, :, 21:] = np.inf
        x[1, 3, :, 1:] = np.nan
        x[1, [0, 2, 5]] = np.nan
        x[0] = np.nan
    for x in (pre[2], pre[3]):
        x[1, 1, :, P:] = np.nan
        x[1, [0, 2]] = np.inf
    want, tol = attention64(q, H, pre, 1, P, kv, 0, 1, seq, hold)
    for most in (190, 193):
        c = Call(mk, q, H, pre, 1, P, kv, 0, 1, seq, keys, most)
        print("prefix attention, empty rows", d, most, flush=True)
        c.run()
        got = c.result()
        check(got, want, tol)
        assert (got[[0, 2, 4, 6]] == 0).all()
    for most in (0, 60, 170):
        cut = [min(k, most) for k in hold]
        want, tol = attention64(q, H, pre, 1, P, kv, 0, 1, seq, cut)
        c = Call(mk, q, H, pre, 1, P, kv, 0, 1, seq, keys, most)
        print("prefix attention, bound below", d, most, flush=True)
        c.run()
        check(c.result(), want, tol)


@pytest.mark.parametrize("d", [64, 128])
def test_any_order_and_garbage_beside(mk, d):
    """Tokens of a sequence that do not follow each other, the same token twice, keys in any order; q of padded rows is
    NaN or infinite, and one live token's is: only its own row shows it."""
    rng = np.random.default_rng(5)
    H, KV, P = 8, 2, 150
    q, pre, kv, _, _ = build(rng, H, KV, d, [1] * 20, P, [90] * 20, 0)
    seq = [0, 1, 0, 1, 2, 2, 1, 0, 0, 5, 5, 4, 5, 4, 3, 3, 3, 3, 0, 1]
    keys = [240, 160, 200, 239, 10, 240, 0, 151, 240, 170, 169, 168, 0, 240, 200, 199, 198, 200, 0, 150]
    want, tol = attention64(q, H, pre, 1, P, kv, 0, 1, seq, keys)
    for i, bad in ((6, np.nan), (12, np.inf), (18, -np.inf), (9, np.nan), (15, np.inf)):
        q[i, 3::7] = bad
    c = Call(mk, q, H, pre, 1, P, kv, 0, 1, seq, keys, 240)
    print("prefix attention, any order", d, flush=True)
    c.run()
    got, ok = c.result(), [i for i in range(20) if i not in (9, 15)]
    check(got[ok], want[ok], tol[ok])
    assert (got[[6, 12, 18]] == 0).all() and np.isnan(got[[9, 15]]).any(axis=1).all()


def test_prefix_in_the_same_cache_agrees_with_attention(mk):
    """Sequences that all hold the prefix's rows: mk_attention's results, by another order of the sums."""
    rng = np.random.default_rng(8)
    H, KV, d, P, n = 32, 8, 128, 300, 12
    kv = make_cache(rng, 2, 4, KV, 420, d)
    for x in kv:
        x[:, :, :, :P] = x[:, 2:3, :, :P]
    seq = [t % 4 for t in range(n)]
    keys = [P + 7 * t + 1 for t in range(n)]
    q = rng.standard_normal((n, H * d)).astype(np.float32)
    want, tol = attention64(q, H, kv, 2, P, kv, P, 1, seq, keys)
    c = Call(mk, q, H, kv, 2, P, kv, P, 1, seq, keys, max(keys), same=True)
    print("prefix attention, one cache", flush=True)
    c.run()
    check(c.result(), want, tol)
    out = mk.alloc(n * H * d * 4)
    mk_.check(mk_.load().mk_attention(mk.h, c.q.ptr, H * d, out.ptr, H * d, n, H, ctypes.byref(c.kv), 1, c.seq.ptr,
                                      c.keys.ptr, None, None, max(keys)))
    check(out.download(np.float32).reshape(n, -1), want, tol)


def test_large_scores_and_scales(mk):
    """Scores whose exponentials span the whole range of fp32, very small and very large rows of q, keys and values."""
    rng = np.random.default_rng(5)
    H, KV, d, P = 8, 2, 128, 200
    q, pre, kv, seq, keys = build(rng, H, KV, d, [1, 2, 1], P, [60, 30, 1], 0)
    q[0] *= 40.0
    q[1] *= 1e-20
    q[2] *= 1e10
    q[3, :d] = 0.0
    for c in (pre, kv):
        c[2][:, :, :, ::3] *= np.float32(1e-3)
        c[3][:, :, :, 1::5] *= np.float32(1e8)
        c[3][:, :, 1] *= np.float32(1e-30)
    want, tol = attention64(q, H, pre, 1, P, kv, 0, 0, seq, keys)
    c = Call(mk, q, H, pre, 1, P, kv, 0, 0, seq, keys, max(keys))
    print("prefix attention, wide ranges", flush=True)
    c.run()
    check(c.result(), want, tol)


def test_cache_past_4_gib(mk):
    """Rows of the last sequence of a cache whose offsets pass 32 bits."""
    H, KV, d, ctx, n_seq = 8, 4, 128, 40000, 220
    rng = np.random.default_rng(2)
    pre = make_cache(rng, 1, 1, KV, 40, d)
    small = make_cache(rng, 1, 1, KV, 50, d)
    rows = n_seq * KV * ctx
    assert rows * d > 1 << 32
    big = [mk.alloc(rows * d), mk.alloc(rows * d), mk.alloc(rows * 4), mk.alloc(rows * 4)]
    for g in range(KV):
        at = ((n_seq - 1) * KV + g) * ctx + ctx - 50
        for b, x, size in zip(big, small, (d, d, 4, 4)):
            b.upload(x[0, 0, g], at * size)
    q = rng.standard_normal((3, H * d)).astype(np.float32)
    want, tol = attention64(q, H, pre, 0, 40, small, 0, 0, [0] * 3, [41, 63, 90])
    c = Call(mk, q, H, pre, 0, 40, small, 0, 0, [n_seq - 1] * 3, [41, 63, 90], 90)
    c.kv = mk_.MkKvCache(*(b.p for b in big), 1, n_seq, KV, d, ctx)
    c.args = c.args[:10] + (ctypes.byref(c.kv), ctx - 50) + c.args[12:]
    print("prefix attention, large cache", flush=True)
    c.run()
    check(c.result(), want, tol)
    for b in big:
        b.free()


def test_captured_and_replayed(mk):
    """Two calls captured into one graph, with a workspace each; the lengths grow between the replays."""
    hip = ctypes.CDLL("libamdhip64.so")
    rng = np.random.default_rng(9)
    H, KV, d, P, most = 8, 2, 128, 300, 420
    calls = []
    for i in range(2):
        q, pre, kv, seq, _ = build(rng, H, KV, d, [1] * 6, P, [most - P] * 6, 0)
        calls.append((Call(mk, q, H, pre, 1, P, kv, 0, 1, seq, [P + 1] * 6, most), q, pre, kv, seq))
    stream = ctypes.c_void_p(mk_.load().mk_stream(mk.h))
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    mk.sync()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    for c, *_ in calls:
        c.run()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
    for i in range(4):
        keys = [[0, P - 5, P + 1 + 30 * i, P + 17 * i + 2, most - i, 9][j] for j in range(6)]
        for c, *_ in calls:
            c.keys.upload(np.asarray(keys, np.int32))
        print("replay", i, flush=True)
        assert hip.hipGraphLaunch(run, stream) == 0
        for c, q, pre, kv, seq in calls:
            want, tol = attention64(q, H, pre, 1, P, kv, 0, 1, seq, keys)
            got = c.result()
            check(got, want, tol)
            c.run()  # eager, between the replays
            assert np.array_equal(got.view(np.uint32), c.result().view(np.uint32))
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:3]) + f"-n{sum(c[3])}-p{c[4]}")
def test_close_as_a_whole(mk, case):
    """The error of every row of the output is as small as sums in fp32 leave it."""
    H, KV, d, new, P, rows, row0 = case
    rng = np.random.default_rng(sum(new) + P + 1)
    q, pre, kv, seq, keys = build(rng, H, KV, d, new, P, rows, row0)
    want, tol = attention_norms64(q, H, pre, 1, P, kv, row0, 1, seq, keys)
    c = Call(mk, q, H, pre, 1, P, kv, row0, 1, seq, keys, max(keys))
    print("prefix attention as a whole", case[:5], flush=True)
    c.run()
    off = np.sqrt(((c.result().reshape(want.shape) - want) ** 2).sum(-1))
    assert (off <= tol).all(), (off / tol).max()
