"""The 4-bit cache in pages on the device: rotary tables, norm + rotation + write, rows read back, and attention over it, against
64-bit forms: decoding, chains of drafts, prompts, pages of every size, tokens without keys, pages that are not there, rows that
nothing was written to, strides, pools past 2^32 bytes, captured graphs."""
import ctypes

import numpy as np
import pytest

import malkin_amd as mk_
from kv4_cases import EPS, Cache, attention64, frequencies64, in4, packed, rotated64, unpacked, values64

pytestmark = pytest.mark.gpu


# ---- tables ----

@pytest.mark.parametrize("dim,scaling,base,factor,n_orig,first,n,attn", [
    (128, mk_.ROPE_PLAIN, 1e6, 1.0, 0, 0, 1, 0.0),
    (128, mk_.ROPE_PLAIN, 1e4, 1.0, 0, 2 ** 31 - 300, 300, 0.0),
    (2, mk_.ROPE_LINEAR, 1e4, 8.0, 0, 5, 77, 0.0),
    (64, mk_.ROPE_NTK, 1e6, 3.7, 0, 1000, 501, 0.0),
    (128, mk_.ROPE_YARN, 1e6, 4.0, 32768, 131000, 400, 0.0),
    (94, mk_.ROPE_YARN, 1e4, 16.0, 4096, 0, 999, 1.25),
    (256, mk_.ROPE_YARN, 5e5, 2.5, 600, 7, 33, 0.0),
])
@pytest.mark.parametrize("divided", [False, True])
def test_tables(mk, dim, scaling, base, factor, n_orig, first, n, attn, divided):
    rng = np.random.default_rng(dim + n)
    div = (1 + 7 * rng.random(dim // 2)).astype(np.float32) if divided else None
    rope = mk_.MkRope(dim, scaling, base, factor, n_orig, 32.0, 1.0, attn)
    cos, sin = (mk.to_device(np.full(n * (dim // 2) + 5, 9.0, np.float32)) for _ in range(2))
    d = mk.to_device(div) if divided else None
    mk_.check(mk_.load().mk_rope_tables(mk.h, ctypes.byref(rope), d.ptr if d else None, first, n, cos.ptr, sin.ptr))
    f, m = frequencies64(dim, scaling, base, factor, n_orig, attn=attn, divide=div)
    pos = (first + np.arange(n, dtype=np.float64))[:, None]
    # The angle in turns is rounded in 64 bits (of up to pos f of them, twice on each side), brought to an eighth of a turn and
    # to 32 bits there (half a step of at most pi / 4); the series adds a few half steps of 1, the factor one.
    tol = m * (2 * np.pi * 4 * 2.0 ** -53 * pos * f / (2 * np.pi) * 4 + 8 * EPS)
    for buf, want in ((cos, np.cos(pos * f) * m), (sin, np.sin(pos * f) * m)):
        got = buf.download(np.float32)
        assert (got[n * (dim // 2):] == 9.0).all()
        assert (np.abs(got[:n * (dim // 2)].reshape(n, -1) - want) <= tol).all()


# ---- norm, rotation, write ----

def write_call(mk, c, x, H, norm, layout, rope_dim, cos, sin, rpos, seq, row, layer=1, in_place=False, pad=0, eps=1e-6):
    n_layer, n_page, page, KV, d, n_seq, max_pages = c.shape
    n, width = len(seq), (H + 2 * KV) * d
    wide = np.full((n, width + pad), 7.0, np.float32)
    wide[:, :width] = x
    up = mk.to_device
    b = dict(x=up(wide), cos=up(cos), sin=up(sin), rpos=up(np.asarray(rpos, np.int32)), seq=up(np.asarray(seq, np.int32)),
             row=up(np.asarray(row, np.int32)), q=up(np.full((n, H * d + pad), 3.0, np.float32)),
             norm=up(np.stack(norm)) if norm is not None else None)
    at = b["x"].offset
    q_out, stride = (b["x"].ptr, width + pad) if in_place else (b["q"].ptr, H * d + pad)
    mk_.check(mk_.load().mk_rope_kv4(
        mk.h, b["x"].ptr, at(4 * H * d), at(4 * (H + KV) * d), width + pad, n, H, b["norm"].ptr if norm is not None else None,
        b["norm"].offset(4 * d) if norm is not None else None, eps, layout, rope_dim, b["cos"].ptr, b["sin"].ptr, len(cos),
        b["rpos"].ptr, b["seq"].ptr, b["row"].ptr, c.ref, layer, q_out, stride))
    after = b["x"].download(np.float32).reshape(n, -1)
    q = after if in_place else b["q"].download(np.float32).reshape(n, -1)
    assert (after[:, width:] == 7.0).all() and (in_place or np.array_equal(after.view(np.uint32), wide.view(np.uint32)))
    return q


WRITES = [  # heads, KV heads, head_dim, page, rope_dim, layout, norm, pad, in place
    (4, 2, 128, 16, 128, mk_.ROPE_HALVES, True, 0, False),
    (16, 8, 128, 32, 64, mk_.ROPE_HALVES, True, 3, True),
    (3, 1, 64, 64, 64, mk_.ROPE_PAIRS, False, 1, False),
    (8, 8, 64, 128, 38, mk_.ROPE_HALVES, True, 2, False),
    (5, 5, 128, 1024, 26, mk_.ROPE_PAIRS, True, 0, True),
    (2, 2, 128, 16, 0, mk_.ROPE_HALVES, False, 0, False),
    (40, 8, 128, 64, 80, mk_.ROPE_HALVES, False, 0, False),
    (40, 8, 128, 64, 128, mk_.ROPE_PAIRS, True, 0, False),
    (25, 8, 64, 256, 64, mk_.ROPE_HALVES, True, 3, True),
]


@pytest.mark.parametrize("case", WRITES, ids=str)
@pytest.mark.parametrize("n", [1, 37, 1300])
def test_write(mk, case, n):
    H, KV, d, page, rope_dim, layout, norm, pad, in_place = case
    rng = np.random.default_rng(H + d + n)
    n_seq, max_pages = 4, 6 if page < 256 else 2
    c = Cache(rng, 2, n_seq * max_pages + 1, page, KV, d, n_seq, max_pages)
    c.fill(rng, [max_pages * page - 3, page + 1, 2 * page, 1])
    c.put(mk)
    at = [(s, r) for s in range(n_seq) for r in range(c.a["len"][s])]
    at = [at[i] for i in rng.permutation(len(at))[:n]]
    n = len(at)
    seq, row = [list(v) for v in zip(*at)]
    n_pos = 50
    rpos = list(rng.integers(0, n_pos, n))
    skipped = []
    if n > 10:  # rows that are left out: no sequence, no such position, no page
        seq[1], seq[3], rpos[4], rpos[6] = -1, n_seq, n_pos, -5
        seq[8], row[8] = 3, page + 2
        row[9] = -1
        row[11], seq[11] = max_pages * page, 0
        skipped = [1, 3, 4, 6, 8, 9, 11]
    x = rng.standard_normal((n, (H + 2 * KV) * d)).astype(np.float32)
    x[:, ::61] *= 5
    cos = rng.standard_normal((n_pos, max(1, rope_dim // 2))).astype(np.float32)
    sin = rng.standard_normal(cos.shape).astype(np.float32)
    w = [(1 + 0.2 * rng.standard_normal(d)).astype(np.float32) for _ in range(2)] if norm else None
    print("kv4 write", case, n, flush=True)
    q = write_call(mk, c, x, H, w, layout, rope_dim, cos, sin, rpos, seq, row, 1, in_place, pad)
    live = [t for t in range(n) if t not in skipped]
    y = x.astype(np.float64).reshape(n, H + 2 * KV, d)
    err = np.zeros_like(y)
    if norm:
        s = 1 / np.sqrt((y[:, :H + KV] ** 2).mean(-1, keepdims=True) + 1e-6)
        y[:, :H] *= s[:, :H] * w[0]
        y[:, H:H + KV] *= s[:, H:] * w[1]
        err[:, :H + KV] = (d / 8 + 16) * EPS * np.abs(y[:, :H + KV])  # a lane's sum, the lanes', the root and two products
    if rope_dim:
        pos = np.clip(rpos, 0, n_pos - 1)
        args = cos[pos, None, :rope_dim // 2].astype(np.float64), sin[pos, None, :rope_dim // 2].astype(np.float64)
        size = rotated64(np.abs(y[:, :H + KV]) * EPS * 4 + err[:, :H + KV], *[np.abs(a) for a in args], layout == mk_.ROPE_PAIRS)
        minus = rotated64(np.abs(y[:, :H + KV]) * EPS * 4 + err[:, :H + KV], np.abs(args[0]), -np.abs(args[1]), layout == mk_.ROPE_PAIRS)
        y[:, :H + KV] = rotated64(y[:, :H + KV], *args, layout == mk_.ROPE_PAIRS)
        err[:, :H + KV] = np.maximum(np.abs(size), np.abs(minus))
    got = q[:, :H * d].reshape(n, H, d)
    assert (np.abs(got[live] - y[live, :H]) <= err[live, :H] + EPS * np.abs(y[live, :H])).all()
    if skipped:
        assert (got[skipped] == (x.reshape(n, -1, d)[skipped, :H] if in_place else 3.0)).all()
    # The cache: everything but the rows written is as it was; those hold the values to half a step of their scale.
    new = dict(zip(("k", "v", "k_scale", "v_scale"), c.get("k", "v", "k_scale", "v_scale")))
    want = {i: v.copy() for i, v in c.a.items()}
    for t in live:
        p, r = c.a["table"][seq[t], row[t] // page], row[t] % page
        for side, h0 in (("k", H), ("v", H + KV)):
            for g in range(KV):
                s = new["k_scale"][p, 1, g, r] if side == "k" else new["v_scale"][p, 1, g, :, r]
                num = unpacked(new[side][p, 1, g, r])
                v, e = y[t, h0 + g], err[t, h0 + g]
                if side == "v":  # its input is what was given: every bit follows
                    num_w, s_w = in4(x[t, (h0 + g) * d:(h0 + g + 1) * d])
                    assert np.array_equal(num, num_w) and np.array_equal(s.view(np.uint16), s_w.view(np.uint16))
                grp = v.reshape(-1, 32)
                m = np.abs(grp).max(-1)
                slack = e.reshape(-1, 32).max(-1)
                assert (np.abs(np.abs(s.astype(np.float64)) - m / 8) <= 2.0 ** -8 * m / 8 + slack / 8 + 2.0 ** -25).all()
                steps = grp / s.astype(np.float64)[:, None]
                far = np.abs(np.clip(steps, -8, 7) - (num.reshape(-1, 32).astype(np.float64) - 8))
                assert (far <= 0.5 + (np.abs(steps) * 4 * EPS + (e.reshape(-1, 32) / np.abs(s.astype(np.float64))[:, None]))).all()
                want[side][p, 1, g, r] = new[side][p, 1, g, r]
                if side == "k":
                    want["k_scale"][p, 1, g, r] = s
                else:
                    want["v_scale"][p, 1, g, :, r] = s
    for name, v in new.items():
        assert np.array_equal(v.view(np.uint8), want[name].view(np.uint8)), name


@pytest.mark.parametrize("layout,norm,d", [(mk_.ROPE_HALVES, True, 128), (mk_.ROPE_PAIRS, False, 64)])
def test_numbers_beside_borders(mk, layout, norm, d):
    """A million numbers of K, each the one that 64 bits give: a rounding of 2^-52 turns one in 10^12, one of 2^-23 some of these."""
    rng = np.random.default_rng(d)
    H, KV, page, n, n_pos = 1, 8 * 128 // d, 64, 1024, 64
    c = Cache(rng, 1, n // page, page, KV, d, 1, n // page)
    c.hold(0, list(rng.permutation(n // page)), n)
    c.put(mk)
    x = rng.standard_normal((n, (H + 2 * KV) * d)).astype(np.float32)
    turn = rng.random((n_pos, d // 2)) * 2 * np.pi
    cos, sin = np.cos(turn).astype(np.float32), np.sin(turn).astype(np.float32)
    w = [(1 + 0.2 * rng.standard_normal(d)).astype(np.float32) for _ in range(2)] if norm else None
    rpos = rng.integers(0, n_pos, n)
    print("kv4 write, borders", layout, norm, d, flush=True)
    write_call(mk, c, x, H, w, layout, d, cos, sin, list(rpos), [0] * n, list(range(n)), 0)
    k = x.reshape(n, -1, d)[:, H:H + KV].astype(np.float64)
    if norm:
        k *= w[1] / np.sqrt((k ** 2).mean(-1, keepdims=True) + np.float64(np.float32(1e-6)))
    num, s = in4(rotated64(k, cos[rpos, None].astype(np.float64), sin[rpos, None].astype(np.float64), layout == mk_.ROPE_PAIRS))
    kd, sd = c.get("k", "k_scale")
    p, r = c.a["table"][0, np.arange(n) // page], np.arange(n) % page
    assert np.array_equal(sd[p, 0, :, r].view(np.uint16), s.reshape(n, KV, -1).view(np.uint16))
    assert np.array_equal(unpacked(kd[p, 0, :, r]), num)


def test_values_at_the_edges(mk):
    """Zeros, the smallest and the largest values, infinities and NaN, extremes of both signs, ties of a half."""
    rng = np.random.default_rng(1)
    d, KV, n = 64, 1, 12
    x = rng.standard_normal((n, 3 * d)).astype(np.float32)
    v = x[:, 2 * d:]
    v[0] = 0
    v[1] = -0.0
    v[2] *= 1e-7
    v[3] = 1e-42
    v[4, :32] = np.nan
    v[4, 32] = np.inf
    v[5, 3] = -np.inf
    v[6] *= 1e30
    v[7, :32] = np.where(np.arange(32) % 2, 2.0, -2.0)
    v[8, :32] = np.arange(32) / 8.0 - 2.0  # m = -2: steps of 0.25, halves between
    v[9, 5], v[9, 6] = np.nan, 40000.0
    v[10] = 3.0
    v[11, :32] = -np.arange(32) * np.float32(2.0 ** -24)
    x[:, :d] = 1
    x[:, d:2 * d] = v
    c = Cache(rng, 1, 3, 16, KV, d, 1, 2)
    c.hold(0, [2, 0], 20)
    c.put(mk)
    one = np.ones((1, 1), np.float32)
    print("kv4 write, edges", flush=True)
    write_call(mk, c, x, 1, None, mk_.ROPE_HALVES, 0, one, one, [0] * n, [0] * n, list(range(4, 4 + n)), 0)
    num, s = in4(v)
    with np.errstate(invalid="ignore"):
        assert np.isfinite(values64(num, s)).all()
    ko, vo = mk.alloc(2 * n * d), mk.alloc(2 * n * d)
    seq, row = mk.to_device(np.zeros(n, np.int32)), mk.to_device(np.arange(4, 4 + n, dtype=np.int32))
    mk_.check(mk_.load().mk_kv4_rows(mk.h, c.ref, 0, seq.ptr, row.ptr, n, ko.ptr, vo.ptr))
    for b in (ko, vo):
        assert np.array_equal(b.download(np.float16).reshape(n, d).astype(np.float64), values64(num, s))


@pytest.mark.parametrize("d,page,KV", [(128, 16, 8), (64, 256, 3)])
def test_rows(mk, d, page, KV):
    rng = np.random.default_rng(d)
    c = Cache(rng, 3, 9, page, KV, d, 3, 4)
    c.fill(rng, [4 * page, page + 3, 0])
    c.a["table"][0, 1] = 9  # not in the pool
    c.put(mk)
    seq = [0, 0, 1, 2, -1, 3, 1, 0, 0]
    row = [0, 4 * page - 1, page + 2, 0, 0, 0, -1, page, 4 * page]
    n = len(seq)
    up = [mk.to_device(np.asarray(v, np.int32)) for v in (seq, row)]
    out = [mk.to_device(np.full(n * KV * d, 5.0, np.float16)) for _ in range(2)]
    mk_.check(mk_.load().mk_kv4_rows(mk.h, c.ref, 2, up[0].ptr, up[1].ptr, n, out[0].ptr, out[1].ptr))
    for b, side in zip(out, "kv"):
        got = b.download(np.float16).reshape(n, KV, d).astype(np.float64)
        for i in range(n):
            for g in range(KV):
                want = np.zeros(d)
                if i < 3:
                    want = c.rows(side, 2, seq[i], g, row[i] + 1)[0][row[i]]
                assert np.array_equal(got[i, g], want)
    # One side alone.
    mk_.check(mk_.load().mk_kv4_rows(mk.h, c.ref, 1, up[0].ptr, up[1].ptr, n, None, out[0].ptr))
    got = out[0].download(np.float16).reshape(n, KV, d).astype(np.float64)
    assert np.array_equal(got[1, KV - 1], c.rows("v", 1, 0, KV - 1, 4 * page)[0][-1])


# ---- attention ----

class Call:
    """Inputs of one call on the device; run() queues it."""

    def __init__(self, mk, c, q, H, layer, seq, keys, most, run, pad=0, q8=False):
        n_layer, n_page, page, KV, d, n_seq, max_pages = c.shape
        self.mk, self.c, self.n, self.H, self.HD, self.stride = mk, c, len(seq), H, H * d, H * d + pad
        wide = np.full((self.n, self.stride), 7.0, np.float32)
        wide[:, :self.HD] = q
        self.q, self.out = mk.to_device(wide), mk.to_device(np.full((self.n, self.stride), 3.0, np.float32))
        self.seq, self.keys = (mk.to_device(np.asarray(x, np.int32)) for x in (seq, keys))
        self.xq = mk.to_device(np.zeros(self.n * self.HD // 32 * 40, np.uint8)) if q8 else None
        self.need = mk_.load().mk_attention_kv4_workspace(self.n, H, KV, d, most, run)
        self.work = mk.to_device(np.full(max(self.need, 16) + 64, 0xA5, np.uint8))
        self.args = (mk.h, self.q.ptr, self.stride, self.out.ptr, self.stride, self.n, H, c.ref, layer, self.seq.ptr,
                     self.keys.ptr, most, run, self.xq.ptr if q8 else None, self.work.ptr, self.need)

    def run(self):
        mk_.check(mk_.load().mk_attention_kv4(*self.args))

    def result(self):
        o = self.out.download(np.float32).reshape(self.n, self.stride)
        assert (o[:, self.HD:] == 3.0).all()  # what lies between rows is left as it was
        assert (self.work.download(np.uint8)[max(self.need, 16):] == 0xA5).all()
        return o[:, :self.HD]


def check(got, want, norm=True, rows=None):
    out, tol, norms = want
    got = got.reshape(out.shape)
    rows = range(len(out)) if rows is None else rows
    for t in rows:
        bad = ~(np.abs(got[t] - out[t]) <= tol[t])
        assert not bad.any(), (t, np.argwhere(bad)[:5], got[t][bad][:5], out[t][bad][:5], tol[t][bad][:5])
        if norm:
            off = np.sqrt(((got[t] - out[t]) ** 2).sum(-1))
            assert (off <= norms[t]).all(), (t, off / np.maximum(norms[t], 1e-300))


# heads, KV heads, head_dim, page, tokens of each sequence, rows that the last token of each sees
CASES = [
    (4, 2, 128, 16, [1], [1]),
    (4, 2, 64, 16, [1, 1], [1, 2]),
    (8, 8, 128, 32, [1, 1, 1], [5, 64, 65]),
    (32, 8, 128, 64, [1] * 8, [1, 17, 63, 64, 65, 127, 128, 400]),
    (40, 8, 128, 16, [5, 5, 1, 3], [40, 7, 1, 300]),
    (8, 2, 64, 128, [3, 1, 9], [50, 2, 700]),
    (16, 1, 128, 32, [2, 1], [90, 33]),
    (32, 1, 64, 16, [1, 2], [41, 66]),
    (20, 1, 128, 64, [1, 3], [20, 200]),
    (4, 2, 128, 16, [70, 33], [90, 33]),
    (32, 8, 128, 64, [300], [420]),
    (8, 2, 128, 1024, [200, 1, 150], [1300, 2100, 150]),
    (4, 2, 128, 32, [1] * 40, [1 + 37 * i for i in range(40)]),
    (16, 8, 128, 16, [1, 1], [5000, 3]),
    (8, 8, 64, 32, [770], [1500]),
    (8, 2, 128, 64, [5] * 10, [300 + 131 * i for i in range(10)]),
    (16, 8, 128, 256, [1], [20000]),
    (2, 2, 64, 16, [1] * 300, [1 + i % 37 for i in range(299)] + [2100]),
    (4, 2, 64, 32, [600, 500, 100], [610, 500, 1100]),
    (2, 2, 64, 16, [1] * 300, [1 + i % 41 for i in range(299)] + [3300]),
]


def build(rng, H, KV, d, page, new, rows, n_layer=2):
    n_seq = len(new) + 1
    slots = [(3 * i + 1) % n_seq if n_seq % 3 else i for i in range(len(new))]
    need = [-(-r // page) for r in rows]
    c = Cache(rng, n_layer, sum(need) + 2, page, KV, d, n_seq, max(need) + 1)
    order = list(rng.permutation(sum(need) + 2))
    for s, m, r in zip(slots, need, rows):
        c.hold(s, [order.pop() for _ in range(m)], r)
    seq = [s for s, m in zip(slots, new) for _ in range(m)]
    keys = [r - m + j + 1 for r, m in zip(rows, new) for j in range(m)]
    return c, (1.5 * rng.standard_normal((len(seq), H * d))).astype(np.float32), seq, keys


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:4]) + f"-n{sum(c[4])}-k{max(c[5])}")
def test_attention(mk, case):
    H, KV, d, page, new, rows = case
    rng = np.random.default_rng(sum(new) + max(rows))
    c, q, seq, keys = build(rng, H, KV, d, page, new, rows)
    c.put(mk)
    want = attention64(c, 1, q, H, seq, keys)
    for run, pad, q8 in ((max(new), 0, False), (1, 5, True), (1000, 4, True)):
        print("kv4 attention", case[:4], len(seq), max(rows), run, flush=True)
        call = Call(mk, c, q, H, 1, seq, keys, max(keys), run, pad, q8)
        call.run()
        got = call.result()
        check(got, want)
        if q8:  # the BlockQ8 rows are those of the output
            ref, dense = mk.alloc(call.n * call.HD // 32 * 40), mk.to_device(got)
            mk_.check(mk_.load().mk_quantize_q8(mk.h, dense.ptr, call.n, call.HD, ref.ptr))
            assert np.array_equal(ref.download(np.uint8), call.xq.download(np.uint8))
        call.run()  # again on the same buffers: the same bits
        assert np.array_equal(got.view(np.uint32), call.result().view(np.uint32))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
def test_empty_rows_bad_pages_and_garbage(mk, d, page):
    """Padded rows get zeros; a bound above every n_keys changes nothing but the split, one below cuts; keys without a page have no
    weight; places that no token sees (scales that are NaN or infinite) reach nothing; a row of q that is NaN or infinite shows in
    its own row only."""
    rng = np.random.default_rng(3)
    H, KV = 8, 2
    rows = [190, 70, 151, 40, 9]
    c, q, _, _ = build(rng, H, KV, d, page, [1] * 5, rows)
    live = [s for s in range(6) if c.a["len"][s]]
    a, b, e, f = live[:4]
    seq = [a, b, -1, a, 99, e, e, f, a, a, a, b]
    keys = [0, 7, 20, 150, 160, 1, -4, 30, 149, 151, 90, int(c.a["len"][b])]
    hold = [0, 7, 0, 150, 0, 1, 0, 30, 149, 151, 90, int(c.a["len"][b])]
    c.a["table"][b, 0] = -1 if page == 16 else c.shape[1]  # the first page of one sequence is not there
    for p in range(c.shape[1]):  # rows past what anyone reads
        for s in live:
            for j in np.flatnonzero(c.a["table"][s] == p):
                seen = max([0] + [h for x, h in zip(seq, hold) if x == s]) - j * page
                if seen < page:
                    c.a["k_scale"][p, :, :, max(seen, 0):] = np.nan
                    c.a["v_scale"][p, :, :, :, max(seen, 0):] = np.nan if p % 2 else np.inf
    q = (1.5 * rng.standard_normal((len(seq), H * d))).astype(np.float32)
    clean = q.copy()
    q[2], q[6], q[9, 3::7] = np.nan, np.inf, np.nan
    c.put(mk)
    with np.errstate(invalid="ignore"):
        want = attention64(c, 1, clean, H, seq, hold)
    ok = [t for t in range(len(seq)) if t != 9]
    for most in (190, 193, 192):
        if most > c.shape[6] * page:
            continue
        for run in (1, 3, 500):
            call = Call(mk, c, q, H, 1, seq, keys, most, run)
            print("kv4 attention, empty rows", d, page, most, run, flush=True)
            call.run()
            got = call.result()
            check(got, want, rows=ok)
            assert (got[[0, 2, 4, 6]] == 0).all() and np.isnan(got[9].reshape(H, d)).any()
    if page == 64:
        assert (want[0][1] == 0).all()  # all its keys lie in the page that is not there
    for most in (0, 60, 140):
        with np.errstate(invalid="ignore"):
            want = attention64(c, 1, clean, H, seq, [min(k, most) for k in hold])
        call = Call(mk, c, q, H, 1, seq, keys, most, 3)
        print("kv4 attention, bound below", d, page, most, flush=True)
        call.run()
        check(call.result(), want, rows=ok)


def test_any_order(mk):
    """Tokens of a sequence that do not follow each other, the same token twice, keys in any order within a run."""
    rng = np.random.default_rng(5)
    H, KV, d, page = 8, 2, 128, 32
    c, _, _, _ = build(rng, H, KV, d, page, [1] * 6, [240] * 6)
    seq = [0, 1, 0, 1, 2, 2, 1, 0, 0, 5, 5, 4, 5, 4, 3, 3, 3, 3, 0, 1] + [2] * 70
    keys = [240, 160, 200, 239, 10, 240, 0, 151, 240, 170, 169, 168, 0, 240, 200, 199, 198, 200, 0, 150]
    keys += [int(x) for x in rng.integers(0, 241, 70)]
    held = [s for s in range(7) if c.a["len"][s]]
    seq = [held[s] for s in seq]
    q = (1.5 * rng.standard_normal((len(seq), H * d))).astype(np.float32)
    c.put(mk)
    want = attention64(c, 0, q, H, seq, keys)
    for run in (1, 70):
        call = Call(mk, c, q, H, 0, seq, keys, 240, run)
        print("kv4 attention, any order", run, flush=True)
        call.run()
        check(call.result(), want)


@pytest.mark.parametrize("new", [1, 40])
def test_large_scores(mk, new):
    """Scores whose exponentials span the whole range of fp32 and far past it, very small and very large rows of q, keys, values."""
    rng = np.random.default_rng(5)
    H, KV, d, page = 8, 2, 128, 16
    c, q, seq, keys = build(rng, H, KV, d, page, [new] * 4, [260] * 4)
    for t in range(len(seq)):
        q[t] *= (40.0, 1e-20, 1e10, 3e4)[t % 4]
    q[3, :d] = 0.0
    for x in ("k_scale", "v_scale"):
        c.a[x][::3] *= np.float16(2.0 ** -9)
        c.a[x][1::5] *= np.float16(2.0 ** 9)
    c.put(mk)
    want = attention64(c, 0, q, H, seq, keys)
    call = Call(mk, c, q, H, 0, seq, keys, max(keys), new)
    print("kv4 attention, wide ranges", new, flush=True)
    call.run()
    check(call.result(), want, norm=False)


def test_growing_scores(mk):
    """Every tile's scores far above the last one's, and far below: shifts set again and again."""
    rng = np.random.default_rng(6)
    H, KV, d, page = 4, 1, 128, 16
    for down in (False, True):
        c, q, seq, keys = build(rng, H, KV, d, page, [1, 6], [2000, 1500])
        q = np.abs(q)
        for s in range(c.shape[5]):
            t = c.a["table"][s]
            for j in np.flatnonzero(t >= 0):
                c.a["k"][t[j]] = 0xFF if rng.random() < 0.5 else 0xEE  # all one sign
                level = 0.002 * (len(t) - j if down else j)
                c.a["k_scale"][t[j]] = np.float16(np.round(level * 4096) / 4096)
        c.put(mk)
        want = attention64(c, 0, q, H, seq, keys)
        call = Call(mk, c, q, H, 0, seq, keys, max(keys), 6)
        print("kv4 attention, growing", down, flush=True)
        call.run()
        check(call.result(), want, norm=False)


def test_pool_past_4_gib(mk):
    """Rows of pages whose offsets pass 32 bits, in k, v and (in values) the scales."""
    H, KV, d, page, n_layer = 8, 4, 128, 1024, 4
    rng = np.random.default_rng(2)
    small = Cache(rng, n_layer, 3, page, KV, d, 2, 3)
    small.hold(0, [0, 1], page + 200)
    small.hold(1, [2], 100)
    n_page = 4300
    per = {x: small.a[x][0].nbytes for x in ("k", "v", "k_scale", "v_scale")}
    assert n_page * per["k"] > 1 << 32
    big = {x: mk.alloc(n_page * per[x]) for x in per}
    to = [n_page - 1, n_page - 3, n_page - 2]
    for i, p in enumerate(to):
        for x in per:
            big[x].upload(small.a[x][i], p * per[x])
    table = np.where(small.a["table"] >= 0, np.asarray(to)[small.a["table"]], -1).astype(np.int32)
    tb = mk.to_device(table)
    q = rng.standard_normal((3, H * d)).astype(np.float32)
    seq, keys = [0, 0, 1], [page + 199, page + 200, 77]
    want = attention64(small, 3, q, H, seq, keys)
    small.c = mk_.MkKv4Cache(*(big[x].p for x in ("k", "v", "k_scale", "v_scale")), tb.p, None, None, n_layer, n_page, page, KV,
                             d, 2, 3)
    call = Call(mk, small, q, H, 3, seq, keys, page + 200, 2)
    print("kv4 attention, large pool", flush=True)
    call.run()
    check(call.result(), want)
    # And a write there, read back.
    x = rng.standard_normal((1, (H + 2 * KV) * d)).astype(np.float32)
    one = np.ones((1, 1), np.float32)
    print("kv4 write, large pool", flush=True)
    write_call(mk, small, x, H, None, mk_.ROPE_HALVES, 0, one, one, [0], [0], [page + 7], 3)
    out = [mk.alloc(2 * KV * d) for _ in range(2)]
    up = [mk.to_device(np.asarray([v], np.int32)) for v in (0, page + 7)]
    mk_.check(mk_.load().mk_kv4_rows(mk.h, small.ref, 3, up[0].ptr, up[1].ptr, 1, out[0].ptr, out[1].ptr))
    for b, h0 in zip(out, (H, H + KV)):
        num, s = in4(x[0, h0 * d:(h0 + KV) * d].reshape(KV, d))
        assert np.array_equal(b.download(np.float16).reshape(KV, d).astype(np.float64), values64(num, s))
    for b in big.values():
        b.free()


@pytest.mark.parametrize("most,new", [(420, 1), (3000, 1), (900, 40)])
def test_captured_and_replayed(mk, most, new):
    """Two calls captured into one graph, with a workspace each; the lengths grow between the replays."""
    hip = ctypes.CDLL("libamdhip64.so")
    rng = np.random.default_rng(9)
    H, KV, d, page = 8, 2, 128, 32
    calls = []
    for i in range(2):
        c, q, seq, _ = build(rng, H, KV, d, page, [new] * 6, [most] * 6)
        c.put(mk)
        calls.append((Call(mk, c, q, H, 0, seq, [1] * len(seq), most, new), c, q, seq))
    stream = ctypes.c_void_p(mk_.load().mk_stream(mk.h))
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    calls[0][0].run()
    mk.sync()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    for call, *_ in calls:
        call.run()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
    for i in range(4):
        keys = [[0, most // 3, 1 + 30 * i, 17 * i + 2, most - i, 9][j] for j in range(6)]
        keys = [max(0, k - new + 1 + j) for k in keys for j in range(new)]
        for call, *_ in calls:
            call.keys.upload(np.asarray(keys, np.int32))
        print("kv4 replay", most, new, i, flush=True)
        assert hip.hipGraphLaunch(run, stream) == 0
        for call, c, q, seq in calls:
            got = call.result()
            check(got, attention64(c, 0, q, H, seq, keys))
            call.run()  # eager, between the replays
            assert np.array_equal(got.view(np.uint32), call.result().view(np.uint32))
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
