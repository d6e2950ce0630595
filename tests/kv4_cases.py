"""Plain 64-bit forms of the 4-bit cache's operators and of the beam selection, in numpy, with what the kernels' sums may be off
by, and a cache on the device, which the GPU tests share."""
import ctypes

import numpy as np

import malkin_amd as mk_

EPS = 2.0 ** -24  # half a step of fp32, relative
GROUP = 32


# ---- numbers in 4 bits ----

def scale_of(x):
    """fp16 scales of groups x [..., 32], as the header has them: exact in every step before the last two roundings."""
    hi, lo = x.max(-1), x.min(-1)
    s = np.clip(np.where(hi >= -lo, hi, lo).astype(np.float64) * -0.125, -4096, 4096)
    u = s.view(np.uint64)
    half = np.uint64(2 ** 44 - 1)  # 8 significant bits, ties to even
    u = (u + half + (u >> np.uint64(45) & np.uint64(1))) & ~np.uint64(2 ** 45 - 1)
    return u.view(np.float64).astype(np.float32).astype(np.float16)


def in4(x):
    """Rows [..., d] as numbers 0..15 and scales: quotients in 64 bits, which are exact beside their borders."""
    g = np.where(np.isnan(x), 0, x).astype(np.float64).reshape(*x.shape[:-1], -1, GROUP)
    s = scale_of(g)
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where((s == 0)[..., None], 0, np.rint(g / s.astype(np.float64)[..., None]))
    n = (np.clip(y, -8, 7) + 8).astype(np.uint8)
    return n.reshape(x.shape), s


def values64(n, s):
    """What the numbers stand for: s (n - 8), which fp16 rounds only where s has more than the 8 bits that are written."""
    v = ((n.astype(np.float64) - 8).reshape(*n.shape[:-1], -1, GROUP) * s.astype(np.float64)[..., None]).reshape(n.shape)
    return v.astype(np.float16).astype(np.float64)


def packed(n):
    return n[..., 0::2] | n[..., 1::2] << 4


def unpacked(b):
    return np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)


# ---- a cache ----

class Cache:
    """The arrays on the host, in the device's layout; put() makes their copies on the device."""

    def __init__(self, rng, n_layer, n_page, page, kv, d, n_seq, max_pages):
        self.shape = (n_layer, n_page, page, kv, d, n_seq, max_pages)
        self.a = {}
        for x in "kv":
            n, s = in4(rng.standard_normal((n_page, n_layer, kv, page, d)).astype(np.float32))
            self.a[x] = packed(n)
            self.a[x + "_scale"] = s if x == "k" else np.ascontiguousarray(np.swapaxes(s, -1, -2))
        self.a["table"] = np.full((n_seq, max_pages), -1, np.int32)
        self.a["len"] = np.zeros(n_seq, np.int32)
        self.a["refs"] = np.zeros(n_page, np.int32)

    def hold(self, seq, pages, rows):
        """Sequence seq holds `rows` rows in `pages` (host side, before put)."""
        self.a["table"][seq, :len(pages)] = pages
        self.a["len"][seq] = rows
        np.add.at(self.a["refs"], np.asarray(pages, int), 1)

    def fill(self, rng, rows):
        """Sequence i holds rows[i] rows in pages from all over the pool."""
        page, order = self.shape[2], list(rng.permutation(self.shape[1]))
        for i, r in enumerate(rows):
            self.hold(i, [order.pop() for _ in range(-(-r // page))], r)

    def put(self, mk):
        self.mk = mk
        self.b = {x: mk.to_device(v) for x, v in self.a.items()}
        n_layer, n_page, page, kv, d, n_seq, max_pages = self.shape
        self.c = mk_.MkKv4Cache(*(self.b[x].p for x in ("k", "v", "k_scale", "v_scale", "table", "len", "refs")), n_layer,
                                n_page, page, kv, d, n_seq, max_pages)
        return self

    @property
    def ref(self):
        return ctypes.byref(self.c)

    def get(self, *names):
        r = [self.b[x].download(self.a[x].dtype).reshape(self.a[x].shape) for x in names]
        return r if len(r) > 1 else r[0]

    def rows(self, side, layer, seq, g, count, a=None):
        """The first `count` rows of a sequence as 64-bit values, and whether each has a page."""
        a, page = a or self.a, self.shape[2]
        j = np.arange(count)
        p = a["table"][seq, j // page]
        ok = (p >= 0) & (p < self.shape[1])
        p = np.where(ok, p, 0)
        n = unpacked(a[side][p, layer, g, j % page])
        s = a["k_scale"][p, layer, g, j % page] if side == "k" else a["v_scale"][p, layer, g, :, j % page]
        return values64(n, s), ok


# ---- rotation ----

def frequencies64(dim, scaling, base, factor, n_orig=0, beta=(32.0, 1.0), attn=0.0, divide=None):
    """Radians per position of each pair, and the factor of cosines and sines."""
    i = np.arange(dim // 2)
    if scaling == mk_.ROPE_NTK:
        base *= factor ** (dim / (dim - 2))
    f = base ** (-2.0 * i / dim)
    if divide is not None:
        f = f / divide.astype(np.float64)
    if scaling == mk_.ROPE_LINEAR:
        f = f / factor
    if scaling != mk_.ROPE_YARN:
        return f, 1.0
    lo, hi = (dim * np.log(n_orig / (2 * np.pi * b)) / (2 * np.log(base)) for b in beta)
    lo, hi = max(np.floor(lo), 0), min(np.ceil(hi), dim - 1)
    ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
    return f / factor * ramp + f * (1 - ramp), attn if attn else 0.1 * np.log(factor) + 1


def rotated64(x, cos, sin, pairs):
    """x [..., d], cos / sin [..., r]: the first 2 r elements of every row."""
    y, r = x.copy(), cos.shape[-1]
    a, b = (np.arange(0, 2 * r, 2), np.arange(1, 2 * r, 2)) if pairs else (np.arange(r), np.arange(r, 2 * r))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


# ---- attention ----

def attention64(cache, layer, q, n_head, seq, keys):
    """Outputs [n][n_head][d], a bound of every value's error, and one of a row's 2-norm.

    Bound: a score is 2 d products (q in two parts of 2^-23 of a value, or 2^-38 of the row's largest where lo is subnormal) and
    two more roundings, so off by at most (2 d + 8) EPS of the sum of their sizes A; that and the rounding of score - shift go
    into p, the hardware's power of two by 2 EPS; the sums over keys add two roundings a key, rescaling the running shift
    another. A weight's parts leave 2^-23 of it, or 2^-25 where lo is subnormal, when the largest was 2^10 (scores past 2^24:
    1) at the time its shift was set: at most 2^-34 of the largest weight.

    Norm: roundings are independent of each other: a sum of L terms walks to half a step times the root of L times the root of
    the terms' squares. A q or weights with the lo part missing, or a key left out, are ten times and more beyond it."""
    n_layer, n_page, page, KV, d, n_seq, max_pages = cache.shape
    G = n_head // KV
    out = np.zeros((len(seq), n_head, d))
    tol, norm = np.zeros_like(out), np.zeros((len(seq), n_head))
    for t in range(len(seq)):
        m = int(keys[t]) if 0 <= seq[t] < n_seq else 0
        if m <= 0:
            continue
        for g in range(KV):
            K, ok = cache.rows("k", layer, seq[t], g, m)
            V, _ = cache.rows("v", layer, seq[t], g, m)
            K, V = K[ok], V[ok]
            if not len(K):
                continue
            for h in range(g * G, (g + 1) * G):
                x = q[t, h * d:(h + 1) * d].astype(np.float64)
                s = K @ x / np.sqrt(d)
                A = np.abs(K) @ (np.abs(x) + 2.0 ** -14 * np.abs(x).max()) / np.sqrt(d)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, h] = p @ V
                span = s.max() - s.min()
                rel = 2 * ((2 * d + 8) * A.max() + 4 * span + 16) + 4 * len(K)
                rest = 2.0 ** -34 if np.abs(s).max() < 2.0 ** 23 else 2.0 ** -24
                tol[t, h] = EPS * rel * (p @ np.abs(V)) + len(K) * rest * p.max() * np.abs(V).max(0)
                B = np.sqrt((K ** 2 @ x ** 2).max() / d)
                S, walk = np.sqrt((p ** 2 @ V ** 2).sum()), 2 * np.sqrt(len(K))
                norm[t, h] = EPS * ((2 * np.sqrt(2 * d) * B + 4 * span + 32 + walk) * S + walk * np.sqrt((out[t, h] ** 2).sum()))
    return out, tol, norm


# ---- pages, one entry after the other ----

def pages_for(rows, page):
    return -(-rows // page)


def fork_model(a, page, dst, src):
    """a: dict of table, len, refs (changed in place)."""
    n_seq = len(a["len"])
    old_t, old_l = a["table"].copy(), a["len"].copy()
    last = {}
    for i, s in enumerate(src):
        d = i if dst is None else int(dst[i])
        if 0 <= d < n_seq:
            last[d] = int(s)
    for d, s in last.items():
        for p in old_t[d][old_t[d] >= 0]:
            a["refs"][p] -= 1
        a["table"][d], a["len"][d] = (old_t[s], old_l[s]) if 0 <= s < n_seq else (-1, 0)
        for p in a["table"][d][a["table"][d] >= 0]:
            a["refs"][p] += 1


def resize_model(a, page, seq, new_len):
    """Statuses; copies (source, destination, rows)."""
    n_seq, room = len(a["len"]), a["table"].shape[1] * page
    seq = list(range(len(new_len))) if seq is None else [int(s) for s in seq]
    status, copies, todo = [0] * len(new_len), [], []
    for i, (s, L) in enumerate(zip(seq, new_len)):
        if not 0 <= s < n_seq or not 0 <= L <= room or s in seq[i + 1:]:
            status[i] = -1
        elif L > a["len"][s]:
            todo.append(i)
        else:
            for j in range(pages_for(L, page), pages_for(a["len"][s], page)):
                a["refs"][a["table"][s, j]] -= 1
                a["table"][s, j] = -1
            a["len"][s] = L
    free = [int(p) for p in np.flatnonzero(a["refs"] <= 0)]
    used, before = 0, {}
    holders = {i: a["refs"][a["table"][seq[i], a["len"][seq[i]] // page]] if a["len"][seq[i]] % page else 0 for i in todo}
    for i in todo:
        s, L, have = seq[i], int(new_len[i]), int(a["len"][seq[i]])
        p = int(a["table"][s, have // page]) if have % page else -1
        copy = p >= 0 and before.get(p, 0) < holders[i] - 1
        before[p] = before.get(p, 0) + 1
        need = int(copy) + pages_for(L, page) - pages_for(have, page)
        first, used = used, used + need
        if need and used > len(free):
            status[i] = 1
            continue
        mine = free[first:used]
        if copy:
            copies.append((p, mine[0], have % page))
            a["table"][s, have // page] = mine[0]
            a["refs"][p] -= 1
            a["refs"][mine[0]] += 1
            mine = mine[1:]
        for j, x in enumerate(mine):
            a["table"][s, pages_for(have, page) + j] = x
            a["refs"][x] += 1
        a["len"][s] = L
    return status, copies


def compact_model(a):
    live = a["refs"] > 0
    n = int(live.sum())
    holes, movers = np.flatnonzero(~live[:n]), n + np.flatnonzero(live[n:])
    to = np.arange(len(live))
    to[movers] = holes
    a["table"][:] = np.where(a["table"] >= 0, to[a["table"]], -1)
    a["refs"][holes] = a["refs"][movers]
    a["refs"][movers] = 0
    return n, [(int(s), int(d), None) for s, d in zip(movers, holes)]


def copied(a, moves, page):
    """The rows that moves copy, in host arrays, all at once."""
    src = {x: a[x].copy() for x in ("k", "v", "k_scale", "v_scale")}
    for s, d, rows in moves:
        r = page if rows is None else rows
        for x in ("k", "v", "k_scale"):
            a[x][d, :, :, :r] = src[x][s, :, :, :r]
        a["v_scale"][d, :, :, :, :r] = src["v_scale"][s, :, :, :, :r]


# ---- beams ----

def beams64(logits, scores, done, eos, beams, k):
    """Per group: (score, row, token) of the k best, and how far apart neighbours of other beams are at least."""
    out, gap = [], np.inf
    for first in range(0, len(logits), beams):
        best = []
        for i in range(first, first + beams):
            start = float(scores[i])
            if not np.isfinite(start):
                continue
            if done is not None and done[i]:
                best.append((start, i, 0.0, int(eos)))
                continue
            z = np.where(np.isnan(logits[i]), -np.inf, np.minimum(logits[i].astype(np.float64), np.finfo(np.float32).max))
            if z.max() == -np.inf:
                continue
            lse = z.max() + np.log(np.exp(z - z.max()).sum())
            order = np.lexsort((np.arange(len(z)), -z))[:k]
            best += [(z[v] - lse + start, i, z[v], int(v)) for v in order if z[v] > -np.inf]
        best.sort(key=lambda e: (-e[0], e[1], -e[2], e[3]))
        for a, b in zip(best[:k], best[1:k + 1]):
            if a[1] != b[1]:
                gap = min(gap, a[0] - b[0])
        best = [(e[0], e[1], e[3]) for e in best[:k]]
        out.append(best + [(-np.inf, -1, -1)] * (k - len(best)))
    return out, gap
