"""Plain 64-bit forms of the shared-prefix attention, the adapters and the verification, in numpy, and what fp32 sums may
be off by, which the GPU tests share."""
import numpy as np

EPS = 2.0 ** -24  # half a step of fp32, relative


def permuted(d):
    """Byte of element e in a K row of the device cache."""
    e = np.arange(d)
    return d // 16 * (e % 16) + e // 16


def make_cache(rng, n_layer, n_seq, kv, n_ctx, d):
    """k, v (int8), k_scale, v_scale of a device cache with N(0, 1) rows."""
    def side():
        x = rng.standard_normal((n_layer, n_seq, kv, n_ctx, d)).astype(np.float32)
        s = (np.abs(x).max(-1) / 127).astype(np.float32)
        return np.rint(x / s[..., None]).astype(np.int8), s
    (k, ks), (v, vs) = side(), side()
    return k, v, ks, vs


def attention64(q, n_head, pre, pseq, n_prefix, kv, row0, layer, seq, keys):
    """Outputs [n][n_head * d] and their bounds. Every score is a sum of d products (and the scale's two), so it is off by
    at most (d + 8) EPS times the sum of their sizes A; exp turns that, and the rounding of s - m, into a relative error
    of p; the sum over keys adds one rounding per key and side, the running maximum's rescaling another.

    fp16 parts: x = hi + lo to half a step of lo, 2^-12 of 2^-11 of x, or 2^-25 where lo is subnormal. A row of q is
    scaled to a largest value of at least 2^13, so the second adds at most 2^-38 of it to each of its values (to A as
    2^-38 / EPS). The weights p vs are scaled so that the largest of a part was at least 2^6 when the shift was set (its
    rounding aside: 2^5.9), scales below 2^-100 counting as that: a weight is off by at most 2^-30.9 of the largest,
    times a value of at most 127."""
    k, v, ks, vs = kv
    n_seq, KV, d = k.shape[1], k.shape[2], k.shape[4]
    G, byte = n_head // KV, permuted(d)
    out = np.zeros((len(seq), n_head, d))
    tol = np.zeros_like(out)
    for t in range(len(seq)):
        m = int(keys[t]) if 0 <= seq[t] < n_seq else 0
        if m <= 0:
            continue
        a, b = min(m, n_prefix), max(0, m - n_prefix)
        for g in range(KV):
            K, V, S = [], [], []
            for (ck, cv, cks, cvs), i, lo, c in ((pre or kv, pseq, 0, a), (kv, seq[t], row0, b)):
                if c:
                    at = (layer, i, g, slice(lo, lo + c))
                    K.append(ck[at][:, byte].astype(np.float64) * cks[at].astype(np.float64)[:, None])
                    V.append(cv[at].astype(np.float64) * cvs[at].astype(np.float64)[:, None])
                    S.append(cvs[at].astype(np.float64))
            S, K, V = np.concatenate(S), np.concatenate(K), np.concatenate(V)
            for h in range(g * G, (g + 1) * G):
                x = q[t, h * d:(h + 1) * d].astype(np.float64)
                s, A = K @ x / np.sqrt(d), np.abs(K) @ (np.abs(x) + 2.0 ** -14 * np.abs(x).max()) / np.sqrt(d)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, h] = p @ V
                rel = 2 * ((d + 8) * A.max() + 2 * (s.max() - s.min()) + 16) + 4 * m
                W = (p * np.maximum(S, 2.0 ** -100)).max()
                tol[t, h] = EPS * rel * (p @ np.abs(V)) + m * 127 * 2.0 ** -30.9 * W
    return out.reshape(len(seq), -1), tol.reshape(len(seq), -1)


def lora64(x, adapters, ids, base, rows):
    """adapters: (a, b, scale) with a [rank][cols], b [rows][rank] (None: takes no part). Outputs and bounds."""
    y = np.zeros((len(x), rows)) if base is None else base.astype(np.float64)
    tol = np.zeros_like(y)
    for t, i in enumerate(ids):
        if not 0 <= i < len(adapters) or adapters[i] is None:
            continue
        a, b, scale = adapters[i]
        a, b, xt = a.astype(np.float64), b.astype(np.float64), x[t].astype(np.float64)
        delta = float(np.float32(scale)) * (b @ (a @ xt))
        size = abs(float(np.float32(scale))) * (np.abs(b) @ (np.abs(a) @ np.abs(xt)))
        y[t] += delta
        # One rounding per product and sum of both products, the scale's, and the final addition's.
        tol[t] = EPS * ((a.shape[1] + a.shape[0] + 24) * size + np.abs(y[t]))
    return y, tol


def softmax64(z, temp):
    z = np.where(np.isnan(z), -np.inf, np.minimum(z.astype(np.float64), np.finfo(np.float32).max))
    p = np.zeros(len(z))
    m = z.max()
    if m == -np.inf:
        return p
    if not temp > 0:
        p[int(np.argmax(z))] = 1.0
        return p
    p = np.exp((z - m) / float(np.float32(temp)))
    return p / p.sum()


def cut64(values, ids, lane, vocab):
    """The distribution of a row of candidates as mk_sample_draw makes it: (ids of the kept, float probabilities)."""
    t = np.float32(lane["temperature"])
    if not t > 0:
        return ids[:1], np.ones(1, np.float32)
    w = np.exp(((values - values[0]) / t).astype(np.float32).astype(np.float64)).astype(np.float32)
    floor, nucleus = float(np.float32(lane["min_p"])) * float(w[0]), float(np.float32(lane["top_p"])) * float(
        w.astype(np.float64).sum())
    run, keep = 0.0, 0
    for i, x in enumerate(w):
        if i and x < floor:
            break
        run, keep = run + float(x), keep + 1
        if run >= nucleus:
            break
    return ids[:keep], (w[:keep].astype(np.float64) / run).astype(np.float32)


def verify64(lane, target, draft, drafts, u, u_next, n_out):
    """target(j), draft(j): (order of ids, probabilities in it) or, draft None, certain drafts."""
    def prob(dist, x):
        at = np.flatnonzero(dist[0] == x)
        return float(dist[1][at[0]]) if len(at) else 0.0

    out, pr, over = [], [], None
    for j in range(lane["n_draft"]):
        x, p = int(drafts[lane["first"] + j]), target(j)
        q = draft(j) if draft else (np.array([x]), np.ones(1))
        qd, pd = prob(q, x), prob(p, x)
        if not (qd > 0 and float(u[lane["first"] + j]) * qd < pd):
            over = q
            break
        out.append(x)
        pr.append(pd)
    p = target(len(out))
    r = p[1].astype(np.float64)
    if over is not None:
        left = {int(i): float(v) for i, v in zip(*over)}
        r = np.array([max(float(v) - left.get(int(i), 0.0), 0.0) for i, v in zip(*p)]) if len(left) < 2000 else \
            np.maximum(p[1] - over[1], 0.0)
        if not r.sum() > 0:
            r = p[1].astype(np.float64)
    acc = len(out)
    if r.sum() > 0:
        run = np.cumsum(r)
        hit = np.flatnonzero((run >= u_next * run[-1]) & (r > 0))
        i = int(hit[0] if len(hit) else np.flatnonzero(r > 0)[-1])
        out.append(int(p[0][i]))
        pr.append(float(p[1][i]))
    return acc, out + [-1] * (n_out - len(out)), pr + [0.0] * (n_out - len(pr))


def cut_any64(values, ids, lane):
    """cut64 of a row with any logits in it: NaN counts as -inf, +inf as the largest float, an infinite temperature as the
    largest float; what is -inf then is no candidate."""
    v = np.where(np.isnan(values), -np.inf, np.minimum(values, np.finfo(np.float32).max)).astype(np.float32)
    on = v > -np.inf
    if not on.any():
        return ids[:0], np.zeros(0, np.float32)
    lane = {k: float(lane[k]) for k in ("temperature", "min_p", "top_p")}
    lane["temperature"] = min(lane["temperature"], float(np.finfo(np.float32).max))
    with np.errstate(over="ignore"):
        return cut64(v[on], ids[on], lane, 0)


def attention_norms64(q, n_head, pre, pseq, n_prefix, kv, row0, layer, seq, keys):
    """Outputs [n][n_head][d] and what fp32 sums leave the 2-norm of a row's error at. Roundings are independent of each
    other: a sum of L terms walks to half a step times the root of L times the root of the terms' squares, B for a score's
    products (two of them, hi and lo) and S for the output's, while the keys' weights have no more than a few half steps of
    the score's range each, and their sum's error moves the whole row. A q or weights with the lo part missing, or a key
    left out, are ten times and more beyond it."""
    k, v, ks, vs = kv
    KV, d, byte = k.shape[2], k.shape[4], permuted(k.shape[4])
    G = n_head // KV
    out, tol = np.zeros((len(seq), n_head, d)), np.zeros((len(seq), n_head))
    for t in range(len(seq)):
        a, b = min(int(keys[t]), n_prefix), max(0, int(keys[t]) - n_prefix)
        for g in range(KV):
            K, V = [], []
            for (ck, cv, cks, cvs), i, lo, c in ((pre or kv, pseq, 0, a), (kv, seq[t], row0, b)):
                at = (layer, i, g, slice(lo, lo + c))
                if c:
                    K.append(ck[at][:, byte].astype(np.float64) * cks[at].astype(np.float64)[:, None])
                    V.append(cv[at].astype(np.float64) * cvs[at].astype(np.float64)[:, None])
            K, V = np.concatenate(K), np.concatenate(V)
            for h in range(g * G, (g + 1) * G):
                x = q[t, h * d:(h + 1) * d].astype(np.float64)
                s, B = K @ x / np.sqrt(d), np.sqrt((K ** 2 @ x ** 2).max() / d)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, h] = p @ V
                S, walk = np.sqrt((p ** 2 @ V ** 2).sum()), 2 * np.sqrt(len(K))
                tol[t, h] = EPS * ((2 * np.sqrt(d) * B + 4 * (s.max() - s.min()) + 32 + walk) * S +
                                   walk * np.sqrt((out[t, h] ** 2).sum()))
    return out, tol


def lora_norms64(x, adapters, ids, rows):
    """The adapters' part alone and what fp32 sums leave the 2-norm of a token's error at: both products' sums walk as in
    attention_norms64, relative to the root of the terms' squares. x in fp16 is twenty times and more beyond it, a column
    left out a thousand."""
    y, tol = np.zeros((len(x), rows)), np.zeros(len(x))
    for t, i in enumerate(ids):
        if not 0 <= i < len(adapters) or adapters[i] is None:
            continue
        a, b, xt = (z.astype(np.float64) for z in (adapters[i][0], adapters[i][1], x[t]))
        scale = float(np.float32(adapters[i][2]))
        y[t] = scale * (b @ (a @ xt))
        size = abs(scale) * np.sqrt((b ** 2 @ (a ** 2 @ xt ** 2)).sum())
        tol[t] = EPS * (np.sqrt(a.shape[1]) + np.sqrt(a.shape[0]) + 8) * size
    return y, tol
