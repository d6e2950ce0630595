"""Operators of a KV cache that is held in 4 bits and in pages, and of the beam search over it, each in its plain form
(elementary torch operations) and as a program calls it through the C ABI (include/malkin_hip.h). A case is a dict of plain
values; its "op" says which operator it is:

  rope       mk_rope_kv4 (norm of q and k, rotary positions, both into place: q rotated, k and v in 4 bits into the cache's
             pages), read back by mk_kv4_rows. "pairs": which elements rotate together (neighbours, or the halves of the
             rotated part); "part": how many elements of a head rotate
  tables     mk_rope_tables: cosines and sines of every position, the frequencies scaled for long contexts
  attention  mk_attention_kv4: "users" sequences with "each" tokens (1: decoding; more: a chain of drafts) or "prompt" tokens
             in all, split unevenly; "rows": of the longest sequence; "pad" rows of a batch of fixed size that hold no token
  pages      the cache's pages: "beams" mk_kv4_fork (every beam goes on from its parent) and mk_kv4_resize (room for a token:
             shared last pages are copied), "turnover" the same calls where users leave, come and take drafts back,
             "compact" mk_kv4_compact
  beam       mk_beam_select: the best continuations over beams and vocabulary. "done": some beams have ended

What is in 4 bits: groups of 32 elements of a row, element n of 0 .. 15 standing for scale * (n - 8), which fp16 holds exactly
(the scale has at most 8 significant bits). Everything follows from the seed; lengths follow from the case.
"""
import math

import torch

own = False

VOCAB = 151936  # Qwen3


def listed():
    return [
        # One token of eight users of an 8B model; the step's first launch after the q|k|v projection.
        {"name": "rope_decode8", "op": "rope", "heads": 32, "kv_heads": 8, "dim": 128, "part": 128, "pairs": False,
         "norm": True, "n": 8, "users": 8, "page": 32, "rows": 700, "positions": 32768, "pad": 0},
        # A prompt's forward without norms, neighbours rotating together in half of each head, in a padded batch.
        {"name": "rope_prompt1500", "op": "rope", "heads": 16, "kv_heads": 8, "dim": 128, "part": 64, "pairs": True,
         "norm": False, "n": 1500, "users": 3, "page": 64, "rows": 2100, "positions": 8192, "pad": 36},
        # The tables of a 128K context, frequencies stretched from 32K (YaRN).
        {"name": "tables_131072", "op": "tables", "part": 128, "scaling": "yarn", "factor": 4.0, "orig": 32768,
         "base": 1e6, "positions": 131072, "first": 0, "divided": False},
        # Two chats on a 0.6B model.
        {"name": "attn_decode2", "op": "attention", "heads": 16, "kv_heads": 8, "dim": 128, "users": 2, "each": 1,
         "prompt": 0, "rows": 300, "page": 16, "pad": 0},
        # Decoding of 24 users of very different lengths, in a batch padded to its captured size.
        {"name": "attn_decode24", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "users": 23, "each": 1,
         "prompt": 0, "rows": 6000, "page": 32, "pad": 1},
        # Four users with documents of up to 120 thousand tokens, five drafted tokens each (four and the last one).
        {"name": "attn_long4", "op": "attention", "heads": 40, "kv_heads": 8, "dim": 128, "users": 4, "each": 5,
         "prompt": 0, "rows": 120000, "page": 64, "pad": 0},
        # Three prompts, later parts of them, packed into one 512-token forward.
        {"name": "attn_prompt512", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "users": 3, "each": 0,
         "prompt": 512, "rows": 2600, "page": 64, "pad": 0},
        # A beam search of 16 requests of four beams each: a step's bookkeeping, small pages.
        {"name": "pages_beams16", "op": "pages", "kind": "beams", "layers": 28, "kv_heads": 8, "dim": 128, "users": 16,
         "beams": 4, "rows": 600, "page": 16, "spare": 120},
        # A server's pool after hours of requests of all lengths: the pages in use moved together.
        {"name": "pages_compact", "op": "pages", "kind": "compact", "layers": 28, "kv_heads": 8, "dim": 128, "users": 40,
         "beams": 1, "rows": 900, "page": 32, "spare": 300},
        # One request of four beams.
        {"name": "beam_one", "op": "beam", "users": 1, "beams": 4, "k": 8, "vocab": VOCAB, "done": False, "ban": False},
        # 24 requests of four beams, some of which have ended, part of the vocabulary masked by a grammar.
        {"name": "beam_batch24", "op": "beam", "users": 24, "beams": 4, "k": 4, "vocab": VOCAB, "done": True, "ban": True},
        # Wide beams over a smaller vocabulary.
        {"name": "beam_wide32", "op": "beam", "users": 5, "beams": 32, "k": 64, "vocab": 32003, "done": True, "ban": False},
    ]


# What the largest listed cases cost: scored (row, key) pairs, keys held, rotated values, table entries, bytes of pages, logits.
MOST_PAIRS, MOST_KEYS, MOST_VALUES = 20 * 40 * 80000, 300000 * 8, 1500 * 32 * 128
MOST_ENTRIES, MOST_POOL, MOST_LOGITS = 131072 * 64, 700 << 20, 96 * VOCAB


def log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    op = rng.choice(["rope", "rope", "tables", "attention", "attention", "attention", "pages", "pages", "beam", "beam"])
    heads, kv = rng.choice([(16, 8), (32, 8), (32, 8), (40, 8), (8, 2), (4, 2), (8, 8)])
    dim, page = rng.choice([64, 128, 128, 128]), rng.choice([16, 32, 64, 128])
    if op == "rope":
        n = log_int(rng, 1, max(1, min(1500, MOST_VALUES // ((heads + 2 * kv) * dim))))
        return {"op": op, "heads": heads, "kv_heads": kv, "dim": dim, "part": rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
                "pairs": rng.random() < 0.4, "norm": rng.random() < 0.6, "n": n, "users": rng.randint(1, min(n, 16)),
                "page": page, "rows": n + log_int(rng, 1, 900), "positions": log_int(rng, 4000, 40000),
                "pad": rng.choice([0, 0, rng.randint(1, 3)])}
    if op == "tables":
        part = 2 * rng.randint(8, 64)
        return {"op": op, "part": part, "scaling": rng.choice(["plain", "linear", "ntk", "yarn"]),
                "factor": rng.choice([2.0, 4.0, 8.0, rng.uniform(1.0, 40.0)]), "orig": rng.choice([4096, 32768, rng.randint(512, 40000)]),
                "base": rng.choice([1e4, 1e6, 5e5]), "positions": log_int(rng, 1, MOST_ENTRIES // (part // 2)),
                "first": rng.choice([0, rng.randint(0, 1000000)]), "divided": rng.random() < 0.3}
    if op == "attention":
        c = {"op": op, "heads": heads, "kv_heads": kv, "dim": dim, "users": log_int(rng, 1, 64),
             "each": rng.choice([1, 1, 1, log_int(rng, 2, 9), 0]), "prompt": 0, "rows": log_int(rng, 9, 30000), "page": page,
             "pad": rng.choice([0, 0, rng.randint(1, 3)])}
        if c["each"] == 0:
            c["users"] = min(c["users"], 8)
            c["prompt"] = log_int(rng, max(16, c["users"]), 512)
        n = c["prompt"] or c["users"] * c["each"]
        c["rows"] = max(c["prompt"], c["each"], min(c["rows"], MOST_PAIRS // (n * heads), MOST_KEYS // (kv * c["users"])))
        return c
    if op == "pages":
        c = {"op": op, "kind": rng.choice(["beams", "beams", "turnover", "compact"]), "layers": rng.choice([4, 28, rng.randint(1, 36)]),
             "kv_heads": kv, "dim": dim, "users": log_int(rng, 1, 24), "beams": 1, "rows": log_int(rng, 5, 600), "page": page,
             "spare": log_int(rng, 20, 200)}
        if c["kind"] == "beams":
            c["beams"] = rng.choice([2, 3, 4, 4, 8])
        row = c["layers"] * kv * (dim + dim // 8)
        c["rows"] = max(1, min(c["rows"], MOST_POOL // 2 // (row * c["users"] * c["beams"])))
        c["spare"] = min(c["spare"], 8 + MOST_POOL // 2 // (row * page)) + 2 * c["users"] * c["beams"]
        return c
    beams = rng.choice([1, 2, 4, 4, 8, log_int(rng, 1, 32)])
    vocab = rng.choice([VOCAB, VOCAB, 32768, rng.randint(1000, 152000)])
    return {"op": op, "users": log_int(rng, 1, max(1, min(24, MOST_LOGITS // (vocab * beams)))), "beams": beams,
            "k": min(64, rng.choice([beams, 2 * beams, rng.randint(1, 64)])), "vocab": vocab, "done": rng.random() < 0.4,
            "ban": rng.random() < 0.3}


# ---- layouts, from the case alone ----

def fraction(i):
    return (0.381966 * (i + 1)) % 1.0


def shares(total, parts):
    """`total` split unevenly."""
    w = [0.3 + fraction(i) for i in range(parts)]
    at = [round(total * sum(w[:i]) / sum(w)) for i in range(parts + 1)]
    return [b - a for a, b in zip(at, at[1:])]


def tokens_of(c):
    """Per user: its tokens in the batch and the rows that the last of them sees."""
    new = [c["each"]] * c["users"] if c.get("each") else shares(c.get("prompt") or c["n"], c["users"])
    return [(m, c["rows"] if i == 0 else max(m, round(c["rows"] * (0.2 + 0.8 * fraction(i))))) for i, m in enumerate(new)]


def batch_of(c):
    """seq and row (position in its sequence) of every token of the batch; rows without a token: -1, -1."""
    seq, row = [], []
    for i, (m, rows) in enumerate(tokens_of(c)):
        seq += [c["users"] - 1 - i] * m
        row += [rows - m + j for j in range(m)]
    return seq + [-1] * c["pad"], row + [-1] * c["pad"]


def lengths_of(c):
    """Rows per sequence of the pages cases: of one request's beams the same."""
    return [c["rows"] if u == 0 else max(1, round(c["rows"] * (0.2 + 0.8 * fraction(u)))) for u in range(c["users"])
            for _ in range(c["beams"])]


def pages_for(rows, page):
    return (rows + page - 1) // page


# ---- inputs ----

def generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def in4(x):
    """Rows [..., d] as numbers 0 .. 15 and fp16 scales [..., d / 32]: the element furthest from 0 becomes 0 (-8 steps)."""
    g = torch.nan_to_num(x.double(), nan=0.0, posinf=math.inf, neginf=-math.inf).unflatten(-1, (-1, 32))
    hi, lo = g.amax(-1), g.amin(-1)
    s = (torch.where(hi >= -lo, hi, lo) / -8).clamp(-4096, 4096).float().bfloat16().half()
    inv = torch.where(s == 0, 0.0, 1.0 / s.double())
    return ((g * inv[..., None]).nan_to_num(nan=0.0).round().clamp(-8, 7) + 8).to(torch.uint8).flatten(-2), s


def packed(n):
    """Two elements a byte, the first in the low half."""
    return n[..., 0::2] | n[..., 1::2] << 4


def unpacked(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def values(n, s):
    """What the numbers stand for, in fp16, exactly."""
    return ((n.half() - 8).unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def tables_in_order(g, counts, n_page, most):
    """Pages of every sequence, taken from all over the pool."""
    order = torch.randperm(n_page, generator=g, device="cuda").int()
    table = torch.full((len(counts), most), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, m in enumerate(counts):
        table[i, :m] = order[at:at + m]
        at += m
    return table


def cache(g, c, layers, n_page, page, fill):
    """k, v, k_scale, v_scale of the pool: rows as the model writes them, or any bytes where only their place matters."""
    kv, d = c["kv_heads"], c["dim"]
    s = {}
    for x in "kv":
        if fill:
            n, sc = in4(normal(g, n_page, layers, kv, page, d))
            s[x] = packed(n)
        else:
            s[x] = torch.randint(0, 256, (n_page, layers, kv, page, d // 2), dtype=torch.uint8, generator=g, device="cuda")
            sc = (0.1 + torch.rand(n_page, layers, kv, page, d // 32, generator=g, device="cuda")).half()
        s[x + "s"] = (sc if x == "k" else sc.transpose(-1, -2)).contiguous()
    return s


def prepare_rope(c, seed):
    g, (seq, row) = generator(seed), batch_of(c)
    counts = [0] * c["users"]
    for i, (_, rows) in enumerate(tokens_of(c)):
        counts[c["users"] - 1 - i] = pages_for(rows, c["page"])
    n_page, n, d, H, KV = sum(counts) + 3, len(seq), c["dim"], c["heads"], c["kv_heads"]
    s = cache(g, c, 1, n_page, c["page"], False)
    s["table"] = tables_in_order(g, counts, n_page, max(counts))
    s["qkv"] = 1.5 * normal(g, n, (H + 2 * KV) * d)
    s["qkv"][:, ::61] *= 5.0  # a few large channels
    s["q_norm"], s["k_norm"] = ((1 + 0.2 * normal(g, d)) if c["norm"] else None for _ in range(2))
    f = 1e6 ** (-torch.arange(c["part"] // 2, dtype=torch.float64, device="cuda") / (c["part"] // 2))
    a = torch.arange(c["positions"], dtype=torch.float64, device="cuda")[:, None] * f
    s["cos"], s["sin"] = a.cos().float(), a.sin().float()
    s["seq"], s["row"] = ints(seq), ints(row)
    s["pos"] = ints([max(r, 0) for r in row])
    s["q"] = torch.zeros(n, H, d, device="cuda")
    s["k_out"], s["v_out"] = (torch.zeros(n, KV, d, dtype=torch.float16, device="cuda") for _ in range(2))
    return s


def prepare_tables(c, seed):
    g, half = generator(seed), c["part"] // 2
    # Which frequencies a model divides by how much is part of its weights.
    s = {"divide": 1 + 7 * torch.rand(half, generator=g, device="cuda") if c["divided"] else None}
    s["base"] = c["base"] * (1 + seed % 97 / 1000)
    s["cos"], s["sin"] = (torch.empty(c["positions"], half, device="cuda") for _ in range(2))
    return s


def prepare_attention(c, seed):
    g, (seq, row) = generator(seed), batch_of(c)
    counts, first, new = [0] * c["users"], [0] * c["users"], [0] * c["users"]
    at = 0
    for i, (m, rows) in enumerate(tokens_of(c)):
        u = c["users"] - 1 - i
        counts[u], first[u], new[u] = pages_for(rows, c["page"]), at, m
        at += m
    n_page = sum(counts) + 2
    s = cache(g, c, 1, n_page, c["page"], True)
    s["table"] = tables_in_order(g, counts, n_page, max(counts))
    s["q"] = 1.5 * normal(g, len(seq), c["heads"], c["dim"])
    s["seq"], s["keys"], s["most"] = ints(seq), ints([r + 1 for r in row]), max(row) + 1
    s["first"], s["new"], s["run"] = ints(first), ints(new), max(new)
    s["out"] = torch.empty_like(s["q"])
    return s


def prepare_pages(c, seed):
    g, lens, B = generator(seed), lengths_of(c), c["beams"]
    n_seq, page = len(lens), c["page"]
    need = [pages_for(m, page) for m in lens]
    most = max(need) + (8 if c["kind"] == "turnover" else 1)
    shared = [m * 4 // 5 for m in need]  # pages that a request's beams have in common
    used = sum(need[i] if i % B == 0 else need[i] - shared[i] for i in range(n_seq))
    n_page = used + c["spare"]
    s = cache(g, c, c["layers"], n_page, page, False)
    order = torch.randperm(n_page, generator=g, device="cuda").tolist()
    table, at = [], 0
    for i, m in enumerate(need):
        have = 0 if i % B == 0 else shared[i]
        table.append((table[i // B * B][:have] if have else []) + order[at:at + m - have] + [-1] * (most - m))
        at += m - have
    refs = [0] * n_page
    for r in table:
        for p in r:
            if p >= 0:
                refs[p] += 1
    # table, len and refs in one array, as it was before a pass and as the pass leaves it.
    s["before"] = ints([p for r in table for p in r] + lens + refs)
    s["meta"], s["most"], s["n_page"] = s["before"].clone(), most, n_page
    pick = torch.rand(n_seq, generator=g, device="cuda").tolist()
    if c["kind"] == "beams":
        src, new = [i // B * B + int(pick[i] * B) for i in range(n_seq)], [m + 1 for m in lens]
    else:  # a fifth of the users leave; of the others some take drafts back, some go on, some have a prompt
        src, new = [-1 if p < 0.2 else i for i, p in enumerate(pick)], []
        for i, p in enumerate(pick):
            m = 0 if p < 0.2 else lens[i]
            new.append(max(0, m - 3) if 0.2 <= p < 0.4 else min(most * page, m + (1 if p < 0.7 else 3 * page + 5)))
    s["src"], s["new"] = ints(src), ints(new)
    s["every"] = torch.arange(n_seq, dtype=torch.int32, device="cuda")
    s["status"], s["live"] = torch.zeros_like(s["every"]), ints([0])
    return s


def prepare_beam(c, seed):
    g, rows, V = generator(seed), c["users"] * c["beams"], c["vocab"]
    z = 1.5 * normal(g, rows, V)
    peak = torch.randint(0, V, (rows, 12), generator=g, device="cuda")
    z.scatter_add_(1, peak, 12 + 2 * normal(g, rows, 12))
    if c["ban"]:
        z[:, torch.rand(V, generator=g, device="cuda") < 0.5] = -math.inf
    s = {"logits": z, "scores": -5.0 * torch.rand(rows, generator=g, device="cuda") - 1.0}
    s["scores"][c["beams"] - 1::4 * c["beams"]] = -math.inf if c["beams"] > 1 else 0.0  # a beam that is not there
    s["done"] = (torch.rand(rows, generator=g, device="cuda") < 0.25).int() if c["done"] else None
    s["eos"] = V - 293
    shape = (c["users"], c["k"])
    s["out"] = {"scores": torch.zeros(shape, device="cuda")}
    s["out"] |= {x: torch.zeros(shape, dtype=torch.int32, device="cuda") for x in ("seq", "tokens")}
    return s


PREPARE = {"rope": prepare_rope, "tables": prepare_tables, "attention": prepare_attention, "pages": prepare_pages,
           "beam": prepare_beam}


def prepare(case, seed):
    s = PREPARE[case["op"]](case, seed)
    s["case"] = dict(case)
    torch.cuda.synchronize()  # inputs made on torch's stream; the library works on its own
    return s


# ---- plain forms ----

def rotated(x, cos, sin, pairs):
    """x [n][heads][d]: the first 2 r elements of every head by cos, sin [n][r]."""
    r = cos.shape[1]
    a, b = (x[..., 0:2 * r:2], x[..., 1:2 * r:2]) if pairs else (x[..., :r], x[..., r:2 * r])
    cos, sin = cos[:, None], sin[:, None]
    y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1 if pairs else -2).flatten(-2)
    return torch.cat([y, x[..., 2 * r:]], -1)


def rope_plain(s):
    """Norm and rotation in 64 bits: what is rounded to 16 steps lies next to a border often enough."""
    c = s["case"]
    H, KV, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    q, k, v = s["qkv"].double().unflatten(1, (-1, d)).split([H, KV, KV], 1)
    if s["q_norm"] is not None:
        q, k = (x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double() for x, w in ((q, s["q_norm"]), (k, s["k_norm"])))
    cos, sin = (s[x][s["pos"].long()].double() for x in ("cos", "sin"))
    q, k = rotated(q, cos, sin, c["pairs"]), rotated(k, cos, sin, c["pairs"])
    live = s["seq"] >= 0
    seq, row = s["seq"].clamp_min(0).long(), s["row"].clamp_min(0).long()
    (kn, ks), (vn, vs) = in4(k), in4(v)
    p, r = s["table"][seq, row // page][live].long(), (row % page)[live]
    s["k"][p, 0, :, r], s["ks"][p, 0, :, r] = packed(kn[live]), ks[live]
    s["v"][p, 0, :, r], s["vs"][p, 0, :, :, r] = packed(vn[live]), vs[live]
    k, v = (torch.where(live[:, None, None], values(*x), 0.0) for x in ((kn, ks), (vn, vs)))
    return {"q": torch.where(live[:, None, None], q, 0.0).float(), "k": k.half(), "v": v.half()}


def frequencies(c, s):
    """Radians a position, and what cosines and sines are multiplied by (Peng et al. 2023 for YaRN)."""
    d, factor, base = c["part"], c["factor"], s["base"]
    i = torch.arange(d // 2, dtype=torch.float64, device="cuda")
    base = torch.tensor(base, device="cuda").double()  # as the call takes it: a float
    if c["scaling"] == "ntk":
        base = base * factor ** (d / (d - 2))
    f = base ** (-2 * i / d)
    if s["divide"] is not None:
        f = f / s["divide"].double()
    if c["scaling"] == "linear":
        return f / factor, 1.0
    if c["scaling"] != "yarn":
        return f, 1.0
    turns = [d * math.log(c["orig"] / (2 * math.pi * b)) / (2 * math.log(float(base))) for b in (32.0, 1.0)]
    low, high = max(math.floor(turns[0]), 0), min(math.ceil(turns[1]), d - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1


def tables_plain(s):
    """In 64 bits: a far position has hundreds of thousands of radians."""
    c = s["case"]
    f, m = frequencies(c, s)
    a = (torch.arange(c["positions"], device="cuda") + c["first"]).double()[:, None] * f
    return {"cos": (a.cos() * m).float(), "sin": (a.sin() * m).float()}


def attention_plain(s):
    """The sequences' tokens side by side, padded; their pages gathered and taken out of 4 bits."""
    c = s["case"]
    n, H, d, KV, m, L = len(s["q"]), c["heads"], c["dim"], c["kv_heads"], s["run"], s["table"].shape[1] * c["page"]
    G, U = H // KV, c["users"]
    p = s["table"].clamp_min(0).long()
    k = values(unpacked(s["k"][p][:, :, 0]), s["ks"][p][:, :, 0])
    v = values(unpacked(s["v"][p][:, :, 0]), s["vs"][p][:, :, 0].transpose(-1, -2))
    k, v = (x.float().transpose(1, 2).reshape(U * KV, L, d) for x in (k, v))  # [users][pages][kv][page][d] before
    at = (s["first"][:, None] + torch.arange(m, device="cuda")).clamp_max(n - 1).long()
    q = s["q"][at].reshape(U, m, KV, G, d).transpose(1, 2).reshape(U * KV, m * G, d) / math.sqrt(d)
    sc = torch.bmm(q, k.transpose(1, 2).contiguous()).reshape(U, KV, m, G, L)
    live = torch.arange(L, device="cuda") < s["keys"][at][..., None]
    sc = torch.where(live[:, None, :, None], sc, -math.inf)
    e = torch.exp(sc - sc.amax(-1, keepdim=True).clamp_min(-1e30))
    w = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.bmm(w.reshape(U * KV, m * G, L), v).reshape(U, KV, m, G, d).transpose(1, 2).reshape(U, m, H, d)
    out = torch.zeros_like(s["q"])
    here = torch.arange(m, device="cuda") < s["new"][:, None]
    out[at[here]] = o[here]
    return {"out": out}


def split_meta(s, meta):
    n = len(s["every"])
    return meta[:n * s["most"]].view(n, s["most"]), meta[n * s["most"]:n * s["most"] + n], meta[n * (s["most"] + 1):]


def counted(table, n_page):
    flat = table.flatten()
    return torch.zeros(n_page + 1, dtype=torch.int32, device="cuda").index_add(
        0, torch.where(flat >= 0, flat, n_page), torch.ones_like(flat))[:n_page]


def pages_plain(s):
    c = s["case"]
    table, length, refs = split_meta(s, s["before"])
    n_page, page, status = s["n_page"], c["page"], s["status"]
    if c["kind"] == "compact":
        live = refs > 0
        n_live = live.sum()
        ids = torch.arange(n_page, device="cuda")
        holes, movers = ids[~live & (ids < n_live)], ids[live & (ids >= n_live)]
        to = ids.clone()
        to[movers] = holes
        table = torch.where(table >= 0, to[table.clamp_min(0).long()].int(), -1)
        src, dst, rows = movers, holes, torch.full_like(holes, page)
        n_live = n_live.int()[None]
    else:
        src = s["src"].long()
        gone = src < 0
        table = torch.where(gone[:, None], -1, table[src.clamp_min(0)])
        length = torch.where(gone, 0, length[src.clamp_min(0)]).long()
        want = s["new"].long()
        had, has = (length + page - 1) // page, (want + page - 1) // page
        j = torch.arange(s["most"], device="cuda")
        table = torch.where(j < torch.minimum(had, has)[:, None], table, -1)
        refs = counted(table, n_page)
        # A shared last page that is written on: every holder but the last to go on takes a copy.
        part, grows = length % page, want > length
        last = table.gather(1, ((length - 1).clamp_min(0) // page)[:, None])[:, 0]
        writes = grows & (part > 0)
        before = ((last[:, None] == last) & writes[:, None] & writes).tril(-1).sum(1)
        copy = writes & (before < refs[last.clamp_min(0).long()] - 1)
        need = torch.where(grows, copy.long() + has - had, 0)
        end = need.cumsum(0)
        free = torch.nonzero(refs == 0)[:, 0]
        fits = (need == 0) | (end <= len(free))
        copy, grows = copy & fits, grows & fits
        taken = (end - need)[:, None] + copy[:, None].long() + j - had[:, None]
        new_page = grows[:, None] & (j >= had[:, None]) & (j < has[:, None])
        pool = torch.cat([free, free.new_zeros(1)])
        table = torch.where(new_page, pool[taken.clamp(0, len(free))].int(), table)
        own_copy = pool[(end - need).clamp(0, len(free))]
        at = copy[:, None] & (j == ((length - 1) // page)[:, None])
        src, dst, rows = last[copy].long(), own_copy[copy], part[copy]
        table = torch.where(at, own_copy[:, None].int(), table)
        length = torch.where(fits, want, length).int()
        status = (~fits).int()
        n_live = s["live"]
    held = torch.arange(page, device="cuda") < rows[:, None]
    for x in "kv":
        s[x][dst] = torch.where(held[:, None, None, :, None], s[x][src], s[x][dst])
        y = x + "s"
        at = held[:, None, None, :, None] if x == "k" else held[:, None, None, None, :]
        s[y][dst] = torch.where(at, s[y][src], s[y][dst])
    return {"table": table, "len": length, "refs": counted(table, n_page), "status": status, "live": n_live,
            **{x: s[x] for x in ("k", "v", "ks", "vs")}}


def beam_plain(s):
    c = s["case"]
    U, B, V = c["users"], c["beams"], c["vocab"]
    z = torch.where(s["logits"].isnan(), -math.inf, s["logits"].clamp_max(3.4028234663852886e38)).double()
    top = z.amax(-1, keepdim=True).clamp_min(-1e300)
    z = z - (top + (z - top).exp().sum(-1, keepdim=True).log()) + s["scores"].double()[:, None]
    if s["done"] is not None:
        only = torch.where(torch.arange(V, device="cuda") == s["eos"], s["scores"].double()[:, None], -math.inf)
        z = torch.where(s["done"][:, None] != 0, only, z)
    z = torch.where(s["scores"].isfinite()[:, None], z, -math.inf).reshape(U, B * V)
    best, at = z.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :c["k"]], at[:, :c["k"]]
    some = best > -math.inf
    first = torch.arange(U, device="cuda")[:, None] * B
    return {"scores": best.float(), "seq": torch.where(some, first + at // V, -1).int(),
            "tokens": torch.where(some, at % V, -1).int()}


# ---- as a program calls them ----

_ctx = None


def library():
    """The native library and the program's one context."""
    global _ctx
    import malkin_amd as mk
    if _ctx is None:
        _ctx = mk.Context(0)
    return mk, mk.load(), _ctx.h


def workspace(s, name, nbytes):
    if name not in s:
        s[name] = torch.empty(max(1, nbytes), dtype=torch.uint8, device="cuda")
    return s[name].data_ptr(), s[name].numel()


def ptr(t):
    return None if t is None else t.data_ptr()


def kv4(mk, s, table, length, refs):
    c = s["case"]
    return mk.MkKv4Cache(*(ptr(s[x]) for x in ("k", "v", "ks", "vs")), ptr(table), ptr(length), ptr(refs), s["k"].shape[1],
                         s["k"].shape[0], c["page"], c["kv_heads"], c["dim"], *table.shape)


def rope_own(s):
    mk, lib, ctx = library()
    if "call" not in s:
        import ctypes
        c = s["case"]
        H, KV, d, n = c["heads"], c["kv_heads"], c["dim"], len(s["q"])
        s["kv"] = kv4(mk, s, s["table"], None, None)
        kv, at = ctypes.byref(s["kv"]), ptr(s["qkv"])
        layout = mk.ROPE_PAIRS if c["pairs"] else mk.ROPE_HALVES
        s["call"] = (ctx, at, at + 4 * H * d, at + 4 * (H + KV) * d, (H + 2 * KV) * d, n, H, ptr(s["q_norm"]),
                     ptr(s["k_norm"]), 1e-6, layout, c["part"], ptr(s["cos"]), ptr(s["sin"]), c["positions"], ptr(s["pos"]),
                     ptr(s["seq"]), ptr(s["row"]), kv, 0, ptr(s["q"]), H * d)
        s["read"] = (ctx, kv, 0, ptr(s["seq"]), ptr(s["row"]), n, ptr(s["k_out"]), ptr(s["v_out"]))
    mk.check(lib.mk_rope_kv4(*s["call"]))
    mk.check(lib.mk_kv4_rows(*s["read"]))
    return {"q": s["q"], "k": s["k_out"], "v": s["v_out"]}


def tables_own(s):
    mk, lib, ctx = library()
    if "call" not in s:
        import ctypes
        c = s["case"]
        kind = {"plain": mk.ROPE_PLAIN, "linear": mk.ROPE_LINEAR, "ntk": mk.ROPE_NTK, "yarn": mk.ROPE_YARN}[c["scaling"]]
        s["rope"] = mk.MkRope(c["part"], kind, s["base"], c["factor"], c["orig"], 32.0, 1.0, 0.0)
        s["call"] = (ctx, ctypes.byref(s["rope"]), ptr(s["divide"]), c["first"], c["positions"], ptr(s["cos"]), ptr(s["sin"]))
    mk.check(lib.mk_rope_tables(*s["call"]))
    return {"cos": s["cos"], "sin": s["sin"]}


def attention_own(s):
    mk, lib, ctx = library()
    if "call" not in s:
        import ctypes
        c = s["case"]
        H, d, KV, n = c["heads"], c["dim"], c["kv_heads"], len(s["q"])
        s["kv"] = kv4(mk, s, s["table"], None, None)
        work = workspace(s, "work", lib.mk_attention_kv4_workspace(n, H, KV, d, s["most"], s["run"]))
        s["call"] = (ctx, ptr(s["q"]), H * d, ptr(s["out"]), H * d, n, H, ctypes.byref(s["kv"]), 0, ptr(s["seq"]),
                     ptr(s["keys"]), s["most"], s["run"], None, *work)
    mk.check(lib.mk_attention_kv4(*s["call"]))
    return {"out": s["out"]}


def pages_own(s):
    mk, lib, ctx = library()
    if "kv" not in s:
        import ctypes
        c = s["case"]
        n = len(s["every"])
        s["kv"] = kv4(mk, s, *split_meta(s, s["meta"]))
        kv = ctypes.byref(s["kv"])
        s["restore"] = (ctx, ptr(s["meta"]), None, ptr(s["before"]), None, len(s["meta"]))
        if c["kind"] == "compact":
            s["compact"] = (ctx, kv, ptr(s["live"]), *workspace(s, "work", lib.mk_kv4_compact_workspace(s["n_page"])))
        else:
            s["fork"] = (ctx, kv, None, ptr(s["src"]), n, *workspace(s, "work", lib.mk_kv4_fork_workspace(n, s["most"])))
            s["resize"] = (ctx, kv, None, ptr(s["new"]), n, ptr(s["status"]),
                           *workspace(s, "work2", lib.mk_kv4_resize_workspace(n, s["n_page"])))
    mk.check(lib.mk_move_ids(*s["restore"]))  # a pass starts from the same pages every time
    if "compact" in s:
        mk.check(lib.mk_kv4_compact(*s["compact"]))
    else:
        mk.check(lib.mk_kv4_fork(*s["fork"]))
        mk.check(lib.mk_kv4_resize(*s["resize"]))
    table, length, refs = split_meta(s, s["meta"])
    return {"table": table, "len": length, "refs": refs, "status": s["status"], "live": s["live"],
            **{x: s[x] for x in ("k", "v", "ks", "vs")}}


def beam_own(s):
    mk, lib, ctx = library()
    if "call" not in s:
        c, out = s["case"], s["out"]
        work = workspace(s, "work", lib.mk_beam_workspace(c["users"], c["beams"], c["vocab"], c["k"]))
        s["call"] = (ctx, ptr(s["logits"]), c["vocab"], c["users"], c["beams"], c["vocab"], ptr(s["scores"]), ptr(s["done"]),
                     s["eos"], c["k"], ptr(out["scores"]), ptr(out["seq"]), ptr(out["tokens"]), *work)
    mk.check(lib.mk_beam_select(*s["call"]))
    return s["out"]


PLAIN = {"rope": rope_plain, "tables": tables_plain, "attention": attention_plain, "pages": pages_plain, "beam": beam_plain}
OWN = {"rope": rope_own, "tables": tables_own, "attention": attention_own, "pages": pages_own, "beam": beam_own}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ---- what a pass cannot do without ----

def moved_rows(c):
    """Rows of whole layers that the pages cases copy, about (which beams share a page depends on the seed)."""
    lens = lengths_of(c)
    if c["kind"] == "compact":  # pages in use beyond as many as there are, all over the pool
        used = sum(pages_for(m, c["page"]) for m in lens)
        return c["page"] * used * c["spare"] / (used + c["spare"])
    return sum(m % c["page"] for m in lens) * (1 - 1 / c["beams"]) * 0.6


def work(case):
    c = case
    if c["op"] == "rope":
        n, row = c["n"], c["kv_heads"] * c["dim"]
        return {"bytes": n * (8 * c["heads"] * c["dim"] + 8 * row + 2 * (row + row // 8) + 4 * row + 4 * c["part"] + 12),
                "flops": n * (c["heads"] + c["kv_heads"]) * (3 * c["part"] + 4 * c["dim"]) + 6 * n * row}
    if c["op"] == "tables":
        return {"bytes": 4 * c["positions"] * c["part"], "flops": 40 * c["positions"] * c["part"]}
    if c["op"] == "attention":
        seq, row = batch_of(c)
        rows = sum(r for _, r in tokens_of(c))
        return {"bytes": 8 * len(seq) * c["heads"] * c["dim"] + rows * c["kv_heads"] * (c["dim"] + c["dim"] // 8) + 8 * len(seq)
                + 4 * rows / c["page"], "flops": 4 * c["heads"] * c["dim"] * sum(r + 1 for r in row)}
    if c["op"] == "pages":
        row = c["layers"] * c["kv_heads"] * (c["dim"] + c["dim"] // 8)
        pages = sum(pages_for(m, c["page"]) for m in lengths_of(c))
        return {"bytes": 2 * row * moved_rows(c) + 16 * pages + 8 * c["spare"], "flops": 0}
    rows = c["users"] * c["beams"]
    return {"bytes": 4 * rows * c["vocab"] + 8 * rows + 12 * c["users"] * c["k"], "flops": 8 * rows * c["vocab"]}


# ---- the same results in 64 bits ----

def exact_rope(c, seed):
    s = prepare_rope(c, seed)
    H, KV, d, r = c["heads"], c["kv_heads"], c["dim"], c["part"] // 2
    seq, row = batch_of(c)
    x = s["qkv"].double().reshape(len(seq), H + 2 * KV, d)
    if s["q_norm"] is not None:
        w = torch.cat([s["q_norm"].expand(H, d), s["k_norm"].expand(KV, d)]).double()
        x[:, :H + KV] *= w * torch.rsqrt((x[:, :H + KV] ** 2).sum(-1, keepdim=True) / d + 1e-6)
    # The rotation as a complex product.
    turn = torch.complex(s["cos"][s["pos"].long()].double(), s["sin"][s["pos"].long()].double())[:, None]
    y = x[:, :H + KV]
    a = torch.arange(r, device="cuda")
    a, b = (2 * a, 2 * a + 1) if c["pairs"] else (a, a + r)
    z = torch.complex(y[..., a], y[..., b]) * turn
    y[..., a], y[..., b] = z.real, z.imag
    x[torch.tensor(seq, device="cuda") < 0] = 0

    def rounded(v):
        g = v.reshape(len(seq), KV, d // 32, 32)
        big = g.gather(-1, g.abs().argmax(-1, keepdim=True))
        m, e = torch.frexp(big / -8)
        sc = torch.ldexp(torch.round(m * 256) / 256, e)  # 8 significant bits
        sc = torch.round(sc * 2 ** 24) / 2 ** 24  # and no finer than fp16's smallest step
        steps = torch.where(sc == 0, 0.0, torch.round(g / torch.where(sc == 0, 1.0, sc)).clamp(-8, 7))
        return (sc * steps).reshape(len(seq), KV, d)

    return {"q": x[:, :H], "k": rounded(x[:, H:H + KV]), "v": rounded(x[:, H + KV:])}


def exact_tables(c, seed):
    s = prepare_tables(c, seed)
    d, base = c["part"], float(torch.tensor(s["base"], dtype=torch.float32))
    freq = []
    for i in range(d // 2):
        b = base * c["factor"] ** (d / (d - 2)) if c["scaling"] == "ntk" else base
        f = math.exp(-2 * i / d * math.log(b))
        if s["divide"] is not None:
            f /= float(s["divide"][i])
        if c["scaling"] == "linear":
            f /= c["factor"]
        elif c["scaling"] == "yarn":
            lo, hi = (d * math.log(c["orig"] / (2 * math.pi * t)) / (2 * math.log(base)) for t in (32.0, 1.0))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), d - 1)
            part = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = f * (part / c["factor"] + 1 - part)
        freq.append(f)
    m = 1 + 0.1 * math.log(c["factor"]) if c["scaling"] == "yarn" else 1.0
    pos = torch.arange(c["first"], c["first"] + c["positions"], dtype=torch.float64, device="cuda")
    w = torch.polar(torch.tensor(m, dtype=torch.float64, device="cuda"), pos[:, None] * torch.tensor(freq, dtype=torch.float64, device="cuda"))
    return {"cos": w.real, "sin": w.imag}


def exact_attention(c, seed):
    s = prepare_attention(c, seed)
    H, d, KV, page = c["heads"], c["dim"], c["kv_heads"], c["page"]
    seq, row = batch_of(c)
    out = torch.zeros(len(seq), H, d, dtype=torch.float64, device="cuda")

    def held(x, u, g, transposed):
        b = s[x][s["table"][u].clamp_min(0).long(), 0, g].to(torch.int32).reshape(-1, d // 2)
        n = torch.empty(len(b), d, dtype=torch.float64, device="cuda")
        n[:, 0::2], n[:, 1::2] = (b % 16).double(), (b // 16).double()
        sc = s[x + "s"][s["table"][u].clamp_min(0).long(), 0, g].double()
        sc = (sc.transpose(1, 2) if transposed else sc).reshape(-1, d // 32)
        return (n - 8) * torch.repeat_interleave(sc, 32, dim=1)

    for u in sorted(set(seq) - {-1}):
        at = torch.tensor([t for t, x in enumerate(seq) if x == u], device="cuda")
        keys = torch.tensor([row[t] + 1 for t in at.tolist()], device="cuda")
        for g in range(KV):
            k, v = held("k", u, g, False), held("v", u, g, True)
            q = s["q"][at, g * (H // KV):(g + 1) * (H // KV)].double()
            z = q @ k.T / d ** 0.5
            z = z.masked_fill(torch.arange(len(k), device="cuda") >= keys[:, None, None], -math.inf)
            out[at, g * (H // KV):(g + 1) * (H // KV)] = torch.softmax(z, -1) @ v
    return {"out": out}


def exact_beam(c, seed):
    s = prepare_beam(c, seed)
    B, V, k = c["beams"], c["vocab"], c["k"]
    scores, seqs, tokens = [], [], []
    for u in range(c["users"]):
        best = []
        for i in range(u * B, (u + 1) * B):
            start = float(s["scores"][i])
            if not math.isfinite(start):
                continue
            if s["done"] is not None and int(s["done"][i]):
                best.append((start, i, s["eos"]))
                continue
            p = torch.log_softmax(s["logits"][i].double(), 0)
            v, at = torch.topk(p, min(k, V))
            best += [(start + a, i, b) for a, b in zip(v.tolist(), at.tolist()) if a > -math.inf]
        best = sorted(best, key=lambda t: (-t[0], t[1], t[2]))[:k]
        best += [(-math.inf, -1, -1)] * (k - len(best))
        scores.append([t[0] for t in best])
        seqs.append([t[1] for t in best])
        tokens.append([t[2] for t in best])
    return {"scores": torch.tensor(scores, dtype=torch.float64, device="cuda"), "seq": ints(seqs), "tokens": ints(tokens)}


def exact(case, seed):
    if case["op"] == "pages":
        return None  # whole numbers only
    return {"rope": exact_rope, "tables": exact_tables, "attention": exact_attention, "beam": exact_beam}[case["op"]](case, seed)
