"""Operators that let a batch of different requests share work, each in its plain form (elementary torch operations)
and as a program calls it through the C ABI (include/malkin_hip.h). A case is a dict of plain values; its "op" says
which operator it is:

  attention  mk_attention_prefix: a batch whose sequences share a long prefix in the int8 KV cache. "users" sequences
             with "each" tokens (1: decoding; more: a chain of drafts) or "prompt" tokens in all, split unevenly; "own"
             rows of its own in the longest sequence; "pad" rows of a batch of fixed size that hold no token
  lora       mk_lora: low-rank adapters chosen per token, added to a projection's output. "spread": how tokens take
             adapters: "each" (one after the other, every fourth token none) or "runs" (prompts, one after the other)
  verify     mk_verify: drafted tokens against the target's whole-vocabulary probabilities. "draft": whether the draft
             model's logits are given; "ban": part of the vocabulary is masked with -inf
  topk       mk_verify_topk: the same over rows cut to their top k

Everything follows from the seed; lengths follow from the case.
"""
import math

import torch

own = False

VOCAB = 151936  # Qwen3
D8 = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # Two chats on a 0.6B model behind one short system prompt: the smallest call, launches count.
        {"name": "attn_decode2", "op": "attention", "heads": 16, "kv_heads": 8, "dim": 128, "users": 2, "each": 1,
         "prompt": 0, "prefix": 256, "own": 24, "row0": 0, "pad": 0},
        # Eight users of an 8B model, 1500 tokens of shared instructions, chats of up to 600 tokens.
        {"name": "attn_decode8", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "users": 8, "each": 1,
         "prompt": 0, "prefix": 1500, "own": 600, "row0": 0, "pad": 0},
        # Many users asking about one long document; the batch is padded to its captured size.
        {"name": "attn_decode64", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "users": 62, "each": 1,
         "prompt": 0, "prefix": 8192, "own": 1024, "row0": 0, "pad": 2},
        # Verification of four drafts for each of 16 users on a 14B model; rows at their absolute positions.
        {"name": "attn_verify16", "op": "attention", "heads": 40, "kv_heads": 8, "dim": 128, "users": 16, "each": 5,
         "prompt": 0, "prefix": 1999, "own": 301, "row0": 1999, "pad": 0},
        # Three prompts behind the shared instructions, packed into one 512-token forward.
        {"name": "attn_prompt512", "op": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "users": 3, "each": 0,
         "prompt": 512, "prefix": 2048, "own": 400, "row0": 0, "pad": 0},
        # A decode step of eight users with rank-16 adapters beside the 8B model's q|k|v projection.
        {"name": "lora_decode8", "op": "lora", "type": "f16", "n": 8, "adapters": 7, "rank": 16, "cols": 4096,
         "rows": 6144, "spread": "each"},
        # 64 users over 24 adapters of different ranks beside the 14B model's q|k|v projection.
        {"name": "lora_batch64", "op": "lora", "type": "bf16", "n": 64, "adapters": 24, "rank": 64, "cols": 5120,
         "rows": 7168, "spread": "each"},
        # A 512-token forward of prompts with three adapters beside the 8B model's gate|up projection.
        {"name": "lora_prompt512", "op": "lora", "type": "f16", "n": 512, "adapters": 3, "rank": 32, "cols": 4096,
         "rows": 24576, "spread": "runs"},
        # One chat with four drafts, sampled from the whole vocabulary.
        {"name": "verify_one", "op": "verify", "lanes": 1, "drafts": 4, "vocab": VOCAB, "draft": True, "ban": False},
        # 24 chats with up to eight drafts each, some greedy, part of the vocabulary masked by a grammar.
        {"name": "verify_batch24", "op": "verify", "lanes": 24, "drafts": 8, "vocab": VOCAB, "draft": True,
         "ban": True},
        # Drafts looked up in the prompt (no draft model), 16 chats.
        {"name": "verify_lookup16", "op": "verify", "lanes": 16, "drafts": 5, "vocab": VOCAB, "draft": False,
         "ban": False},
        # 32 chats with the usual sampling parameters: rows cut to their top 40.
        {"name": "topk_batch32", "op": "topk", "lanes": 32, "drafts": 8, "vocab": VOCAB, "k": 40, "draft": True},
    ]


# What the largest listed cases cost: scored (row, key) pairs, multiply-adds, logits.
MOST_PAIRS, MOST_MACS, MOST_LOGITS = 512 * 32 * 2448, 512 * 32 * (4096 + 24576), 240 * VOCAB


def log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "lora", "lora", "verify", "verify", "topk"])
    if op == "attention":
        heads, kv = rng.choice([(16, 8), (32, 8), (32, 8), (40, 8), (8, 2), (4, 2)])
        c = {"op": op, "heads": heads, "kv_heads": kv, "dim": rng.choice([64, 128, 128, 128]), "users": log_int(rng, 1, 64),
             "each": rng.choice([1, 1, 1, log_int(rng, 2, 9), 0]), "prompt": 0, "prefix": log_int(rng, 16, 12000),
             "own": log_int(rng, 9, 1500), "row0": 0, "pad": rng.choice([0, 0, rng.randint(1, 3)])}
        if c["each"] == 0:
            c["users"] = min(c["users"], 8)
            c["prompt"] = log_int(rng, max(16, c["users"]), 512)
            c["own"] = max(c["own"], c["prompt"])
        n = c["prompt"] or c["users"] * c["each"]
        c["prefix"] = min(c["prefix"], max(16, MOST_PAIRS // (n * heads) - c["own"]))
        if c["prefix"] < 2100:
            c["row0"] = rng.choice([0, c["prefix"], rng.randint(0, 40)])
        return c
    if op == "lora":
        cols, rows = rng.choice([(1024, 4096), (2560, 6144), (4096, 6144), (4096, 4096), (5120, 7168), (4096, 24576),
                                 (9728, 2560), (12288, 4096), (32 * rng.randint(8, 160), 8 * rng.randint(16, 1200))])
        rank, n = rng.choice([8, 16, 16, 32, 64, rng.randint(1, 64)]), log_int(rng, 1, 512)
        return {"op": op, "type": rng.choice(["f16", "f16", "bf16", "f32"]), "cols": cols, "rows": rows, "rank": rank,
                "n": max(1, min(n, MOST_MACS // (rank * (cols + rows)))), "adapters": log_int(rng, 1, 32),
                "spread": "runs" if n > 64 else rng.choice(["each", "each", "runs"])}
    drafts = rng.randint(1, 8)
    c = {"op": op, "lanes": log_int(rng, 1, min(48, MOST_LOGITS // (VOCAB * (2 * drafts + 1)))), "drafts": drafts,
         "vocab": rng.choice([VOCAB, VOCAB, 32768, rng.randint(1000, 152000)]), "draft": rng.random() < 0.75}
    if op == "topk":
        return {**c, "k": rng.choice([40, 40, 20, 1, log_int(rng, 2, 1000)])}
    return {**c, "ban": rng.random() < 0.4}


# ---- layouts, from the case alone ----

def fraction(i):
    return (0.381966 * (i + 1)) % 1.0


def tokens_of(c):
    """Per user: its tokens in the batch and the rows of its own that the last of them sees."""
    if c["each"]:
        new = [c["each"]] * c["users"]
    else:
        w = [0.3 + fraction(i) for i in range(c["users"])]
        at = [round(c["prompt"] * sum(w[:i]) / sum(w)) for i in range(c["users"] + 1)]
        new = [b - a for a, b in zip(at, at[1:])]
    return [(m, c["own"] if i == 0 else max(m, round(c["own"] * (0.2 + 0.8 * fraction(i))))) for i, m in enumerate(new)]


def attention_layout(c):
    """seq and n_keys of every row of the batch; rows without a token have no keys."""
    seq, keys = [], []
    for i, (m, rows) in enumerate(tokens_of(c)):
        seq += [c["users"] - 1 - i] * m
        keys += [c["prefix"] + rows - m + j + 1 for j in range(m)]
    return seq + [0] * c["pad"], keys + [0] * c["pad"]


def lora_ranks(c):
    return [max(1, c["rank"] >> (i % 4 if c["adapters"] > 8 else 0)) for i in range(c["adapters"])]


def lora_ids(c):
    if c["spread"] == "each":
        return [-1 if t % 4 == 3 else t % c["adapters"] for t in range(c["n"])]
    return [min(t * (c["adapters"] + 1) // c["n"], c["adapters"]) % (c["adapters"] + 1) - 1 for t in range(c["n"])]


def drafts_of(c):
    """Per lane: its number of drafts."""
    return [c["drafts"] if i == 0 else 1 + int(c["drafts"] * fraction(i)) for i in range(c["lanes"])]


# ---- inputs ----

def generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cache(g, seqs, kv, rows, d):
    """One side of an int8 KV cache (K or V) as the KV write fills it: N(0, 1) rows, amax / 127 steps."""
    x = normal(g, seqs, kv, rows, d)
    s = x.abs().amax(-1) / 127
    return (x / s[..., None]).round().to(torch.int8), s.contiguous()


def prepare_attention(c, seed):
    g, n_seq, n_ctx = generator(seed), c["users"], c["row0"] + c["own"]
    seq, keys = attention_layout(c)
    d, n = c["dim"], len(seq)
    s = {"q": 1.5 * normal(g, n, c["heads"], d), "seq": ints(seq), "keys": ints(keys), "most": max(keys)}
    s["pk"], s["pks"] = cache(g, 2, c["kv_heads"], c["prefix"], d)
    s["pv"], s["pvs"] = cache(g, 2, c["kv_heads"], c["prefix"], d)
    s["k"], s["ks"] = cache(g, n_seq, c["kv_heads"], n_ctx, d)
    s["v"], s["vs"] = cache(g, n_seq, c["kv_heads"], n_ctx, d)
    s["out"] = torch.empty_like(s["q"])
    return s


def prepare_lora(c, seed):
    """Adapters as a program loads them: A [rank][cols] and B [rows][rank] of each behind one another in two buffers,
    and the table of their addresses."""
    g, t, ranks = generator(seed), D8[c["type"]], lora_ranks(c)
    cols, rows, n = c["cols"], c["rows"], c["n"]
    s = {"x": normal(g, n, cols), "base": normal(g, n, rows), "ids": ints(lora_ids(c)), "ranks": ints(ranks),
         "a": (normal(g, sum(ranks), cols) / math.sqrt(cols)).to(t),
         "b": (0.3 * normal(g, sum(ranks) * rows)).to(t), "rank": max(ranks)}
    s["x"][:, ::97] *= 6.0  # a few large channels
    s["scale"] = torch.tensor([2.0 / (1 + i % 3) for i in range(len(ranks))], device="cuda")
    s["first"] = ints([sum(ranks[:i]) for i in range(len(ranks))])
    words = torch.zeros(len(ranks), 3, dtype=torch.int64)
    words[:, 0] = s["a"].data_ptr() + s["first"].cpu().long() * cols * t.itemsize
    words[:, 1] = s["b"].data_ptr() + s["first"].cpu().long() * rows * t.itemsize
    words[:, 2] = s["scale"].cpu().view(torch.int32).long() | s["ranks"].cpu().long() << 32
    s["table"] = words.cuda()  # {const void* a, *b; float scale; int32_t rank}
    s["y"] = torch.empty_like(s["base"])
    return s


def lanes_of(c):
    """row, first, n_draft of every lane."""
    m = drafts_of(c)
    return [(sum(m[:i]) + i, sum(m[:i]), m[i]) for i in range(c["lanes"])]


def prepare_verify(c, seed):
    g, lanes, V = generator(seed), lanes_of(c), c["vocab"]
    n = sum(m for _, _, m in lanes)
    rows = n + c["lanes"]
    hold = [r + j for r, _, m in lanes for j in range(m)]  # the target row of every draft
    # Target logits: a flat background and some likely tokens; the draft's: the same, less well.
    z = 1.5 * normal(g, rows, V)
    peak = torch.randint(0, V, (rows, 12), generator=g, device="cuda")
    z.scatter_add_(1, peak, 12 + 2 * normal(g, rows, 12))
    w = z[ints(hold)] + 0.5 * normal(g, n, V)
    if c.get("ban"):
        ban = torch.rand(V, generator=g, device="cuda") < 0.5
        z[:, ban] = -math.inf
        w[:, ban] = -math.inf
    temp = [0.0 if i % 8 == 5 else 0.6 + 0.1 * (i % 7) for i in range(c["lanes"])]
    noise = -(-torch.rand(n, V, generator=g, device="cuda").clamp_min(1e-30).log()).log()
    t_row = torch.tensor([temp[i] for i, (_, _, m) in enumerate(lanes) for _ in range(m)], device="cuda")
    drafts = (w / t_row.clamp_min(1e-3)[:, None] + noise * (t_row > 0)[:, None]).argmax(1).int()
    s = {"drafts": drafts, "u": torch.rand(n, generator=g, device="cuda", dtype=torch.float64),
         "u_next": torch.rand(c["lanes"], generator=g, device="cuda", dtype=torch.float64), "most": c["drafts"],
         "row": ints([v[0] for v in lanes]), "first": ints([v[1] for v in lanes]), "n": ints([v[2] for v in lanes]),
         "temp": torch.tensor(temp, device="cuda"), "top": torch.tensor([0.05, 0.95], device="cuda"), "vocab": V}
    if c["op"] == "topk":
        k = min(c["k"], V)
        s["z"], s["z_id"] = torch.topk(z, k, dim=1)
        s["z_id"] = s["z_id"].int()
        s["w"], s["w_id"] = torch.topk(w, k, dim=1)
        s["w_id"] = s["w_id"].int()
        head = (s["w"] / t_row.clamp_min(1e-3)[:, None] + noise[:, :k] * (t_row > 0)[:, None]).argmax(1, keepdim=True)
        s["drafts"] = s["w_id"].gather(1, head)[:, 0].contiguous()
    else:
        s["z"], s["w"] = z, w
    if not c["draft"]:
        s["w"] = None
    table = torch.stack([s["row"], s["first"], s["n"], s["temp"].view(torch.int32)], 1)
    table = torch.cat([table, s["top"].view(torch.int32).expand(c["lanes"], 2)], 1)
    s["lanes"] = table.contiguous()  # mk_verify_lane
    s["accepted"] = torch.empty(c["lanes"], dtype=torch.int32, device="cuda")
    s["tokens"] = torch.empty(c["lanes"], c["drafts"] + 1, dtype=torch.int32, device="cuda")
    s["probs"] = torch.empty(c["lanes"], c["drafts"] + 1, device="cuda")
    return s


PREPARE = {"attention": prepare_attention, "lora": prepare_lora, "verify": prepare_verify, "topk": prepare_verify}


def prepare(case, seed):
    s = PREPARE[case["op"]](case, seed)
    s["case"] = dict(case)
    torch.cuda.synchronize()  # inputs made on torch's stream; the library works on its own
    return s


# ---- plain forms ----

def attention_plain(s):
    """Scores of the prefix for all rows at once, scores of each sequence's own rows, one softmax over both."""
    c = s["case"]
    n, H, d, KV, P = len(s["q"]), c["heads"], c["dim"], c["kv_heads"], c["prefix"]
    G, own_n = H // KV, s["most"] - P
    # K rows hold element e at byte d / 16 * (e % 16) + e / 16: the same order for q.
    q = s["q"].reshape(n, KV, G, d // 16, 16).transpose(-1, -2).reshape(n, KV, G, d) / math.sqrt(d)
    at = slice(c["row0"], c["row0"] + own_n)
    seq = s["seq"].long()
    k, v = (s[x][seq][:, :, at].float() * s[x + "s"][seq][:, :, at, None] for x in "kv")
    pk, pv = (s["p" + x][1].float() * s["p" + x + "s"][1][..., None] for x in "kv")
    qp = q.permute(1, 0, 2, 3).reshape(KV, n * G, d)
    sp = torch.bmm(qp, pk.transpose(1, 2).contiguous()).reshape(KV, n, G, P).transpose(0, 1)
    so = torch.bmm(q.reshape(n * KV, G, d), k.reshape(n * KV, own_n, d).transpose(1, 2).contiguous())
    sc = torch.cat([sp, so.reshape(n, KV, G, own_n)], -1)
    live = torch.arange(P + own_n, device="cuda") < s["keys"][:, None]
    sc = torch.where(live[:, None, None], sc, -math.inf)
    e = torch.exp(sc - sc.amax(-1, keepdim=True).clamp_min(-1e30))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    op = torch.bmm(p[..., :P].transpose(0, 1).reshape(KV, n * G, P), pv).reshape(KV, n, G, d).transpose(0, 1)
    oo = torch.bmm(p[..., P:].reshape(n * KV, G, own_n), v.reshape(n * KV, own_n, d)).reshape(n, KV, G, d)
    return {"out": (op + oo).reshape(n, H, d)}


def lora_plain(s):
    """All adapters of the batch as one pair of products, with the columns of other adapters' ranks zeroed."""
    c = s["case"]
    ranks, rows = s["ranks"].long(), c["rows"]
    total = s["a"].shape[0]
    owner = torch.repeat_interleave(torch.arange(len(ranks), device="cuda"), ranks, output_size=total)
    h = s["x"] @ s["a"].float().T
    h = torch.where(s["ids"][:, None] == owner, h * s["scale"][owner], 0.0)
    # Column j of B, all adapters side by side: element (row, j - first) of its adapter's [rows][rank] matrix.
    first = s["first"].long()[owner]
    j = torch.arange(total, device="cuda") - first
    at = first * rows + j + torch.arange(rows, device="cuda")[:, None] * ranks[owner]
    return {"y": s["base"] + h @ s["b"][at].float().T}


def first_of(hit, otherwise):
    """The first place along the last axis where `hit` holds."""
    m = hit.shape[-1]
    i = torch.where(hit, torch.arange(m, device=hit.device), m).amin(-1)
    return torch.where(i == m, otherwise, i)


def distribution(z, t):
    """softmax(z / t) of every row in 64 bits; t <= 0: all of it on the first maximum."""
    z, t = z.double(), t.double()[:, None]
    m = z.amax(-1, keepdim=True)
    e = torch.exp((z - m) / torch.where(t > 0, t, 1.0))
    cold = torch.arange(z.shape[1], device=z.device) == first_of(z == m, 0)[:, None]
    return torch.where(t > 0, e / e.sum(-1, keepdim=True), cold.double())


def emitted(s, n_acc, tail, tail_p, pd):
    """Accepted drafts, then the drawn token, then -1; and their probabilities."""
    j = torch.arange(s["most"] + 1, device="cuda")
    at = (s["first"][:, None] + j).clamp_max(len(s["drafts"]) - 1).long()
    a = n_acc[:, None]
    tokens = torch.where(j < a, s["drafts"][at], torch.where(j == a, tail[:, None].int(), -1))
    probs = torch.where(j < a, pd[at].float(), torch.where(j == a, tail_p[:, None].float(), 0.0))
    return {"accepted": n_acc.int(), "tokens": tokens, "probs": probs}


def owners(s):
    """The lane of every draft, and its place there."""
    n = len(s["drafts"])
    lane = torch.repeat_interleave(torch.arange(len(s["n"]), device="cuda"), s["n"].long(), output_size=n)
    return lane, torch.arange(n, device="cuda") - s["first"][lane].long()


def accepted_of(s, lane, place, ok):
    """Drafts accepted before each lane's first refusal."""
    grid = torch.zeros(len(s["n"]), s["most"] + 1, dtype=torch.bool, device="cuda")
    grid[lane, place] = ok
    return first_of(~grid, s["most"])


def verify_plain(s):
    lane, place = owners(s)
    row_lane = torch.repeat_interleave(torch.arange(len(s["n"]), device="cuda"), s["n"].long() + 1,
                                       output_size=len(s["z"]))
    P = distribution(s["z"], s["temp"][row_lane])
    d = s["drafts"].long()
    pd = P[s["row"][lane].long() + place, d]
    if s["w"] is not None:
        Q = distribution(s["w"], s["temp"][lane])
        qd = Q[torch.arange(len(d), device="cuda"), d]
    else:
        qd = torch.ones_like(pd)
    n_acc = accepted_of(s, lane, place, (qd > 0) & (s["u"] * qd < pd))
    p = P[s["row"].long() + n_acc]
    stop = (s["first"].long() + n_acc).clamp_max(len(d) - 1)
    refused = (n_acc < s["n"])[:, None]
    if s["w"] is not None:
        q = Q[stop]
    else:
        q = (torch.arange(s["vocab"], device="cuda") == d[stop][:, None]).double()
    r = (p - torch.where(refused, q, 0.0)).clamp_min(0.0)
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, p)
    run = r.cumsum(-1)
    last = s["vocab"] - 1 - first_of((r > 0).flip(-1), 0)
    tok = first_of((run >= s["u_next"][:, None] * run[:, -1:]) & (r > 0), last)
    return emitted(s, n_acc, tok, p.gather(1, tok[:, None])[:, 0], pd)


def cut(s, values, temp):
    """Probabilities of rows of candidates, highest first, as the sampler makes them: 32-bit weights, the head above
    min_p of the first up to top_p of their 64-bit total."""
    t = temp[:, None]
    hot = t > 0
    w = torch.exp(((values - values[:, :1]) / torch.where(hot, t, 1.0)).double()).float().double()
    run = w.cumsum(-1)
    k = torch.full((len(w),), w.shape[1], device="cuda")
    keep = torch.minimum(first_of(w < s["top"][0].double() * w[:, :1], k),
                         first_of(run >= s["top"][1].double() * run[:, -1:], k - 1) + 1)
    keep = torch.where(hot[:, 0], keep, 1)
    w = torch.where(torch.arange(w.shape[1], device="cuda") < keep[:, None], w, 0.0)
    return (w / w.sum(-1, keepdim=True)).float()


def topk_plain(s):
    lane, place = owners(s)
    row_lane = torch.repeat_interleave(torch.arange(len(s["n"]), device="cuda"), s["n"].long() + 1,
                                       output_size=len(s["z"]))
    P, d = cut(s, s["z"], s["temp"][row_lane]), s["drafts"]
    at = s["row"][lane].long() + place
    pd = torch.where(s["z_id"][at] == d[:, None], P[at], 0.0).sum(-1)
    if s["w"] is not None:
        Q = cut(s, s["w"], s["temp"][lane])
        qd = torch.where(s["w_id"] == d[:, None], Q, 0.0).sum(-1)
    else:
        qd = torch.ones_like(pd)
    n_acc = accepted_of(s, lane, place, (qd > 0) & (s["u"] * qd.double() < pd.double()))
    stop = (s["first"].long() + n_acc).clamp_max(len(d) - 1)
    p, ids = P[s["row"].long() + n_acc], s["z_id"][s["row"].long() + n_acc]
    if s["w"] is not None:
        q = torch.where(ids[:, :, None] == s["w_id"][stop][:, None, :], Q[stop][:, None, :], 0.0).sum(-1)
    else:
        q = (ids == d[stop][:, None]).float()
    r = (p - torch.where((n_acc < s["n"])[:, None], q, 0.0)).clamp_min(0.0)
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, p).double()
    run = r.cumsum(-1)
    last = r.shape[1] - 1 - first_of((r > 0).flip(-1), 0)
    i = first_of((run >= s["u_next"][:, None] * run[:, -1:]) & (r > 0), last)[:, None]
    return emitted(s, n_acc, ids.gather(1, i)[:, 0], p.gather(1, i)[:, 0], pd)


# ---- as a program calls them ----

_ctx = None


def library():
    """The native library and the program's one context."""
    global _ctx
    import malkin_amd as mk
    if _ctx is None:
        _ctx = mk.Context(0)
    return mk, mk.load(), _ctx.h


def workspace(s, nbytes):
    if "work" not in s:
        s["work"] = torch.empty(max(1, nbytes), dtype=torch.uint8, device="cuda")
    return s["work"].data_ptr(), s["work"].numel()


def ptr(t):
    return None if t is None else t.data_ptr()


def attention_own(s):
    mk, lib, ctx = library()
    if "call" not in s:
        import ctypes
        c = s["case"]
        H, d, KV = c["heads"], c["dim"], c["kv_heads"]

        def kv(k, v, ks, vs):
            return mk.MkKvCache(ptr(k), ptr(v), ptr(ks), ptr(vs), 1, k.shape[0], KV, d, k.shape[2])

        s["caches"] = kv(s["pk"], s["pv"], s["pks"], s["pvs"]), kv(s["k"], s["v"], s["ks"], s["vs"])
        pre, mine = (ctypes.byref(x) for x in s["caches"])
        n = len(s["q"])
        work = workspace(s, lib.mk_attention_prefix_workspace(n, H, KV, d, c["prefix"], s["most"]))
        s["call"] = (ctx, ptr(s["q"]), H * d, ptr(s["out"]), H * d, n, H, pre, 1, c["prefix"], mine, c["row0"], 0,
                     ptr(s["seq"]), ptr(s["keys"]), s["most"], None, *work)
    mk.check(lib.mk_attention_prefix(*s["call"]))
    return {"out": s["out"]}


def lora_own(s):
    mk, lib, ctx = library()
    if "call" not in s:
        c = s["case"]
        work = workspace(s, lib.mk_lora_workspace(c["n"], s["rank"], c["cols"]))
        kind = {"f32": mk.F32, "f16": mk.F16, "bf16": mk.BF16}[c["type"]]
        s["call"] = (ctx, kind, ptr(s["table"]), c["adapters"], s["rank"], ptr(s["ids"]), ptr(s["x"]), c["cols"], c["n"],
                     c["rows"], c["cols"], ptr(s["base"]), c["rows"], ptr(s["y"]), c["rows"], *work)
    mk.check(lib.mk_lora(*s["call"]))
    return {"y": s["y"]}


def verify_own(s):
    mk, lib, ctx = library()
    if "call" not in s:
        rows, n, lanes = len(s["z"]), len(s["drafts"]), len(s["n"])
        tail = (ptr(s["lanes"]), lanes, s["most"], ptr(s["drafts"]), ptr(s["u"]), ptr(s["u_next"]), ptr(s["accepted"]),
                ptr(s["tokens"]), ptr(s["probs"]))
        if "z_id" in s:
            k = s["z"].shape[1]
            q = s["w"] is not None
            s["call"] = (ctx, ptr(s["z"]), ptr(s["z_id"]), k, rows, ptr(s["w"]), ptr(s["w_id"]) if q else None, k, n,
                         *tail)
        else:
            work = workspace(s, lib.mk_verify_workspace(lanes, s["most"], s["vocab"]))
            s["call"] = (ctx, ptr(s["z"]), s["vocab"], rows, ptr(s["w"]), s["vocab"], n, s["vocab"], *tail, *work)
    mk.check((lib.mk_verify_topk if "z_id" in s else lib.mk_verify)(*s["call"]))
    return {"accepted": s["accepted"], "tokens": s["tokens"], "probs": s["probs"]}


PLAIN = {"attention": attention_plain, "lora": lora_plain, "verify": verify_plain, "topk": topk_plain}
OWN = {"attention": attention_own, "lora": lora_own, "verify": verify_own, "topk": verify_own}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ---- what a pass cannot do without ----

def work(case):
    c = case
    if c["op"] == "attention":
        seq, keys = attention_layout(c)
        row = c["kv_heads"] * 2 * (c["dim"] + 4)
        rows = c["prefix"] + sum(r for _, r in tokens_of(c))
        return {"bytes": 8 * len(seq) * c["heads"] * c["dim"] + rows * row + 8 * len(seq),
                "flops": 4 * c["heads"] * c["dim"] * sum(keys)}
    if c["op"] == "lora":
        ranks, ids = lora_ranks(c), lora_ids(c)
        size = {"f32": 4, "f16": 2, "bf16": 2}[c["type"]]
        used, width = sum(ranks[i] for i in set(ids) if i >= 0), c["cols"] + c["rows"]
        return {"bytes": used * width * size + 4 * c["n"] * (c["cols"] + 2 * c["rows"]) + 4 * c["n"],
                "flops": 2 * width * sum(ranks[i] for i in ids if i >= 0)}
    n = sum(drafts_of(c))
    out = 24 * n + c["lanes"] * (36 + 8 * (c["drafts"] + 1))
    rows = n + c["lanes"] + (n if c["draft"] else 0)
    if c["op"] == "topk":
        return {"bytes": 8 * rows * min(c["k"], c["vocab"]) + out, "flops": 8 * rows * min(c["k"], c["vocab"])}
    return {"bytes": 4 * rows * c["vocab"] + out, "flops": 8 * rows * c["vocab"]}


# ---- the same results in 64 bits ----

def exact_attention(c, seed):
    s = prepare_attention(c, seed)
    seq, keys = attention_layout(c)
    H, d, KV, P = c["heads"], c["dim"], c["kv_heads"], c["prefix"]
    byte = torch.arange(d, device="cuda")
    byte = d // 16 * (byte % 16) + byte // 16  # where a K row holds element e

    def rows(x, i, a, b):
        r = s[x][i, :, a:b].double() * s[x + "s"][i, :, a:b, None].double()
        return r[..., byte] if x.endswith("k") else r

    pre = [rows("pk", 1, 0, P), rows("pv", 1, 0, P)]
    out = torch.zeros(len(seq), H, d, dtype=torch.float64, device="cuda")
    for t, (i, m) in enumerate(zip(seq, keys)):
        if m == 0:
            continue
        k, v = (torch.cat([a, rows(x, i, c["row0"], c["row0"] + m - P)], 1) for a, x in zip(pre, "kv"))
        w = torch.softmax(s["q"][t].double().reshape(KV, H // KV, d) @ k.transpose(1, 2).contiguous() / d ** 0.5, -1)
        out[t] = (w @ v).reshape(H, d)
    return {"out": out}


def exact_lora(c, seed):
    s = prepare_lora(c, seed)
    y, ids, ranks, rows = s["base"].double(), lora_ids(c), lora_ranks(c), c["rows"]
    for i in sorted(set(ids) - {-1}):
        at = torch.tensor([t for t, j in enumerate(ids) if j == i], device="cuda")
        f, r = sum(ranks[:i]), ranks[i]
        a, b = s["a"][f:f + r].double(), s["b"][f * rows:(f + r) * rows].double().reshape(rows, r)
        y[at] += float(s["scale"][i]) * ((s["x"][at].double() @ a.T) @ b.T)
    return {"y": y}


def exact_verify(c, seed):
    s = prepare_verify(c, seed)
    acc, tokens, probs = [], [], []

    def dense(z, t):
        z = z.double()
        if t <= 0:
            p = torch.zeros_like(z)
            p[int((z == z.max()).nonzero()[0])] = 1.0
            return p
        return torch.softmax(z / t, -1)

    def listed_row(z, ids, t):
        p = torch.zeros(s["vocab"], dtype=torch.float64, device="cuda")
        if t <= 0:
            p[ids[0].long()] = 1.0
            return p
        w = torch.exp((z.double() - z[0].double()) / t)
        lo, hi = (float(x) for x in s["top"])
        keep, total, run = 0, float(w.sum()), 0.0
        for x in w.tolist():
            if keep and x < lo * float(w[0]):
                break
            run, keep = run + x, keep + 1
            if run >= hi * total:
                break
        p[ids[:keep].long()] = w[:keep] / w[:keep].sum()
        return p

    for i, (row, first, m) in enumerate(lanes_of(c)):
        t = float(s["temp"][i])
        top = c["op"] == "topk"

        def target(j):
            return listed_row(s["z"][row + j], s["z_id"][row + j], t) if top else dense(s["z"][row + j], t)

        def draft(j):
            if s["w"] is None:
                q = torch.zeros(s["vocab"], dtype=torch.float64, device="cuda")
                q[int(s["drafts"][first + j])] = 1.0
                return q
            return listed_row(s["w"][first + j], s["w_id"][first + j], t) if top else dense(s["w"][first + j], t)

        out, pr, p = [], [], target(0)
        for j in range(m):
            q, x = draft(j), int(s["drafts"][first + j])
            if not (float(q[x]) > 0 and float(s["u"][first + j]) * float(q[x]) < float(p[x])):
                r = (p - q).clamp_min(0.0)
                break
            out.append(x)
            pr.append(float(p[x]))
            r = p = target(j + 1)
        r = r if float(r.sum()) > 0 else p
        # Candidates are walked in their order, highest first, a whole vocabulary in the order of its ids.
        order = s["z_id"][row + len(out)].long() if top else torch.arange(s["vocab"], device="cuda")
        r = r[order]
        run = r.cumsum(0)
        hit = ((run >= float(s["u_next"][i]) * run[-1]) & (r > 0)).nonzero()
        x = int(order[hit[0] if len(hit) else (r > 0).nonzero()[-1]])
        acc.append(len(out))
        out.append(x)
        pr.append(float(p[x]))
        tokens.append(out + [-1] * (c["drafts"] + 1 - len(out)))
        probs.append(pr + [0.0] * (c["drafts"] + 1 - len(pr)))
    return {"accepted": ints(acc), "tokens": ints(tokens),
            "probs": torch.tensor(probs, dtype=torch.float64, device="cuda")}


def exact(case, seed):
    f = {"attention": exact_attention, "lora": exact_lora}.get(case["op"], exact_verify)
    return f(case, seed)
