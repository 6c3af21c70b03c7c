"""Attention and token-probability cases: the calls that a program decoding
with a paged key-value cache makes between the ternary projections and after
the LM head, through the package's public entry points.

Kinds (the `kind` of a case):
  append    `kv_append`: rotary embedding of the new tokens' queries and keys,
            keys and values written into the pages of their sequences
  attention `paged_attention`: one query token per row over the pages of its
            sequence; with `accumulate` also the attention weight that every
            cached position received, added to the cache's scores
  evict     `kv_evict`: each sequence cut down to `budget` positions per
            key-value head, the first `sink`, the last `recent` and those of
            the highest scores between them
  logprobs  `token_logprobs`: log probabilities of given tokens, entropy and
            the `top` most likely tokens of each row of logits
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
ROPE_BASE = 10000.0


def _xtern():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xor-net_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import xtern
    return xtern


# --- the cases -------------------------------------------------------------
# Lengths: sequence i of S holds max_len * (1 - ragged * u_i) positions, u_i
# spread over [0, 1); ragged = 0 gives them all max_len.

def listed():
    return [
        # one decoded token of a 2560-wide model (20 query heads, 5 key-value
        # heads of 128): the smallest call, launch latency alone
        dict(name="append_token", kind="append", dtype="bf16", R=1, S=1, hq=20, hkv=5, D=128, page=16,
             max_len=700, skip=0),
        # a decode batch of a 3200-wide model, heads of 100 and a cache kept
        # in f32; every seventh row is padding
        dict(name="append_ragged", kind="append", dtype="f32", R=77, S=77, hq=32, hkv=32, D=100, page=24,
             max_len=300, skip=7),
        # a chunk of 4096 prompt tokens of eight sequences, 4096-wide model
        dict(name="append_prompt", kind="append", dtype="f16", R=4096, S=8, hq=32, hkv=8, D=128, page=64,
             max_len=2048, skip=0),
        # one token of one chat of the 2560-wide model
        dict(name="attn_token", kind="attention", dtype="bf16", R=1, hq=20, hkv=5, D=128, page=16,
             max_len=700, ragged=0.0, accumulate=False),
        # one token behind a document of 131072 tokens: few rows, a long axis
        dict(name="attn_long", kind="attention", dtype="bf16", R=1, hq=32, hkv=8, D=128, page=64,
             max_len=131072, ragged=0.0, accumulate=False),
        # a serving batch of 64 sequences of very different lengths
        dict(name="attn_batch", kind="attention", dtype="f16", R=64, hq=32, hkv=8, D=128, page=32,
             max_len=8192, ragged=1.0, accumulate=False),
        # heads of 100 that share nothing, f32 cache, odd pages, the weights
        # of every position accumulated for a later eviction
        dict(name="attn_scores", kind="attention", dtype="f32", R=9, hq=32, hkv=32, D=100, page=24,
             max_len=2500, ragged=0.7, accumulate=True),
        # one chat cut from about a thousand positions to half
        dict(name="evict_chat", kind="evict", dtype="bf16", S=1, hkv=5, D=128, page=16, max_len=1027,
             ragged=0.0, budget=512, sink=4, recent=64),
        # a serving batch cut to 2048 positions, some of it short already
        dict(name="evict_batch", kind="evict", dtype="f16", S=32, hkv=8, D=128, page=32, max_len=8192,
             ragged=1.0, budget=2048, sink=4, recent=256),
        # the logits of one decoded token, its 20 most likely alternatives
        dict(name="logprobs_token", kind="logprobs", dtype="f32", M=1, V=128256, T=1, top=20, masked=0.0),
        # four answers scored under a third of the vocabulary, half precision,
        # rows that no vector width divides
        dict(name="logprobs_masked", kind="logprobs", dtype="f16", M=37, V=32003, T=4, top=5, masked=0.67),
        # a 1024-token text scored token by token
        dict(name="logprobs_text", kind="logprobs", dtype="f32", M=1024, V=128256, T=1, top=1, masked=0.0),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    """Query heads, key-value heads and head size: of the listed models, and
    other ratios and sizes."""
    hkv = rng.choice([1, 2, 4, 5, 8])
    return hkv * rng.choice([1, 2, 4, 5, 8, 12]), hkv, rng.choice([64, 80, 96, 100, 128, 128, 192, 256])


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "evict", "logprobs"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "logprobs":
        M, V = _log(rng, 1, 1024), _log(rng, 1000, 200000)
        M = max(1, min(M, 1024 * 128256 // V))
        return dict(kind=kind, dtype=dtype, M=M, V=V, T=rng.choice([1, 1, 4]), top=rng.choice([0, 1, 5, 20, 64]),
                    masked=rng.choice([0.0, 0.5, 0.99]))
    hq, hkv, D = _heads(rng)
    page = rng.choice([1, 8, 16, 24, 32, 64, 128])
    row = 2 * hkv * D * SIZE[dtype]  # cached bytes of one position
    if kind == "append":
        S = _log(rng, 1, 64)
        R = min(S * _log(rng, 1, 512), 4096, max(1, (1 << 27) // (8 * D * (hq + hkv))))
        S = min(S, R)
        return dict(kind=kind, dtype=dtype, R=R, S=S, hq=hq, hkv=hkv, D=D, page=page,
                    max_len=_log(rng, 600, 4000), skip=rng.choice([0, 0, 5]))
    S, L = _log(rng, 1, 64), _log(rng, 1 if kind == "attention" else 64, 100000)
    if kind == "attention":
        L = max(1, min(L, (1 << 29) // (S * row)))
        return dict(kind=kind, dtype=dtype, R=S, hq=hq, hkv=hkv, D=D, page=page, max_len=L,
                    ragged=rng.choice([0.0, 0.5, 1.0]), accumulate=rng.random() < 0.4)
    L = max(64, min(L, (1 << 29) // (S * row)))
    budget = max(16, int(L * rng.uniform(0.2, 0.9)))
    return dict(kind=kind, dtype=dtype, S=S, hkv=hkv, D=D, page=page, max_len=L,
                ragged=rng.choice([0.0, 0.5, 1.0]), budget=budget, sink=rng.choice([0, 4]),
                recent=rng.choice([0, 1, budget // 4]))


# --- inputs ----------------------------------------------------------------

def _lengths(S, max_len, ragged):
    """Lengths of S sequences, the first of them the longest."""
    return [max(1, int(max_len * (1.0 - ragged * ((i * 0.6180339887) % 1.0)))) for i in range(S)]


def _pages(lens, page):
    return sum((n + page - 1) // page for n in lens)


def _cache(g, c, lens, scores):
    """Pages in random order, keys and values of the written positions, the
    rest of the pool zero; [page][head][slot][d] in memory, seen as
    [page][slot][head][d]."""
    page, hkv, D = c["page"], c["hkv"], c["D"]
    per = [(n + page - 1) // page for n in lens]
    total, widest = sum(per), max(per)
    perm = torch.randperm(total + 2, generator=g, device=DEV)[:total].to(torch.int32)
    table = torch.full((len(lens), widest), -1, dtype=torch.int32, device=DEV)
    at = torch.arange(widest, device=DEV)[None, :]
    per_t = torch.tensor(per, device=DEV)[:, None]
    start = torch.cumsum(per_t, 0) - per_t
    table = torch.where(at < per_t, perm[(start + at).clamp(max=total - 1)], table).contiguous()
    shape = (total + 2, hkv, page, D)
    k = torch.empty(shape, dtype=DTYPES[c["dtype"]], device=DEV).normal_(generator=g)
    v = torch.empty(shape, dtype=DTYPES[c["dtype"]], device=DEV).normal_(generator=g)
    score = None
    if scores:  # accumulated weights: heavy-tailed, many near zero
        score = torch.rand(shape[:3], generator=g, device=DEV).pow_(6)
    return k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3), score, table


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    f32 = dict(dtype=torch.float32, device=DEV)
    s = dict(case=c)
    if c["kind"] == "logprobs":
        x = torch.empty((c["M"], c["V"]), **f32).normal_(generator=g).mul_(2.5)
        # a few tokens that the model is sure of, more or less
        hot = torch.randint(0, c["V"], (c["M"], 3), generator=g, device=DEV)
        x.scatter_add_(1, hot, 12.0 * torch.rand((c["M"], 3), generator=g, device=DEV))
        if c["masked"]:
            x.masked_fill_(torch.rand(x.shape, generator=g, device=DEV) < c["masked"], -math.inf)
        s["logits"] = x.to(DTYPES[c["dtype"]])
        t = torch.randint(0, c["V"], (c["M"], c["T"]), generator=g, device=DEV)
        t[:, 0] = hot[:, 0]
        s["tokens"] = t.to(torch.int32)
        return s
    if c["kind"] == "append":
        S, R = c["S"], c["R"]
        each = -(-R // S)
        rows = torch.arange(R, device=DEV)
        base = _lengths(S, max(1, c["max_len"] - each), 0.5)  # cached before the call
        k, v, score, table = _cache(g, c, [n + each for n in base], False)
        seq = rows // each
        slots = torch.tensor(base, device=DEV)[seq] + rows % each
        s["positions"] = slots.to(torch.int32)
        if c["skip"]:
            slots = torch.where(rows % c["skip"] == c["skip"] - 1, -1, slots)
        s.update(k_cache=k, v_cache=v, table=table, seq=seq.to(torch.int32), slots=slots.to(torch.int32))
        s["q"] = torch.empty((R, c["hq"], c["D"]), **f32).normal_(generator=g)
        s["k"] = torch.empty((R, c["hkv"], c["D"]), **f32).normal_(generator=g)
        s["v"] = torch.empty((R, c["hkv"], c["D"]), **f32).normal_(generator=g)
        freq = ROPE_BASE ** (-torch.arange(0, c["D"], 2, dtype=torch.float64, device=DEV) / c["D"])
        angle = torch.arange(c["max_len"] + each, dtype=torch.float64, device=DEV)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_out"] = torch.zeros_like(s["q"])
    else:
        lens = _lengths(c.get("R") or c["S"], c["max_len"], c["ragged"])
        k, v, score, table = _cache(g, c, lens, c["kind"] == "evict" or c["accumulate"])
        s.update(k_cache=k, v_cache=v, score=score, table=table,
                 lengths=torch.tensor(lens, dtype=torch.int32, device=DEV))
        if c["kind"] == "attention":
            # (a spread of two: some heads look at few positions, some at many)
            spread = torch.rand((1, c["hq"], 1), generator=g, device=DEV) * 2
            s["q"] = torch.empty((c["R"], c["hq"], c["D"]), **f32).normal_(generator=g) * spread
    if own:
        xtern = _xtern()
        s["cache"] = xtern.KvCache(s["k_cache"], s["v_cache"], s.get("score"))
    return s


# --- one pass --------------------------------------------------------------

def run(state):
    return globals()["_" + state["case"]["kind"]](state)


def _append(s):
    if own:
        _xtern().kv_append(s["cache"], s["table"], s["slots"], s["k"], s["v"], q=s["q"], seq=s["seq"],
                           positions=s["positions"], rope=(s["cos"], s["sin"]), q_out=s["q_out"])
        return s["q_out"], s["k_cache"], s["v_cache"]
    page, half = s["case"]["page"], s["case"]["D"] // 2
    rows = s["slots"] >= 0
    slots, seq = s["slots"][rows].long(), s["seq"][rows].long()
    at = s["positions"][rows].long()
    cos, sin = s["cos"][at][:, None, :], s["sin"][at][:, None, :]
    pages = s["table"][seq, slots // page].long()

    def turned(x):
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    s["q_out"][rows] = turned(s["q"][rows])
    s["k_cache"][pages, slots % page] = turned(s["k"][rows]).to(s["k_cache"].dtype)
    s["v_cache"][pages, slots % page] = s["v"][rows].to(s["v_cache"].dtype)
    return s["q_out"], s["k_cache"], s["v_cache"]


def _attention(s):
    c = s["case"]
    if own:
        o, lse = _xtern().paged_attention(s["cache"], s["table"], s["lengths"], s["q"], lse=True,
                                          accumulate=c["accumulate"])
        return (o, lse, s["score"]) if c["accumulate"] else (o, lse)
    R, hq, hkv, D, page = c["R"], c["hq"], c["hkv"], c["D"], c["page"]
    table = s["table"].long().clamp(min=0)
    L = table.shape[1] * page
    valid = (torch.arange(L, device=DEV)[None, :] < s["lengths"][:, None])[:, None, None, :]
    k = s["k_cache"][table].float().reshape(R, L, hkv, D).permute(0, 2, 3, 1)
    q = s["q"].reshape(R, hkv, hq // hkv, D) * (1.0 / math.sqrt(D))
    x = torch.matmul(q, k).masked_fill(~valid, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    l = e.sum(-1, keepdim=True)
    p = e / l
    v = s["v_cache"][table].float().reshape(R, L, hkv, D).permute(0, 2, 1, 3)
    v = torch.where(valid.transpose(-1, -2), v, torch.zeros((), device=DEV))
    o = torch.matmul(p, v).reshape(R, hq, D)
    lse = (m + torch.log(l)).reshape(R, hq)
    if not c["accumulate"]:
        return o, lse
    # [R, hkv, L] weights -> the pages' [hkv, page] scores; every written page
    # belongs to one sequence
    w = p.sum(2).reshape(R, hkv, -1, page).permute(0, 2, 1, 3)
    there = s["table"] >= 0
    s["score"].index_add_(0, table[there], w[there])
    return o, lse, s["score"]


def _evict(s):
    c = s["case"]
    if own:
        lens, kept = _xtern().kv_evict(s["cache"], s["table"], s["lengths"], c["budget"], sink=c["sink"],
                                       recent=c["recent"])
        return lens, kept, s["k_cache"], s["v_cache"], s["score"]
    S, hkv, page, budget = c["S"], c["hkv"], c["page"], c["budget"]
    table = s["table"].long().clamp(min=0)
    L = table.shape[1] * page
    at = torch.arange(L, device=DEV)[None, :]
    n = s["lengths"].long()[:, None]
    score = s["score"][table].permute(0, 2, 1, 3).reshape(S, hkv, L)
    always = (at < c["sink"]) | (at >= n - c["recent"])
    score = torch.where(always[:, None, :], math.inf, score)
    score = torch.where((at < n)[:, None, :], score, -math.inf)
    take = min(budget, L)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :take]
    best = torch.sort(best, dim=-1).values
    short = (n <= budget)[:, None, :]  # sequences that stay as they are
    rank = torch.arange(take, device=DEV)
    best = torch.where(short, rank, best)
    kept = torch.full((S, hkv, budget), -1, dtype=torch.int32, device=DEV)
    kept[..., :take] = torch.where(rank < n[:, None, :], best, -1).to(torch.int32)
    moved = (~short) & (rank < budget)
    b, h, to = torch.nonzero(moved.expand(S, hkv, take), as_tuple=True)
    src = best[b, h, to]
    from_page, to_page = table[b, src // page], table[b, to // page]
    rows = s["k_cache"][from_page, src % page, h], s["v_cache"][from_page, src % page, h]
    old = s["score"][from_page, h, src % page]
    s["k_cache"][to_page, to % page, h], s["v_cache"][to_page, to % page, h] = rows
    s["score"][to_page, h, to % page] = old
    return n[:, 0].clamp(max=budget).to(torch.int32), kept, s["k_cache"], s["v_cache"], s["score"]


def _logprobs(s):
    c = s["case"]
    if own:
        lp, entropy, ids, top = _xtern().token_logprobs(s["logits"], s["tokens"], top=c["top"])
        return (lp, entropy, ids, top) if c["top"] else (lp, entropy)
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    z = torch.where(x == -math.inf, 0.0, x - m)
    e = torch.where(x == -math.inf, 0.0, torch.exp(z))
    total = e.sum(-1, keepdim=True)
    lse = torch.log(total)
    lp = x.gather(1, s["tokens"].long()) - m - lse
    entropy = lse[:, 0] - (e * z).sum(-1) / total[:, 0]
    if not c["top"]:
        return lp, entropy
    best = torch.sort(x, dim=-1, descending=True, stable=True)
    return lp, entropy, best.indices[:, :c["top"]].to(torch.int32), best.values[:, :c["top"]] - m - lse


# --- what a pass cannot do without -----------------------------------------

def work(case):
    c = case
    if c["kind"] == "logprobs":
        return dict(bytes=c["M"] * (c["V"] * SIZE[c["dtype"]] + 8 * c["T"] + 4 + 8 * c["top"]),
                    flops=6 * c["M"] * c["V"])
    es, D, hkv = SIZE[c["dtype"]], c["D"], c["hkv"]
    if c["kind"] == "append":
        R = c["R"] - (c["R"] // c["skip"] if c["skip"] else 0)
        return dict(bytes=R * (8 * c["hq"] * D + 8 * hkv * D + 2 * es * hkv * D + 4 * D + 12),
                    flops=3 * R * (c["hq"] + hkv) * D)
    lens = _lengths(c.get("R") or c["S"], c["max_len"], c["ragged"])
    n = sum(lens)
    if c["kind"] == "attention":
        b = n * hkv * 2 * D * es + 4 * _pages(lens, c["page"]) + c["R"] * c["hq"] * (8 * D + 4)
        return dict(bytes=b + (8 * n * hkv if c["accumulate"] else 0), flops=4 * n * c["hq"] * D)
    long = [x for x in lens if x > c["budget"]]
    moved = len(long) * (c["budget"] - min(c["sink"], c["budget"]))
    return dict(bytes=hkv * (4 * sum(long) + 2 * moved * (2 * D * es + 4) + 4 * c["budget"] * c["S"]) + 8 * c["S"],
                flops=n * hkv)


# --- the definition in 64 bits ---------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["kind"] == "logprobs":
        lps, ents, tops = [], [], []
        for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
            p = torch.softmax(x.double(), -1)
            # ln p from the logits: p itself underflows
            lse = torch.logsumexp(x.double(), -1)
            lps.append(torch.gather(x.double(), 1, t.long()) - lse[:, None])
            ents.append(torch.special.entr(p).sum(-1))
            if c["top"]:
                tops.append(torch.topk(x.double(), c["top"]).values - lse[:, None])
        out = [torch.cat(lps), torch.cat(ents)]
        return out + [None, torch.cat(tops)] if c["top"] else out
    page, D = c["page"], c["D"]
    table, kc, vc = s["table"].tolist(), s["k_cache"], s["v_cache"]
    if c["kind"] == "append":
        out, kc, vc = s["q_out"].double(), kc.double(), vc.double()
        slots, seq, pos = s["slots"].tolist(), s["seq"].tolist(), s["positions"].tolist()
        rows = [r for r in range(c["R"]) if slots[r] >= 0]
        where = torch.tensor([[table[seq[r]][slots[r] // page], slots[r] % page] for r in rows], device=DEV)
        rows_t = torch.tensor(rows, device=DEV)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[torch.tensor([pos[r] for r in rows], device=DEV)]

        def rotate(x):
            z = torch.complex(*x.double().split(D // 2, -1)) * turn[:, None, :]
            return torch.cat([z.real, z.imag], -1)

        out[rows_t] = rotate(s["q"][rows_t])
        kc[where[:, 0], where[:, 1]] = rotate(s["k"][rows_t])
        vc[where[:, 0], where[:, 1]] = s["v"][rows_t].double()
        return out, kc, vc
    lens = s["lengths"].tolist()
    if c["kind"] == "attention":
        G = c["hq"] // c["hkv"]
        outs, lses, score = [], [], None
        if c["accumulate"]:
            score = s["score"].double()
        for r, n in enumerate(lens):
            pages = torch.tensor(table[r][:-(-n // page)], device=DEV)
            k = kc[pages].flatten(0, 1)[:n].double()
            v = vc[pages].flatten(0, 1)[:n].double()
            o, l = [], []
            for h in range(c["hkv"]):
                x = s["q"][r, h * G:(h + 1) * G].double() @ k[:, h].t() / math.sqrt(D)
                w = torch.softmax(x, -1)
                o.append(w @ v[:, h])
                l.append(torch.logsumexp(x, -1))
                if score is not None:
                    full = torch.zeros(len(pages) * page, dtype=torch.float64, device=DEV)
                    full[:n] = w.sum(0)
                    score[pages, h] += full.view(-1, page)
            outs.append(torch.cat(o))
            lses.append(torch.cat(l))
        out = [torch.stack(outs), torch.stack(lses)]
        return out if score is None else out + [score]
    # eviction moves what is there, no number of it is computed
    return None
