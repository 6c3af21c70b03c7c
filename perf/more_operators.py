"""Cases of a decode step over a cache held in 8 bits, and of the tokens that a
smaller model drafted for it: the calls between the ternary projections and
after the LM head, through the package's public entry points.

Kinds (the `kind` of a case):
  store      `kv_append` into an 8-bit cache: norms of the new tokens' query and
             key heads, rotation, one scale for each token and head; and
             `kv_read` of the new keys and values as the cache now holds them
  read       `kv_read` of a range of cached positions
  attention  `paged_attention` over an 8-bit or a 16-bit cache, with a window of
             the newest positions and the first few that stay visible, and with
             several tokens of a sequence (drafts, a chunk of a prompt) at once
  verify     `verify_drafts`: drafted tokens accepted or not by the target's
             probabilities and given random numbers, and one token drawn after
             the last one that was
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
ROPE_BASE = 10000.0
EPS = 1e-6
LEAST = 2.0 ** -119  # a head whose largest magnitude is below this is held as zeros


def _xtern():
    if "xtern" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xor-net_amd"))
    import xtern
    return xtern


# --- the cases -------------------------------------------------------------
# Lengths: sequence i of S holds max_len * (1 - ragged * u_i) positions, u_i
# spread over [0, 1); ragged = 0 gives them all max_len.  tokens: new tokens of
# each sequence, the last of them at its last position.

def listed():
    return [
        # one decoded token of a 2560-wide model (20 query heads, 5 key-value
        # heads of 128): the smallest call, launch latency alone
        dict(name="store_token", kind="store", R=1, S=1, hq=20, hkv=5, D=128, rot=128, norm=True, page=16,
             max_len=700, skip=0, out="bf16"),
        # a decode batch of a 3200-wide model, heads of 100 that are rotated in
        # part and have no norms; every seventh row is padding
        dict(name="store_ragged", kind="store", R=77, S=77, hq=32, hkv=32, D=100, rot=50, norm=False, page=24,
             max_len=300, skip=7, out="f32"),
        # a chunk of 4096 prompt tokens of eight sequences, 4096-wide model
        dict(name="store_prompt", kind="store", R=4096, S=8, hq=32, hkv=8, D=128, rot=128, norm=True, page=64,
             max_len=2048, skip=0, out="bf16"),
        # a short conversation handed to another process
        dict(name="read_chat", kind="read", S=1, n=701, hkv=5, D=128, page=16, out="f16"),
        # a shared prefix of 65536 tokens read back at full width
        dict(name="read_long", kind="read", S=1, n=65536, hkv=8, D=128, page=64, out="bf16"),
        # one token of one chat of the 2560-wide model
        dict(name="attn_token", kind="attention", dtype="i8", S=1, tokens=1, hq=20, hkv=5, D=128, page=16,
             max_len=700, ragged=0.0, window=0, sink=0),
        # one token behind a document of 131072 tokens: few rows, a long axis
        dict(name="attn_long", kind="attention", dtype="i8", S=1, tokens=1, hq=32, hkv=8, D=128, page=64,
             max_len=131072, ragged=0.0, window=0, sink=0),
        # a serving batch of 64 sequences of very different lengths
        dict(name="attn_batch", kind="attention", dtype="i8", S=64, tokens=1, hq=32, hkv=8, D=128, page=32,
             max_len=8192, ragged=1.0, window=0, sink=0),
        # four drafted tokens and the one before them of 24 sequences, a layer
        # that sees the newest 1024 positions and the first 4
        dict(name="attn_drafts", kind="attention", dtype="i8", S=24, tokens=5, hq=20, hkv=5, D=128, page=16,
             max_len=4001, ragged=0.8, window=1024, sink=4),
        # a windowed layer over a 16-bit cache, odd pages, some sequences
        # shorter than the window
        dict(name="attn_window", kind="attention", dtype="bf16", S=33, tokens=1, hq=32, hkv=8, D=100, page=24,
             max_len=30011, ragged=1.0, window=4096, sink=4),
        # four drafts of one chat, verified with the draft model's logits
        dict(name="verify_one", kind="verify", dtype="f32", S=1, T=4, V=128256, draft=True, masked=0.0, temps=False),
        # four drafts each of 64 sequences of their own temperatures (some take
        # the most likely token), rows that no vector width divides
        dict(name="verify_batch", kind="verify", dtype="bf16", S=64, T=4, V=128003, draft=True, masked=0.3,
             temps=True),
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
    kind = rng.choice(["store", "read", "attention", "attention", "verify"])
    if kind == "verify":
        S, T, V = _log(rng, 1, 64), rng.choice([0, 1, 3, 4, 8]), _log(rng, 1000, 200000)
        S = max(1, min(S, 64 * 9 * 128003 // (V * (2 * T + 1))))
        return dict(kind=kind, dtype=rng.choice(["f32", "f16", "bf16"]), S=S, T=T, V=V,
                    draft=rng.random() < 0.6, masked=rng.choice([0.0, 0.5, 0.99]), temps=rng.random() < 0.5)
    hq, hkv, D = _heads(rng)
    page = rng.choice([1, 8, 16, 24, 32, 64, 128])
    if kind == "store":
        S = _log(rng, 1, 64)
        R = min(S * _log(rng, 1, 512), 4096, max(1, (1 << 27) // (8 * D * (hq + hkv))))
        return dict(kind=kind, R=R, S=min(S, R), hq=hq, hkv=hkv, D=D, rot=rng.choice([0, D, D, D // 4 * 2]),
                    norm=rng.random() < 0.7, page=page, max_len=_log(rng, 600, 4000), skip=rng.choice([0, 0, 5]),
                    out=rng.choice(["f32", "f16", "bf16"]))
    if kind == "read":
        S, out = _log(rng, 1, 32), rng.choice(["f32", "f16", "bf16"])
        n = min(_log(rng, 1, 65536), 400_000_000 // (S * hkv * (2 * D + 8 + 2 * D * SIZE[out])))
        return dict(kind=kind, S=S, n=n, hkv=hkv, D=D, page=page, out=out)
    dtype = rng.choice(["i8", "i8", "i8", "f32", "f16", "bf16"])
    S, L, tokens = _log(rng, 1, 64), _log(rng, 1, 100000), rng.choice([1, 1, 2, 5, 8, 33])
    L = max(tokens, min(L, (1 << 28) // (S * 2 * hkv * D * SIZE[dtype])))
    while tokens > 1 and (S * L * tokens * hq > 1 << 25 or S * tokens > 1024):
        tokens //= 2
    window = rng.choice([0, 1, 100, 1024, 4096])
    return dict(kind=kind, dtype=dtype, S=S, tokens=tokens, hq=hq, hkv=hkv, D=D, page=page, max_len=L,
                ragged=rng.choice([0.0, 0.5, 1.0]), window=window, sink=rng.choice([0, 1, 4, 64]) if window else 0)


# --- inputs ----------------------------------------------------------------

def _lengths(S, max_len, ragged):
    """Lengths of S sequences, the first of them the longest."""
    return [max(1, int(max_len * (1.0 - ragged * ((i * 0.6180339887) % 1.0)))) for i in range(S)]


def _pages(lens, page):
    return sum((n + page - 1) // page for n in lens)


def _table(g, c, lens):
    """A page table of pages in random order, and the size of the pool."""
    page = c["page"]
    per = [(n + page - 1) // page for n in lens]
    total, widest = sum(per), max(per)
    perm = torch.randperm(total + 2, generator=g, device=DEV)[:total].to(torch.int32)
    at = torch.arange(widest, device=DEV)[None, :]
    per_t = torch.tensor(per, device=DEV)[:, None]
    start = torch.cumsum(per_t, 0) - per_t
    none = torch.full((), -1, dtype=torch.int32, device=DEV)
    return torch.where(at < per_t, perm[(start + at).clamp(max=total - 1)], none).contiguous(), total + 2


def _pool(g, c, pages, dtype):
    """Keys or values [page][head][slot][d] in memory, seen as
    [page][slot][head][d], and for an 8-bit pool the scales [page][head][slot].
    Some of a head's elements are larger than the others."""
    shape = (pages, c["hkv"], c["page"], c["D"])
    if dtype != "i8":
        return torch.empty(shape, dtype=DTYPES[dtype], device=DEV).normal_(generator=g).permute(0, 2, 1, 3), None
    x, scale = torch.empty(shape, dtype=torch.int8, device=DEV), torch.empty(shape[:3], device=DEV)
    wide = 1.0 + 3.0 * torch.rand((c["hkv"], 1, c["D"]), generator=g, device=DEV).pow_(8)
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for i in range(0, pages, step):
        y = torch.empty((min(step, pages - i),) + shape[1:], device=DEV).normal_(generator=g).mul_(wide)
        s = y.abs().amax(-1) / 127.0
        x[i:i + step] = torch.round(y / s[..., None]).to(torch.int8)
        scale[i:i + step] = s
    return x.permute(0, 2, 1, 3), scale


def _logits(g, shape, V, c, keep=None):
    x = torch.empty(shape + (V,), device=DEV).normal_(generator=g).mul_(2.5)
    # a few tokens that the model is sure of, more or less
    hot = torch.randint(0, V, shape + (3,), generator=g, device=DEV)
    x.scatter_add_(-1, hot, 12.0 * torch.rand(hot.shape, generator=g, device=DEV))
    if keep is not None:
        x.masked_fill_(~keep, -math.inf)
        x.scatter_(-1, hot[..., :1], 3.0)  # (something is left of every row)
    return x


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    f32 = dict(dtype=torch.float32, device=DEV)
    s = dict(case=c)
    if c["kind"] == "verify":
        S, T, V = c["S"], c["T"], c["V"]
        keep = None
        if c["masked"]:
            keep = torch.rand((S, 1, V), generator=g, device=DEV) >= c["masked"]
        x = _logits(g, (S, T + 1), V, c, keep)
        # the smaller model's logits: near the target's
        y = 0.9 * x[:, :T] + torch.empty((S, T, V), **f32).normal_(generator=g)
        s["target"] = x.to(DTYPES[c["dtype"]])
        s["draft"] = y.to(DTYPES[c["dtype"]]) if c["draft"] else None
        s["temperature"] = None
        if c["temps"]:
            s["temperature"] = 0.6 + 0.8 * torch.rand(S, generator=g, device=DEV)
            s["temperature"][::5] = 0.0
        # drawn from the draft's probabilities; without them the most likely
        # tokens, or any
        y = s["draft"].float() if c["draft"] else y
        noise = -torch.log(-torch.log(torch.rand((S, T, V), generator=g, device=DEV).clamp(1e-9, 1 - 1e-7)))
        s["drafted"] = (y + noise).argmax(-1).to(torch.int32) if T else torch.zeros((S, 0), dtype=torch.int32, device=DEV)
        s["uniforms"] = torch.rand((S, T + 1), generator=g, device=DEV)
        s["counts"] = None
        if S > 1 and T:  # some sequences have fewer drafts
            s["counts"] = torch.randint(T // 2, T + 1, (S,), generator=g, device=DEV).to(torch.int32)
        return s
    if c["kind"] == "store":
        S, R = c["S"], c["R"]
        each = -(-R // S)
        rows = torch.arange(R, device=DEV)
        base = _lengths(S, max(1, c["max_len"] - each), 0.5)  # cached before the call
        s["table"], pages = _table(g, c, [n + each for n in base])
        seq = rows // each
        slots = torch.tensor(base, device=DEV)[seq] + rows % each
        s["positions"] = slots.to(torch.int32)
        if c["skip"]:
            slots = torch.where(rows % c["skip"] == c["skip"] - 1, -1, slots)
        s.update(seq=seq.to(torch.int32), slots=slots.to(torch.int32))
        for name, h in (("q", c["hq"]), ("k", c["hkv"]), ("v", c["hkv"])):
            s[name] = torch.empty((R, h, c["D"]), **f32).normal_(generator=g)
        s["norm"] = s["rope"] = None
        if c["norm"]:
            s["norm"] = tuple(1.0 + 0.2 * torch.empty(c["D"], **f32).normal_(generator=g) for _ in range(2)) + (EPS,)
        if c["rot"]:
            freq = ROPE_BASE ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device=DEV) / c["rot"])
            angle = torch.arange(c["max_len"] + each, dtype=torch.float64, device=DEV)[:, None] * freq
            s["rope"] = angle.cos().float(), angle.sin().float()
        s["q_out"] = torch.zeros_like(s["q"])
        dtype = "i8"
    elif c["kind"] == "read":
        S, n = c["S"], c["n"]
        s["table"], pages = _table(g, c, [n] * S)
        rows = torch.arange(S * n, device=DEV)
        s.update(seq=(rows // n).to(torch.int32), slots=(rows % n).to(torch.int32))
        dtype = "i8"
    else:
        S, T, dtype = c["S"], c["tokens"], c["dtype"]
        lens = [max(T, n) for n in _lengths(S, c["max_len"], c["ragged"])]
        s["table"], pages = _table(g, c, lens)
        back = torch.arange(T - 1, -1, -1, device=DEV)
        s["lengths"] = (torch.tensor(lens, device=DEV)[:, None] - back).reshape(-1).to(torch.int32)
        # (a spread of two: some heads look at few positions, some at many)
        spread = torch.rand((1, c["hq"], 1), generator=g, device=DEV) * 2
        s["q"] = torch.empty((S * T, c["hq"], c["D"]), **f32).normal_(generator=g) * spread
        s["seq"] = torch.arange(S, device=DEV).repeat_interleave(T).to(torch.int32)
    s["k_cache"], s["k_scale"] = _pool(g, c, pages, dtype)
    s["v_cache"], s["v_scale"] = _pool(g, c, pages, dtype)
    if own:
        s["cache"] = _xtern().KvCache(s["k_cache"], s["v_cache"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return s


# --- one pass --------------------------------------------------------------

def run(state):
    return globals()["_" + state["case"]["kind"]](state)


def _store(s):
    c = s["case"]
    if own:
        xtern = _xtern()
        xtern.kv_append(s["cache"], s["table"], s["slots"], s["k"], s["v"], q=s["q"], seq=s["seq"],
                        positions=s["positions"], rope=s["rope"], norm=s["norm"], q_out=s["q_out"])
        k, v = xtern.kv_read(s["cache"], s["table"], s["slots"], seq=s["seq"], dtype=DTYPES[c["out"]])
        return s["q_out"], k, v
    # in 64 bits: a value next to the border of two codes falls where the exact
    # one does
    page, half = c["page"], c["rot"] // 2
    rows = s["slots"] >= 0
    slots, seq = s["slots"][rows].long(), s["seq"][rows].long()
    pages = s["table"][seq, slots // page].long()
    q, k, v = s["q"][rows].double(), s["k"][rows].double(), s["v"][rows].double()
    if c["norm"]:
        wq, wk, eps = s["norm"]
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + eps) * wq.double()
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + eps) * wk.double()
    if c["rot"]:
        at = s["positions"][rows].long()
        cos, sin = (t[at][:, None, :].double() for t in s["rope"])

        def turned(x):
            a, b = x[..., :half], x[..., half:2 * half]
            return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)

        q, k = turned(q), turned(k)

    def codes(x):
        top = x.float().abs().amax(-1).double()
        scale = torch.where(top < LEAST, 0.0, top / 127.0).float()
        y = torch.where(scale[..., None] == 0.0, 0.0, x / scale[..., None].double())
        return torch.round(y).to(torch.int8), scale

    s["q_out"][rows] = q.float()
    for x, cache, scales in ((k, s["k_cache"], s["k_scale"]), (v, s["v_cache"], s["v_scale"])):
        code, scale = codes(x)
        cache[pages, slots % page] = code
        scales[pages, :, slots % page] = scale
    return (s["q_out"],) + _values(s)


def _values(s):
    """Keys and values of the rows' positions; zeros for a row without one."""
    c = s["case"]
    there = s["slots"] >= 0
    slots = s["slots"].long().clamp(min=0)
    pages = s["table"][s["seq"].long(), slots // c["page"]].long().clamp(min=0)
    at = slots % c["page"]
    out = []
    for cache, scales in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])):
        x = cache[pages, at].float() * scales[pages, :, at][..., None]
        out.append(torch.where(there[:, None, None], x, 0.0).to(DTYPES[c["out"]]))
    return tuple(out)


def _read(s):
    if own:
        return _xtern().kv_read(s["cache"], s["table"], s["slots"], seq=s["seq"], dtype=DTYPES[s["case"]["out"]])
    return _values(s)


def _attention(s):
    c = s["case"]
    S, T, hq, hkv, D, page = c["S"], c["tokens"], c["hq"], c["hkv"], c["D"], c["page"]
    if own:
        return _xtern().paged_attention(s["cache"], s["table"], s["lengths"], s["q"], seq=s["seq"], lse=True,
                                        window=c["window"] or None, sink=c["sink"], tokens=T)
    n = s["lengths"].view(S, T, 1).long()
    L = s["table"].shape[1] * page
    if c["window"]:
        # the positions that some token of the sequence sees, side by side: the
        # first `sink`, and from the first token's window on
        start = (n[:, :1, 0] - c["window"]).clamp(min=c["sink"])
        L = min(L, c["sink"] + c["window"] + T - 1)
        i = torch.arange(L, device=DEV)[None, :]
        at = torch.where(i < c["sink"], i, start + i - c["sink"])[:, None, :]
        valid = (at < n) & ((at < c["sink"]) | (at >= n - c["window"]))
    else:
        at = torch.arange(L, device=DEV).expand(S, 1, L)
        valid = at < n
    inside = at[:, 0].clamp(max=s["table"].shape[1] * page - 1)
    pages = torch.gather(s["table"].long(), 1, inside // page).clamp(min=0)

    def cached(x, scale):
        y = x[pages, inside % page].float()
        if scale is not None:
            y = y * scale[pages, :, inside % page][..., None]
        seen = valid.any(1)[:, :, None, None]
        return torch.where(seen, y, 0.0).permute(0, 2, 1, 3)

    k = cached(s["k_cache"], s["k_scale"])
    q = s["q"].view(S, T, hkv, hq // hkv, D).permute(0, 2, 1, 3, 4).reshape(S, hkv, -1, D) * (1.0 / math.sqrt(D))
    x = torch.matmul(q, k.transpose(-1, -2)).view(S, hkv, T, -1, L).masked_fill(~valid[:, None, :, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    l = e.sum(-1, keepdim=True)
    v = cached(s["v_cache"], s["v_scale"])
    o = torch.matmul((e / l).reshape(S, hkv, -1, L), v).view(S, hkv, T, -1, D)
    lse = (m + torch.log(l))[..., 0]
    return o.permute(0, 2, 1, 3, 4).reshape(S * T, hq, D), lse.permute(0, 2, 1, 3).reshape(S * T, hq)


def _verify(s):
    c = s["case"]
    S, T, V = c["S"], c["T"], c["V"]
    if own:
        temperature = 1.0 if s["temperature"] is None else s["temperature"]
        return _xtern().verify_drafts(s["target"], s["drafted"], s["uniforms"], draft=s["draft"], counts=s["counts"],
                                      temperature=temperature)

    def chances(x):
        x = x.double()
        if s["temperature"] is None:
            t = torch.ones((S, 1, 1), dtype=torch.float64, device=DEV)
        else:
            t = s["temperature"].double()[:, None, None]
        first = torch.zeros_like(x).scatter_(-1, x.argmax(-1, keepdim=True), 1.0) if x.numel() else x
        x = x / torch.where(t == 0.0, 1.0, t)
        e = torch.exp(x - x.amax(-1, keepdim=True))
        return torch.where(t == 0.0, first, e / e.sum(-1, keepdim=True))

    p, u = chances(s["target"]), s["uniforms"].double()
    drafted = s["drafted"].long()
    count = torch.full((S,), T, device=DEV) if s["counts"] is None else s["counts"].long()
    one = torch.zeros((S, T, V), dtype=torch.float64, device=DEV).scatter_(-1, drafted[..., None], 1.0)
    q = one if s["draft"] is None else chances(s["draft"])
    px, qx = p[:, :T].gather(-1, drafted[..., None])[..., 0], q.gather(-1, drafted[..., None])[..., 0]
    taken = (u[:, :T] * qx < px) & (torch.arange(T, device=DEV) < count[:, None])
    n = taken.long().cumprod(-1).sum(-1)
    each = torch.arange(S, device=DEV)
    left = p[each, n]
    if T:
        less = torch.where((n < count)[:, None], q[each, n.clamp(max=T - 1)], 0.0)
        rest = (left - less).clamp(min=0.0)
        left = torch.where(rest.sum(-1, keepdim=True) > 0.0, rest, left)
    cum = left.cumsum(-1)
    new = (cum <= u[:, T:] * cum[:, -1:]).sum(-1).clamp(max=V - 1)
    place = torch.arange(T + 1, device=DEV)
    known = torch.cat([drafted, new[:, None]], 1)
    tokens = torch.where(place < n[:, None], known, torch.where(place == n[:, None], new[:, None], -1))
    lp = torch.log(p.gather(-1, tokens.clamp(min=0)[..., None])[..., 0])
    lp = torch.where(tokens < 0, 0.0, lp)
    return n.to(torch.int32), tokens.to(torch.int32), lp.float()


# --- what a pass cannot do without -----------------------------------------

def _seen(c):
    """Cached positions that some token of each sequence sees, and the pairs of
    a token and a position that it sees."""
    T, w = c["tokens"], c["window"]
    some = pairs = 0
    for n in (max(T, x) for x in _lengths(c["S"], c["max_len"], c["ragged"])):
        some += min(n, c["sink"] + w + T - 1) if w else n
        pairs += sum(min(n - t, c["sink"] + w) if w else n - t for t in range(T))
    return some, pairs


def work(case):
    c = case
    if c["kind"] == "verify":
        rows = c["S"] * (c["T"] + 1 + (c["T"] if c["draft"] else 0))
        return dict(bytes=rows * c["V"] * SIZE[c["dtype"]] + c["S"] * (c["T"] + 1) * 16, flops=4 * rows * c["V"])
    D, hkv = c["D"], c["hkv"]
    if c["kind"] == "read":
        R = c["S"] * c["n"]
        return dict(bytes=R * (hkv * (2 * D + 8 + 2 * D * SIZE[c["out"]]) + 8), flops=2 * R * hkv * D)
    if c["kind"] == "store":
        R = c["R"] - (c["R"] // c["skip"] if c["skip"] else 0)
        append = 8 * c["hq"] * D + hkv * (8 * D + 2 * D + 8) + 4 * c["rot"] + 12
        back = hkv * (2 * D + 8 + 2 * D * SIZE[c["out"]])
        return dict(bytes=R * (append + back), flops=8 * R * (c["hq"] + 2 * hkv) * D)
    some, pairs = _seen(c)
    position = hkv * 2 * (D * SIZE[c["dtype"]] + (4 if c["dtype"] == "i8" else 0))
    return dict(bytes=some * position + c["S"] * c["tokens"] * c["hq"] * (8 * D + 4),
                flops=4 * pairs * c["hq"] * D)


# --- the definition in 64 bits ---------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["kind"]](s["case"], s)


def _exact_codes(x):
    """What a head x [.., D] in 64 bits is held as: whole multiples of a step,
    the float32 next to a 127th of the largest magnitude."""
    top = torch.maximum(x.amax(-1, keepdim=True), -x.amin(-1, keepdim=True)).to(torch.float32).to(torch.float64)
    step = (top / 127).to(torch.float32).to(torch.float64)
    step = step * (top >= LEAST)
    return (x / step.clamp(min=1e-300)).round() * step


def _exact_store(c, s):
    R, half = c["R"], c["rot"] // 2
    there = [r for r, n in enumerate(s["slots"].tolist()) if n >= 0]
    rows = torch.tensor(there, device=DEV)

    def head(x, weight):
        x = x[rows].to(torch.float64)
        if weight is not None:
            x = x * (x.square().sum(-1) / c["D"] + EPS).rsqrt()[..., None] * weight.to(torch.float64)
        if half:
            at = s["positions"][rows].long()
            turn = torch.complex(s["rope"][0][at].double(), s["rope"][1][at].double())[:, None, :]
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
            x = torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)
        return x

    wq, wk, _ = s["norm"] if c["norm"] else (None, None, None)
    q = torch.zeros((R, c["hq"], c["D"]), dtype=torch.float64, device=DEV)
    k, v = (torch.zeros((R, c["hkv"], c["D"]), dtype=torch.float64, device=DEV) for _ in range(2))
    q[rows] = head(s["q"], wq)
    k[rows] = _exact_codes(head(s["k"], wk))
    v[rows] = _exact_codes(s["v"][rows].to(torch.float64))
    return q, k, v


def _exact_read(c, s):
    table, page, out = s["table"].tolist(), c["page"], []
    where = torch.tensor([[table[b][i // page], i % page] for b in range(c["S"]) for i in range(c["n"])], device=DEV)
    for x, scale in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])):
        out.append(torch.mul(x[where[:, 0], where[:, 1]].to(torch.float64),
                             scale[where[:, 0], :, where[:, 1]].to(torch.float64)[..., None]))
    return out


def _exact_attention(c, s):
    page, G, T = c["page"], c["hq"] // c["hkv"], c["tokens"]
    table, lens = s["table"].tolist(), s["lengths"].tolist()
    if sum(lens) * c["hkv"] * c["D"] > 1 << 34:
        return None

    def wide(x, scale, pages, n):
        y = x[pages].flatten(0, 1)[:n].to(torch.float64)
        return y if scale is None else y * scale[pages].transpose(1, 2).flatten(0, 1)[:n, :, None].to(torch.float64)

    outs, lses = [], []
    for b in range(c["S"]):
        n = lens[b * T + T - 1]
        pages = torch.tensor(table[b][:-(-n // page)], device=DEV)
        k, v = wide(s["k_cache"], s["k_scale"], pages, n), wide(s["v_cache"], s["v_scale"], pages, n)
        for t in range(T):
            r = b * T + t
            m = lens[r]
            first = max(0, m - c["window"]) if c["window"] else 0
            see = torch.tensor(list(range(min(c["sink"], first))) + list(range(first, m)), device=DEV)
            qq = s["q"][r].to(torch.float64).view(c["hkv"], G, -1)
            x = torch.matmul(qq, k[see].permute(1, 2, 0).contiguous()) * c["D"] ** -0.5
            lses.append(torch.logsumexp(x, -1).flatten())
            outs.append(torch.matmul(torch.softmax(x, -1), v[see].transpose(0, 1).contiguous()).flatten(0, 1))
    return torch.stack(outs), torch.stack(lses)


def _exact_verify(c, s):
    T, V = c["T"], c["V"]
    accepted, tokens, lps = [], [], []
    for b in range(c["S"]):
        t = 1.0 if s["temperature"] is None else float(s["temperature"][b])
        u = s["uniforms"][b].tolist()
        drafts = s["drafted"][b].tolist()
        count = T if s["counts"] is None else int(s["counts"][b])

        def logs(x):
            x = x.to(torch.float64)
            if t == 0.0:
                y = torch.full_like(x, -math.inf)
                y[int(torch.nonzero(x == x.max())[0])] = 0.0
                return y
            return torch.log_softmax(x / t, -1)

        said, lp, left, n = [], [], None, 0
        while True:
            p = logs(s["target"][b, n])
            if n == count:
                left = p.exp()
                break
            if c["draft"]:
                q = logs(s["draft"][b, n])
            else:
                q = torch.full_like(p, -math.inf)
                q[drafts[n]] = 0.0
            if not u[n] * math.exp(float(q[drafts[n]])) < math.exp(float(p[drafts[n]])):
                left = torch.relu(p.exp() - q.exp())
                if float(left.sum()) == 0.0:
                    left = p.exp()
                break
            said.append(drafts[n])
            lp.append(float(p[drafts[n]]))
            n += 1
        cum = torch.cumsum(left, 0)
        new = min(int(torch.searchsorted(cum, cum[-1:] * u[T], right=True)), V - 1)
        accepted.append(n)
        tokens.append(said + [new] + [-1] * (T - n))
        lps.append(lp + [float(p[new])] + [0.0] * (T - n))
    return (torch.tensor(accepted, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32),
            torch.tensor(lps, dtype=torch.float64))
