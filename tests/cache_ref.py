"""Plain 64-bit forms of the paged-cache operators and of the token
probabilities, on the host, with the error bounds that 32-bit kernels keep
(EPS is half a step of float32)."""
import numpy as np
import torch

EPS = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F64 = torch.float64


def pool(rng, num_pages, page, H, D, dtype, layout, score):
    """k, v (views [P, page, H, D] on the host) of a layout, every element NaN,
    and a score pool.  Returns (k, v, score, memory tensors to move)."""
    nan = float("nan")
    if layout == "page_head_slot":
        mem = [torch.full((num_pages, H, page, D), nan, dtype=dtype) for _ in range(2)]
        view = [lambda m: m.transpose(1, 2)] * 2
    elif layout == "page_slot_head":
        mem = [torch.full((num_pages, page, H, D), nan, dtype=dtype) for _ in range(2)]
        view = [lambda m: m] * 2
    elif layout == "joint":  # k and v of a page side by side
        mem = [torch.full((num_pages, 2, page, H, D), nan, dtype=dtype)]
        view = [lambda m: m[:, 0], lambda m: m[:, 1]]
    elif layout == "head_first":  # one slab per head, pages inside
        mem = [torch.full((H, num_pages, page, D), nan, dtype=dtype) for _ in range(2)]
        view = [lambda m: m.permute(1, 2, 0, 3)] * 2
    else:  # "odd": rows of D + 1 elements that start one element in
        mem = [torch.full((num_pages, page, H, D + 1), nan, dtype=dtype) for _ in range(2)]
        view = [lambda m: m[..., 1:]] * 2
    if len(mem) == 1:
        mem = [mem[0], mem[0]]
    sc = torch.from_numpy(rng.random((num_pages, H, page)).astype(np.float32)) if score else None
    return mem, view, sc


LAYOUTS = ["page_head_slot", "page_slot_head", "joint", "head_first", "odd"]


def tables(rng, lens, page, num_pages, spare=1):
    """A page table of random distinct pages, -1 behind each sequence's."""
    per = [(n + page - 1) // page for n in lens]
    t = np.full((len(lens), max(per + [1]) + spare), -1, np.int32)
    ids = iter(rng.permutation(num_pages))
    for i, k in enumerate(per):
        for j in range(k):
            t[i, j] = next(ids)
    return t


def positions(table_row, n, page, num_pages):
    """[(position, page, slot)] of a sequence's first n positions that exist."""
    n = max(0, min(int(n), len(table_row) * page))
    return [(p, int(table_row[p // page]), p % page) for p in range(n)
            if 0 <= table_row[p // page] < num_pages]


def attention(k, v, table, page, q, lengths, seq, scale, score=None):
    """(out, lse, new score, bounds of the three) of paged_attention; k, v
    [P, page, H, D] on the host, q [R, hq, D]."""
    R, hq, D = q.shape
    P, H = k.shape[0], k.shape[2]
    G = hq // H
    out, lse = torch.zeros((R, hq, D), dtype=F64), torch.full((R, hq), -np.inf, dtype=F64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    new = score.to(F64).clone() if score is not None else None
    stol = torch.zeros_like(new) if score is not None else None
    for r in range(R):
        b = r if seq is None else int(seq[r])
        if not 0 <= b < len(table):
            continue
        at = positions(table[b], lengths[r], page, P)
        if not at:
            continue
        pg = torch.tensor([x[1] for x in at])
        sl = torch.tensor([x[2] for x in at])
        n = len(at)
        for h in range(H):
            kk, vv = k[pg, sl, h].to(F64), v[pg, sl, h].to(F64)
            qq = q[r, h * G:(h + 1) * G].to(F64)
            s = scale * qq @ kk.t()
            if bool((s == -np.inf).all(1).any()):
                raise ValueError("not a case of this reference")
            p = torch.softmax(s, -1)
            out[r, h * G:(h + 1) * G] = p @ vv
            lse[r, h * G:(h + 1) * G] = torch.logsumexp(s, -1)
            # s_j: a sum of D rounded products and the scaling; exp's argument
            # is rounded, at most the row's spread in size; the sums over n
            # positions in any order; exp, the division and the rounding
            ds = ((D + 8) * EPS * abs(scale) * (qq.abs() @ kk.abs().t()).amax(-1)
                  + 4 * EPS * s.abs().amax(-1))
            rel = 2 * ds + (2 * n + 32) * EPS
            tol[r, h * G:(h + 1) * G] = rel[:, None] * (p @ vv.abs())
            ltol[r, h * G:(h + 1) * G] = ds + (n + 32) * EPS + 4 * EPS * lse[r, h * G:(h + 1) * G].abs()
            if new is not None:
                new.index_put_((pg, torch.tensor(h), sl), p.sum(0), accumulate=True)
                stol.index_put_((pg, torch.tensor(h), sl), (rel[:, None] * p).sum(0) + (G + 2) * EPS * p.sum(0),
                                accumulate=True)
    if new is not None:
        stol += 2 * EPS * new.abs()
    return out, lse, new, tol, ltol, stol


def evict(k, v, score, table, page, lengths, budget, sink, recent):
    """kv_evict in place on host tensors; returns (new lengths, kept)."""
    P, H = k.shape[0], k.shape[2]
    S = len(table)
    new = np.zeros(S, np.int32)
    kept = np.full((S, H, budget), -1, np.int32)
    for b in range(S):
        n = max(0, min(int(lengths[b]), table.shape[1] * page))
        new[b] = min(n, budget)
        if n <= budget:
            kept[b, :, :n] = np.arange(n)
            continue
        where = [(int(table[b][p // page]), p % page) for p in range(n)]
        for h in range(H):
            def rank(p):
                pg, sl = where[p]
                if not 0 <= pg < P:
                    return (2, 0.0, p)
                x = float(score[pg, h, sl])
                return (1, 0.0, p) if x != x else (0, -x, p)
            mid = sorted(range(sink, n - recent), key=rank)[:budget - sink - recent]
            stay = sorted(list(range(sink)) + mid + list(range(n - recent, n)))
            kept[b, h] = stay
            for j, p in enumerate(stay):  # ascending: a target never is a later source
                (pf, sf), (pt, st) = where[p], where[j]
                if p != j and 0 <= pf < P and 0 <= pt < P:
                    k[pt, st, h] = k[pf, sf, h]
                    v[pt, st, h] = v[pf, sf, h]
                    score[pt, h, st] = score[pf, h, sf]
    return new, kept


def logprobs(x, tokens, top):
    """(lp, entropy, ids, top lp, bounds of lp, entropy and top lp) of rows
    with neither NaN nor +inf."""
    x = x.to(F64)
    M, V = x.shape
    m = x.amax(-1, keepdim=True)
    none = (m == -np.inf)
    d = torch.where(x == -np.inf, torch.zeros((), dtype=F64), x - torch.where(none, 0.0, m))
    e = torch.where(x == -np.inf, torch.zeros((), dtype=F64), d.exp())
    first = (x == m).to(torch.int8).argmax(-1, keepdim=True)
    e1 = e.scatter(1, first, 0.0)  # without one maximum
    z = e1.sum(-1, keepdim=True)
    ln = torch.log1p(z)
    lp_all = torch.where(none, x, x - m - ln)
    xz = -(e1 * d).sum(-1, keepdim=True)
    H = (ln + xz / (1 + z))[:, 0]
    # each e is off by its rounded argument and exp itself, the sums by their
    # order (at most V / 64 terms one after the other, and a tree)
    rel = (V / 64 + 64) * EPS * z + 4 * EPS * xz
    # Below 2^-126 a float32 exp may give 0: each term e and d e (|d| < 128
    # where e is above the least subnormal, 2^-149) is then off by less than
    # 2^-126 and 2^-119, V of them by V 2^-119.  (64 bits hold entropies of
    # 1e-60, 32 bits none below 1e-45.)
    rel = rel + V * 2.0 ** -119
    lptol = rel / (1 + z) + 4 * EPS * ln
    htol = (rel / (1 + z) * (1 + xz / (1 + z)) + (V / 64 + 64) * EPS * xz / (1 + z)
            + 4 * EPS * (e1 * d * d).sum(-1, keepdim=True) / (1 + z))[:, 0] + 8 * EPS * H
    tol_of = lambda v: lptol + 4 * EPS * torch.where(torch.isfinite(v), v.abs(), torch.zeros((), dtype=F64))  # noqa: E731
    lp = ltol = None
    if tokens is not None:
        t = tokens.long()
        lp = lp_all.gather(1, t.clamp(0, V - 1))
        lp = torch.where(t < 0, 0.0, torch.where(t >= V, float("nan"), lp))
        ltol = tol_of(lp)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    tlp = lp_all.gather(1, order)
    return lp, torch.where(none[:, 0], 0.0, H), order, tlp, ltol, htol, tol_of(tlp)


def close(got, want, tol, what):
    """Every element within its bound; infinities and NaN in the same places."""
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, what
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    ok = same | ((got - want).abs() <= tol)
    if not bool(ok.all()):
        worst = torch.where(ok, 0.0, (got - want).abs() / tol.clamp(min=1e-300))
        i = int(worst.argmax())
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.numel()} out of bounds; element {i}: "
                             f"{got.flatten()[i].item()!r} want {want.flatten()[i].item()!r} "
                             f"bound {tol.flatten()[i].item():.3g}")
