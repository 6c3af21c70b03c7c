"""Plain 64-bit forms of the store (norms, rotation, 8-bit codes), of windowed
attention of several tokens, and of the verification of drafts, on the host,
with the error bounds that the kernels keep (EPS is half a step of float32)."""
import numpy as np
import torch

EPS = 2.0 ** -24
F64 = torch.float64
LEAST = 2.0 ** -119


def heads(x, weight, eps, cos=None, sin=None):
    """x [.., D] in 64 bits: normed (weight not None), then its first 2 *
    len(cos) elements rotated."""
    x = x.to(F64)
    if weight is not None:
        x = weight.to(F64) * x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if cos is not None:
        h = cos.shape[-1]
        a, b, c, s = x[..., :h], x[..., h:2 * h], cos.to(F64), sin.to(F64)
        x = torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)
    return x


def codes(y):
    """(int8 codes, float32 scale) of heads y [.., D] in 64 bits."""
    f = y.to(torch.float32)
    top = f.abs().amax(-1)
    whole = torch.isfinite(f).all(-1)
    zero = whole & (top < LEAST)
    scale = (top.to(F64) / 127).to(torch.float32)
    scale = torch.where(whole, torch.where(zero, 0.0, scale), float("nan"))
    c = torch.where((whole & ~zero)[..., None], (y / scale.to(F64)[..., None]).round(), 0.0)
    return c.to(torch.int8), scale


def visible(table_row, n, page, num_pages, window, sink):
    """[(position, page, slot)] that a row of length n sees."""
    n = max(0, min(int(n), len(table_row) * page))
    return [(p, int(table_row[p // page]), p % page) for p in range(n)
            if (not window or p < sink or p >= n - window) and 0 <= table_row[p // page] < num_pages]


def attention(k, v, table, page, q, lengths, seq, scale, ks=None, vs=None, window=0, sink=0, tokens=1, score=None):
    """(out, lse, new score, bounds of the three); k, v [P, page, H, D] on the
    host, ks, vs None or [P, H, page] (k, v are codes then), q [R, hq, D]."""
    R, hq, D = q.shape
    P, H = k.shape[0], k.shape[2]
    G = hq // H
    out, lse = torch.zeros((R, hq, D), dtype=F64), torch.full((R, hq), -np.inf, dtype=F64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    new = score.to(F64).clone() if score is not None else None
    stol = torch.zeros_like(new) if score is not None else None
    for r in range(R):
        b = r // tokens if seq is None else int(seq[r // tokens * tokens])
        if not 0 <= b < len(table):
            continue
        at = visible(table[b], lengths[r], page, P, window, sink)
        if not at:
            continue
        pg, sl = torch.tensor([x[1] for x in at]), torch.tensor([x[2] for x in at])
        n = len(at)
        for h in range(H):
            kk, vv = k[pg, sl, h].to(F64), v[pg, sl, h].to(F64)
            if ks is not None:
                kk, vv = kk * ks[pg, h, sl].to(F64)[:, None], vv * vs[pg, h, sl].to(F64)[:, None]
            qq = q[r, h * G:(h + 1) * G].to(F64)
            s = scale * qq @ kk.t()
            p = torch.softmax(s, -1)
            to = slice(h * G, (h + 1) * G)
            out[r, to], lse[r, to] = p @ vv, torch.logsumexp(s, -1)
            # s_j: a sum of D rounded products and the scaling, or whole numbers:
            # the query off by half of 2^-22 of its largest element, and the
            # roundings of the scaled sum; exp's argument is rounded, at most the
            # row's spread in size; the sums over n positions in any order
            ds = (D + 8) * EPS * abs(scale) * (qq.abs() @ kk.abs().t()).amax(-1) + 8 * EPS * s.abs().amax(-1)
            if ks is not None:
                ds = ds + 2 * EPS * abs(scale) * qq.abs().amax(-1) * kk.abs().sum(-1).max()
            rel = 2 * ds + (2 * n + 32) * EPS
            tol[r, to] = rel[:, None] * (p @ vv.abs())
            if ks is not None:
                # weights p vs off by half of 2^-22 of the largest of their tile,
                # 64 positions that are at most 63 apart
                w = p * vs[pg, h, sl].to(F64).abs()
                w = torch.nn.functional.max_pool1d(w[:, None], 127, 1, 63)[:, 0]
                tol[r, to] += 2 * EPS * (w @ v[pg, sl, h].to(F64).abs())
            ltol[r, to] = ds + (n + 32) * EPS + 4 * EPS * lse[r, to].abs()
            if new is not None:
                new.index_put_((pg, torch.tensor(h), sl), p.sum(0), accumulate=True)
                stol.index_put_((pg, torch.tensor(h), sl), (rel[:, None] * p).sum(0) + (G + 2) * EPS * p.sum(0),
                                accumulate=True)
    if new is not None:
        stol += 2 * EPS * new.abs()
    return out, lse, new, tol, ltol, stol


def chances(x, temperature):
    """softmax(x / temperature) in 64 bits, None for what is none."""
    x = x.to(F64).numpy()
    if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all():
        return None
    if temperature == 0:
        p = np.zeros_like(x)
        p[int(np.argmax(x))] = 1.0
        return p
    x = x / temperature
    e = np.exp(x - x.max())
    return e / e.sum()


def verify(target, drafted, uniforms, draft=None, counts=None, temperature=1.0):
    """(accepted, tokens, logprobs) of verify_drafts; logprobs in 64 bits."""
    S, T, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    accepted, tokens = np.zeros(S, np.int32), np.full((S, T + 1), -1, np.int32)
    lp = np.zeros((S, T + 1))
    for b in range(S):
        temp = float(np.float32(temperature if np.isscalar(temperature) else temperature[b]))  # (an f32 of the call)
        count = T if counts is None else min(T, int(counts[b]))
        if count < 0 or not 0 <= temp < np.inf:
            continue
        u = uniforms[b].to(F64).numpy()
        n = 0
        while True:
            p, x, q = chances(target[b, n], temp), -1, None
            if n < count and 0 <= int(drafted[b, n]) < V:
                x = int(drafted[b, n])
                q = np.zeros(V)
                q[x] = 1.0
                if draft is not None:
                    q = chances(draft[b, n], temp)
            if p is None or (x >= 0 and q is None):
                break
            if x >= 0 and u[n] * q[x] < p[x]:
                tokens[b, n], lp[b, n] = x, np.log(p[x])
                n += 1
                continue
            left = p if x < 0 else np.maximum(p - q, 0.0)
            if not left.sum() > 0:
                left = p
            cum = np.cumsum(left)
            new = int(np.searchsorted(cum, u[T] * cum[-1], side="right")) if u[T] == u[T] else V
            new = min(new, int(np.nonzero(left)[0][-1]))
            tokens[b, n], lp[b, n] = new, np.log(p[new])
            break
        accepted[b] = n
    return accepted, tokens, lp
