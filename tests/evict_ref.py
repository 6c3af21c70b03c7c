"""Eviction from its definition, on the host: of a sequence longer than the
budget, the positions that have a page, in order, are a list; the first `sink`,
the last `recent` and the highest scores between them (ties to the lowest, NaN
below every number) become its first entries, and the length ends behind them."""
import numpy as np

import cache_ref as ref


def evict(k, v, score, table, page, lengths, budget, sink, recent):
    """(new lengths, kept, k, v, score) of kv_evict; k, v [P, page, H, D] and
    score [P, H, page] are left as they are."""
    P, H = k.shape[0], k.shape[2]
    out = k.clone(), v.clone(), score.clone()
    new, kept = np.zeros(len(table), np.int32), np.full((len(table), H, budget), -1, np.int32)
    for b, row in enumerate(table):
        n = max(0, min(int(lengths[b]), len(row) * page))
        if n <= budget:
            new[b], kept[b, :, :n] = n, np.arange(n)
            continue
        live = ref.positions(row, n, page, P)
        last = min(len(live), budget)
        new[b] = live[last - 1][0] + 1 if last else 0
        for h in range(H):
            stay = live
            if len(live) > budget:
                def rank(x):
                    s = float(score[x[1], h, x[2]])
                    return (1, 0.0, x[0]) if s != s else (0, -s, x[0])
                end = len(live) - recent
                middle = sorted(live[sink:end], key=rank)[:budget - sink - recent]
                stay = live[:sink] + sorted(middle) + live[end:]
            for j, (p, pg, sl) in enumerate(stay):
                _, to, ts = live[j]
                kept[b, h, j] = p
                out[0][to, ts, h], out[1][to, ts, h] = k[pg, sl, h], v[pg, sl, h]
                out[2][to, h, ts] = score[pg, h, sl]
    return (new, kept) + out
