"""The plain form of the eviction against hand-worked tables with missing
pages: what an attention sees afterwards is what was kept."""
import numpy as np
import pytest
import torch

import cache_ref as ref
import evict_ref


def pool(P, page, H=2, seed=0):
    r = np.random.default_rng(seed)
    k, v = (torch.from_numpy(r.standard_normal((P, page, H, 4))) for _ in range(2))
    return k, v, torch.from_numpy(r.random((P, H, page)).astype(np.float32))


def seen(x, row, n, page, h):
    return [x[pg, sl, h] for _, pg, sl in ref.positions(row, n, page, x.shape[0])]


@pytest.mark.parametrize("row,page,n,budget,sink,recent,new", [
    ([-1, -1, 2, 3], 16, 64, 20, 0, 4, 52),      # the front given back
    ([0, 1, -1, 2], 16, 50, 30, 0, 18, 30),      # a page missing among the recent ones
    ([0, -1, 2, 7], 16, 64, 20, 4, 4, 36),       # a page past the pool
    ([-1, 1], 16, 20, 10, 2, 2, 20),             # fewer left than the budget: all stay
    ([-1, -1], 16, 32, 10, 2, 2, 0),             # nothing left
    ([0, 1], 16, 32, 20, 4, 4, 20),              # no holes
    ([-1, -1], 16, 9, 10, 2, 2, 9)], ids=str)    # not cut
def test_what_attention_sees(row, page, n, budget, sink, recent, new):
    k, v, score = pool(4, page)
    table = np.array([row], np.int32)
    lens, kept, k1, v1, s1 = evict_ref.evict(k, v, score, table, page, [n], budget, sink, recent)
    assert lens[0] == new
    if n <= budget:
        assert torch.equal(k, k1) and kept[0, 0].tolist() == list(range(n)) + [-1] * (budget - n)
        return
    live = {p: (pg, sl) for p, pg, sl in ref.positions(row, n, page, 4)}
    for h in range(2):
        stay = [p for p in kept[0, h] if p >= 0]
        assert len(stay) == min(budget, len(live)) and stay == sorted(stay) and set(stay) <= set(live)
        for x, x1 in ((k, k1), (v, v1)):
            want = [x[live[p] + (h,)] for p in stay]
            got = seen(x1, row, lens[0], page, h)
            assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
        order = sorted(live)
        assert set(order[:sink]) <= set(stay) or len(live) <= budget
        assert len(live) <= budget or set(order[len(order) - recent:]) <= set(stay)
        # none of the rest has a higher score than one that was chosen
        rest = [float(score[live[p][0], h, live[p][1]]) for p in set(live) - set(stay)]
        chosen = [float(score[live[p][0], h, live[p][1]]) for p in stay if p in order[sink:len(order) - recent]]
        assert not rest or not chosen or max(rest) <= min(chosen)


def test_without_holes_as_the_other_form():
    k, v, score = pool(12, 8, seed=3)
    table = np.random.default_rng(1).permutation(12).reshape(2, 6).astype(np.int32)
    new, kept, k1, v1, s1 = evict_ref.evict(k, v, score, table, 8, [48, 30], 21, 3, 5)
    wnew, wkept = ref.evict(k, v, score, table, 8, [48, 30], 21, 3, 5)  # (in place)
    assert np.array_equal(new, wnew) and np.array_equal(kept, wkept)
    assert torch.equal(k, k1) and torch.equal(v, v1) and torch.equal(score, s1)
