"""Draws whose border lies on a sum of probabilities: equal logits and shares
of a few bits, where every order of additions meets it."""
import numpy as np
import pytest
import torch

import xtern
from test_gpu_cache import log

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")
INF = float("inf")


def draw(rows, values, V, shares):
    """One token of each sequence b from logits of V tokens, values[b] at the ids
    rows[b] and -inf elsewhere."""
    S = len(rows)
    x = torch.full((S, 1, V), -INF, dtype=torch.float32, device="cuda")
    for b, (ids, v) in enumerate(zip(rows, values)):
        x[b, 0, torch.tensor(ids, device="cuda")] = torch.as_tensor(v, dtype=torch.float32).cuda()
    got = xtern.verify_drafts(x, torch.zeros((S, 0), **I32), torch.tensor(shares, dtype=torch.float32, device="cuda")[:, None])
    torch.cuda.synchronize()
    return got[1][:, 0].cpu().numpy(), got[2][:, 0].cpu().numpy()


TIED = [  # (vocabulary, ids): a half of them, in other orders of addition, is a little more or less than a half
    (131072, [512 * i for i in (15, 25, 40, 48, 71, 123, 127, 137, 168, 185, 190, 204)]),
    (131072, [512 * i for i in (4, 32, 56, 67, 82, 157, 174, 193, 204, 213, 222, 255)]),
    (262144, [512 * i + 7 for i in (3, 110, 234, 250, 266, 320, 367, 392, 437, 465, 472, 503)]),
    (524288, [512 * i + 511 for i in (39, 54, 85, 145, 419, 437, 613, 649, 737, 756, 829, 983)]),
    (358400, [512 * i for i in (48, 52, 95, 104, 115, 155, 163, 432, 557, 579, 586, 628)]),
]


@pytest.mark.parametrize("i", range(len(TIED)))
def test_no_masked_token(i):
    V, ids = TIED[i]
    log(f"tie {V}")
    token, lp = draw([ids], [1.0], V, [0.5])
    assert token[0] in ids and np.isfinite(lp[0])


@pytest.mark.parametrize("V,S", [(131072, 800), (358400, 300)])
def test_no_masked_token_among_many(V, S):
    """Tokens of two sizes, each as often in the first half of the mass as in the
    second, and half of it asked for."""
    log(f"ties {V}")
    rng = np.random.default_rng(V)
    rows, values = [], []
    for _ in range(S):
        n = int(rng.integers(2, 10))
        ids = np.sort(rng.choice(V // 512, 2 * n, replace=False)) * 512 + rng.integers(0, 512, 2 * n)
        v = rng.choice([0.0, float(rng.uniform(-3, -0.1))], n)
        rows.append(ids.tolist())
        values.append(np.concatenate([v, rng.permutation(v)]))
    token, lp = draw(rows, values, V, [0.5] * S)
    for b in range(S):
        assert token[b] in rows[b] and np.isfinite(lp[b]), (b, token[b], rows[b])


def test_equal_logits_exactly():
    """n equally likely tokens: the one behind the share's whole part of n, also
    where the share falls on the end of one."""
    rng = np.random.default_rng(1)
    V, S = 3001, 3000
    n = rng.integers(1, 40, S)
    share = rng.integers(0, 16, S) / 16
    x = np.full((S, 1, V), -np.inf, np.float32)
    want = np.zeros(S, np.int64)
    for b in range(S):
        ids = np.sort(rng.choice(V, n[b], replace=False))
        x[b, 0, ids] = rng.choice([0.0, -7.25, 55.0])
        want[b] = ids[int(share[b] * 16) * int(n[b]) // 16]  # (as many tokens before it as the share covers whole)
    for temperature in (1.0, 0.3):
        got = xtern.verify_drafts(torch.from_numpy(x).cuda(), torch.zeros((S, 0), **I32),
                                  torch.from_numpy(share.astype(np.float32)[:, None]).cuda(), temperature=temperature)
        wrong = np.nonzero(got[1][:, 0].cpu().numpy() != want)[0]
        assert not len(wrong), (len(wrong), [(int(n[b]), share[b]) for b in wrong[:5]])


@pytest.mark.parametrize("certain", [True, False], ids=["certain", "draft"])
def test_equal_logits_of_target_and_draft(certain):
    """n tokens of the target, m of them (and others) the draft model's, a draft
    among both: accepted while u / m < 1 / n, the borders included; after it, what
    is left of the target in whole parts."""
    rng = np.random.default_rng(2)
    V, S = 500, 3000
    x, y = (np.full((S, k, V), -np.inf, np.float32) for k in (2, 1))
    drafted, u = np.zeros((S, 1), np.int32), np.zeros((S, 2), np.float32)
    want = np.full((S, 2), -1, np.int64)
    for b in range(S):
        n, m = (int(i) for i in rng.integers(1, 25, 2))
        p = np.sort(rng.choice(V, n, replace=False))
        q = np.sort(np.concatenate([p[:1 + n // 2], np.setdiff1d(rng.choice(V, m, replace=False), p)]))
        after = np.sort(rng.choice(V, n, replace=False))
        x[b, 0, p], x[b, 1, after], y[b, 0, q] = 1.5, -3.0, 0.25
        m = 1 if certain else len(q)
        drafted[b] = d = int(rng.choice(p[:1 + n // 2]))
        eighths = int(rng.integers(0, 8))
        k = (m * 16) // n
        u[b] = (k if 0 < k < 16 and rng.random() < 0.7 else rng.integers(0, 16)) / 16, eighths / 8
        if int(u[b, 0] * 16) * n < 16 * m:
            want[b] = d, after[eighths * n // 8]
            continue
        # max(1 / n - q, 0) in units of 1 / (n m)
        left = np.zeros(V, np.int64)
        left[p] = m
        if certain:
            left[d] = 0
        else:
            left[q] = np.maximum(left[q] - n, 0)
        if not left.sum():
            left[p] = m
        cum = np.cumsum(left)
        want[b, 0] = np.nonzero(8 * cum > eighths * cum[-1])[0][0]
    got = xtern.verify_drafts(*(torch.from_numpy(a).cuda() for a in (x, drafted, u)),
                              draft=None if certain else torch.from_numpy(y).cuda())
    wrong = np.nonzero((got[1].cpu().numpy() != want).any(1))[0]
    assert not len(wrong), (len(wrong), wrong[:5], got[1][wrong[:5]].tolist(), want[wrong[:5]].tolist())
