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
