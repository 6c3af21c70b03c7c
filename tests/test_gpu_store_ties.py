"""Elements that lie in the middle between two codes: the even one is stored,
for every scale, as the quotient by the scale has it."""
import numpy as np
import pytest
import torch

import xtern
from test_gpu_cache import log

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


def heads(scales, D, seed):
    """(values [n, D], codes): 127 s, then (k + 1/2) s, all of them exact in
    float32 (s a whole number of 12 bits, or that times a power of two)."""
    rng = np.random.default_rng(seed)
    k = rng.integers(-127, 127, (len(scales), D))
    y = (k + 0.5) * np.asarray(scales)[:, None]
    y[:, 0] = 127.0 * np.asarray(scales)
    want = np.where(k % 2 == 0, k, k + 1)  # (the even one of k and k + 1)
    want[:, 0] = 127
    assert (y.astype(np.float32) == y).all()
    return torch.from_numpy(y.astype(np.float32)), torch.from_numpy(want.astype(np.int8))


def check(scales, D, rope, seed=0):
    H = 8
    scales = np.asarray(scales, np.float64)
    scales = scales[:len(scales) // H * H]
    R = len(scales) // H
    (k, kc), (v, vc) = (heads(s, D, seed + i) for i, s in enumerate((scales, scales[::-1])))
    shape = lambda x: x.view(R, H, D)  # noqa: E731
    cache = xtern.KvCache.new((R + 15) // 16, 16, H, D, dtype=torch.int8)
    table = torch.arange((R + 15) // 16, **I32)[None]
    slots, seq = torch.arange(R, **I32), torch.zeros(R, **I32)
    turn = None
    if rope:  # a quarter turn: element i becomes minus element i + h, and that element i
        h = D // 2
        turn = torch.zeros((R, h), device="cuda"), torch.ones((R, h), device="cuda")
        kc = torch.cat([-kc[:, h:2 * h], kc[:, :h], kc[:, 2 * h:]], 1)
    xtern.kv_append(cache, table, slots, shape(k).cuda(), shape(v).cuda(), seq=seq, rope=turn)
    torch.cuda.synchronize()
    at = slots.long() // 16, slots.long() % 16
    for held, got_s, codes, s in ((cache.k, cache.k_scale, kc, scales), (cache.v, cache.v_scale, vc, scales[::-1])):
        assert np.array_equal(got_s[at[0], :, at[1]].cpu().numpy().reshape(-1), s.astype(np.float32))
        got = held[at].cpu().view(-1, D)
        wrong = (got != codes).nonzero()
        assert not len(wrong), (len(wrong), [(float(s[i]), d, int(got[i, d]), int(codes[i, d])) for i, d in wrong[:5].tolist()])


@pytest.mark.parametrize("D", [256, 128, 100, 64, 37])
@pytest.mark.parametrize("rope", [False, True], ids=["plain", "turned"])
def test_codes_at_ties(D, rope):
    log(f"ties {D} {rope}")
    check([49, 98, 103, 3, 7, 127, 4095, 1], D, rope)
    check(np.arange(1, 4096, 2), D, rope)
    check(np.arange(1, 4096, 2) * 2.0 ** -30, D, rope, seed=5)
