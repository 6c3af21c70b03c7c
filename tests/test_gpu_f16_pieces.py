"""f16 caches: what counts in a row may be far below the row's largest weight
or largest query element, and still has the precision of 32 bits."""
import numpy as np
import pytest
import torch

import cache_ref as ref
import xtern

pytestmark = pytest.mark.gpu

PAGE = 16


def attend(k, v, q, scale, dtype):
    """k, v [n, H, D], q [hq, D]: over pages in order, and the plain form."""
    n, H, D = k.shape
    P = (n + PAGE - 1) // PAGE
    mem = [torch.zeros((P * PAGE, H, D), dtype=dtype) for _ in range(2)]
    mem[0][:n], mem[1][:n] = k.to(dtype), v.to(dtype)
    mem = [m.reshape(P, PAGE, H, D) for m in mem]
    table = np.arange(P, dtype=np.int32).reshape(1, P)
    want = ref.attention(mem[0], mem[1], table, PAGE, q[None], [n], None, scale)
    cache = xtern.KvCache(mem[0].cuda(), mem[1].cuda())
    out, lse = xtern.paged_attention(cache, torch.from_numpy(table).cuda(), torch.tensor([n], dtype=torch.int32).cuda(),
                                     q[None].cuda(), scale=scale, lse=True)
    ref.close(out, want[0], want[3], "out")
    ref.close(lse, want[1], want[4], "lse")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("D", [8, 64, 128, 256])
@pytest.mark.parametrize("bits", [10, 20, 26, 30, 34])
def test_weights_far_below_the_largest(dtype, D, bits):
    """One position takes all the weight and holds zeros; the others, 2^-bits
    of it each, are all that is read.  (The score is one product, so the
    bounds of the scores are a few steps.)"""
    rng = np.random.default_rng(bits)
    for n, top in ((5, 0), (40, 17), (700, 650)):
        k = torch.zeros((n, 1, D))
        k[:, 0, 1] = torch.from_numpy(rng.uniform(0, 1, n).astype(np.float32))
        k[top, 0, 1] = bits
        v = torch.from_numpy(rng.uniform(0.5, 1, (n, 1, D)).astype(np.float32)) * 1000
        v[top] = 0.0
        q = torch.zeros((2, D))
        q[:, 1] = 1.0
        attend(k, v, q, float(np.log(2.0)), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bits", [10, 20, 26, 30])
def test_query_elements_far_below_the_largest(dtype, bits):
    """The largest query element meets zeros; the scores come from one that is
    2^-bits of it, times large keys."""
    rng = np.random.default_rng(bits + 100)
    for D in (8, 64, 128, 256):
        n = 60
        k = torch.zeros((n, 1, D))
        k[:, 0, 3] = torch.from_numpy(rng.uniform(-60000, 60000, n).astype(np.float32))
        v = torch.from_numpy(rng.standard_normal((n, 1, D)).astype(np.float32))
        q = torch.zeros((3, D))
        q[:, 0] = 1.0
        q[:, 3] = torch.from_numpy(rng.uniform(1, 2, 3).astype(np.float32)) * 2.0 ** -bits
        attend(k, v, q, 8.0 / (60000 * 2.0 ** -bits), dtype)
