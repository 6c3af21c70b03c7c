"""Device memory that the cache calls keep: bounded, whatever the table could
hold, with the results of the small table."""
import numpy as np
import pytest
import torch

import xtern
from test_gpu_cache import log

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")
WIDE = 1 << 16  # entries of a wide table, of 16 positions each
BOUND = 3 << 29  # 1.5 GiB: the workspaces' limit, counters and parts beside it


def used(call):
    """The call's results, on a stream of its own (and so with workspaces of
    its own), and the device memory that it took beside torch's."""
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        call(small=True)  # (code objects, small workspaces)
        st.synchronize()
        free = torch.cuda.mem_get_info()[0]
        held = torch.cuda.memory_reserved()
        out = call(small=False)
        st.synchronize()
        return out, free - torch.cuda.mem_get_info()[0] - (torch.cuda.memory_reserved() - held)


def cache_of(rng, pages, H, D, dtype):
    c = xtern.KvCache.new(pages, 16, H, D, dtype=dtype, score=True)
    for x in (c.k, c.v, c.score):
        x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32)))
    return c


def tables(rng, lens, seqs):
    """The same pages in a narrow table and in a wide one of `seqs` rows."""
    per = [(n + 15) // 16 for n in lens]
    ids = rng.permutation(sum(per)).astype(np.int32)
    narrow = np.full((len(lens), max(per)), -1, np.int32)
    at = 0
    for b, k in enumerate(per):
        narrow[b, :k] = ids[at:at + k]
        at += k
    wide = torch.full((seqs, WIDE), -1, **I32)
    wide[:len(lens), :max(per)] = torch.from_numpy(narrow).cuda()
    return sum(per), torch.from_numpy(narrow).cuda(), wide


@pytest.mark.parametrize("named", [False, True], ids=["rows", "seq"])
@pytest.mark.parametrize("dtype,R", [(torch.float32, 40), (torch.bfloat16, 40), (torch.float16, 1100)], ids=str)
def test_scores_of_a_wide_table(dtype, R, named):
    """40 (1100) rows of 64 query heads over a table for 2^20 positions: 10.7
    (295) GB of scores if all were held at once.  Same results as over the
    narrow table."""
    log(f"accumulate {dtype} {R} {named}")
    rng = np.random.default_rng(6)
    hq, H, D = 64, 2, 64
    lens = [int(x) for x in rng.integers(0, 128, R)]
    P, narrow, wide = tables(rng, lens, R)
    first = cache_of(rng, P, H, D, dtype)
    q = torch.from_numpy(rng.standard_normal((R, hq, D)).astype(np.float32)).cuda()
    order = rng.permutation(R) if named else np.arange(R)
    seq = torch.from_numpy(order.astype(np.int32)).cuda() if named else None
    lengths = torch.tensor([lens[b] for b in order], **I32)

    def call(small):
        c = xtern.KvCache(first.k, first.v, first.score.clone())
        out, lse = xtern.paged_attention(c, narrow if small else wide, lengths, q, seq=seq, lse=True, accumulate=True)
        return out, lse, c.score

    (out, lse, score), took = used(call)
    want = call(small=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(score, want[2])
    log(f"took {took / 2 ** 20:.0f} MiB")
    assert took < BOUND


def test_more_rows_than_sequences_are_none():
    """The C call's rows without a sequence, in a later part of the rows."""
    rng = np.random.default_rng(7)
    R, hq, H, D = 40, 64, 2, 64
    P, narrow, wide = tables(rng, [50], 1)
    c = cache_of(rng, P, H, D, torch.float16)
    first = c.score.clone()
    q = torch.from_numpy(rng.standard_normal((R, hq, D)).astype(np.float32)).cuda()
    lengths = torch.full((R,), 50, **I32)
    out = torch.full_like(q, 7.0)
    L = xtern.lib()
    from xtern.cache import _table
    t, _ = _table(wide, torch.cuda.current_device())
    assert L.xt_paged_attention(c._ref, t, None, lengths.data_ptr(), q.data_ptr(), hq * D, hq, 0.1, R, out.data_ptr(),
                                hq * D, None, 1, torch.cuda.current_stream().cuda_stream) == xtern.XT_OK
    torch.cuda.synchronize()
    assert bool(out[0].any()) and not bool(out[1:].any())
    assert float((c.score - first).sum()) == pytest.approx(hq, rel=1e-4)

def test_eviction_of_a_wide_table():
    """48 sequences of 16 heads over a table for 2^20 positions: 3.2 GB of keys
    if all were held at once."""
    rng = np.random.default_rng(8)
    S, H, D = 48, 16, 8
    lens = [20000, 300, 17000, 0] + [int(x) for x in rng.integers(0, 200, S - 5)] + [18011]
    P, narrow, wide = tables(rng, lens, S)
    first = cache_of(rng, P, H, D, torch.bfloat16)
    lengths = torch.tensor(lens, **I32)

    def call(small):
        c = xtern.KvCache(*(x.clone() for x in (first.k, first.v, first.score)))
        out = xtern.kv_evict(c, narrow if small else wide, lengths, 150, sink=4, recent=30)
        return (*out, c.k, c.v, c.score)

    out, took = used(call)
    assert all(torch.equal(a, b) for a, b in zip(out, call(small=True)))
    log(f"took {took / 2 ** 20:.0f} MiB")
    assert took < BOUND
