"""Eviction over tables with missing pages: front pages given back, pages
missing among the first, the last and the middle positions, whole sequences
without one; every way the kernels take.  What attention sees afterwards is
what was kept."""
import numpy as np
import pytest
import torch

import cache_ref as ref
import evict_ref
import xtern
from test_gpu_cache import DTYPES, Pool, log, same_bits

pytestmark = pytest.mark.gpu


def case(dtype, H, D, page, lens, budget, sink, recent, holes, layout="page_head_slot", seed=0, scores=None,
         lengths=None):
    """holes: per sequence, the table entries that are no page."""
    rng = np.random.default_rng(seed)
    num = sum((n + page - 1) // page for n in lens) + 2
    pool = Pool(rng, num, page, H, D, dtype, layout, score=True)
    table = ref.tables(rng, lens, page, num)
    pool.fill(rng, table, lens)
    pool.score = torch.from_numpy(rng.choice([0.0, -0.0, 0.25, 0.5, 1.0, 3.0], pool.score.shape).astype(np.float32)
                                  * rng.integers(1, 40, pool.score.shape).astype(np.float32))
    if scores:
        scores(pool.score)
    for b, entries in holes.items():
        for i, e in enumerate(entries):
            table[b, e] = (-1, num, -2 ** 31, 2 ** 31 - 1)[i % 4]
    lengths = np.asarray(lens if lengths is None else lengths, np.int32)
    cache, dtable = pool.upload(), torch.from_numpy(table).cuda()
    new, kept = xtern.kv_evict(cache, dtable, torch.from_numpy(lengths).cuda(), budget, sink=sink, recent=recent)
    torch.cuda.synchronize()
    want = evict_ref.evict(pool.k, pool.v, pool.score, table, page, lengths, budget, sink, recent)
    assert new.tolist() == want[0].tolist()
    assert np.array_equal(kept.cpu().numpy(), want[1])
    assert same_bits(pool.dscore, want[4])
    assert same_bits(cache.k, want[2]) and same_bits(cache.v, want[3])
    return pool, cache, table, dtable, new, kept


def test_front_given_back():
    """A sliding window cut down: attention over the result is attention over
    the kept positions."""
    for dtype in DTYPES:
        pool, cache, table, dtable, new, kept = case(dtype, 2, 64, 16, [64], 20, 0, 4, {0: [0, 1]})
        assert new.tolist() == [52]
        q = torch.randn((1, 2, 64), generator=torch.Generator().manual_seed(1))
        out = xtern.paged_attention(cache, dtable, new, q.cuda())
        for h in range(2):
            at = [(int(table[0, p // 16]), p % 16) for p in kept[0, h].tolist()]
            k, v = (torch.stack([x[pg, sl, h] for pg, sl in at]).double() for x in (pool.k, pool.v))
            s = q[0, h].double() @ k.t() / 8
            tol = 2 * (72 * ref.EPS * (q[0, h].double().abs() @ k.abs().t()).max() / 8 + 80 * ref.EPS)
            p = torch.softmax(s, 0)
            ref.close(out[0, h], p @ v, tol * (p @ v.abs()), f"{dtype} head {h}")


def test_page_missing_among_the_recent():
    for dtype in DTYPES:
        case(dtype, 3, 64, 16, [50], 30, 0, 18, {0: [2]})


SHAPES = [(64, "page_head_slot"), (100, "odd"), (37, "joint"), (3, "page_slot_head"), (256, "head_first")]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D,layout", SHAPES)
def test_layouts(dtype, D, layout):
    log(f"evict holes {dtype} {D} {layout}")
    case(dtype, 3, D, 16, [100, 133, 50, 90, 200, 70, 48], 50, 4, 8,
         {0: [0], 1: [1, 3, 7], 3: [5], 4: list(range(0, 10)), 5: list(range(0, 5)), 6: [0, 1, 2]}, layout=layout)


@pytest.mark.parametrize("page", [1, 3, 16, 100])
@pytest.mark.parametrize("rule", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (20, 10, 10), (20, 20, 0), (20, 0, 20), (20, 0, 0),
                                  (63, 3, 7), (200, 0, 0), (199, 4, 5), (299, 4, 5)], ids=str)
def test_rules(page, rule):
    """Pages lost anywhere, at every budget: more, as many and fewer positions
    left than it takes."""
    log(f"evict holes page {page} {rule}")
    n = [300, 64, 301, 299, 21]
    rng = np.random.default_rng(page)
    holes = {b: sorted(rng.choice((x + page - 1) // page, (x + page - 1) // page // 3, replace=False).tolist())
             for b, x in enumerate(n)}
    holes[0] = list(range(0, 100 // page))                    # 200 left (of pages that divide 100)
    holes[3] = list(range(200 // page, (299 + page - 1) // page))  # and nothing behind 200
    case(torch.bfloat16, 2, 32, page, n, *rule, holes, seed=page)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_long(dtype):
    """Keys in registers and through the workspace, tables of more entries
    than a workgroup has threads."""
    for n, page, budget, lost in ((5000, 1, 700, range(100, 2300)), (20011, 32, 3000, range(0, 40)),
                                  (20011, 32, 3000, range(3, 500, 7)), (17000, 16, 900, range(0, 1000)),
                                  (16384 + 64, 16, 16383, [5]), (14000, 5000, 800, [0]), (40000, 20000, 900, [1])):
        log(f"evict holes {dtype} {n} {page} {budget}")
        case(dtype, 8, 4 if dtype == torch.float32 else 8, page, [n, 40], budget, min(4, budget), 33, {0: lost, 1: [0]})


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D,layout", [(64, "page_head_slot"), (100, "odd"), (37, "joint"), (256, "head_first")])
def test_many_rows_of_few_heads(dtype, D, layout):
    """Moved through the workspace: holes before, between and behind."""
    log(f"evict holes {dtype} {D} {layout}")
    case(dtype, 1, D, 16, [6000, 4900, 4300], 4400, 7, 100, {0: list(range(50)), 1: [3, 4, 200, 305], 2: [0]},
         layout=layout)
    case(dtype, 2, D, 1, [5900], 4096 + 3, 3, 0, {0: list(range(1000, 5900, 5))})


def test_scores():
    """Equal scores, NaN, infinities, negative ones around the holes; lengths
    that the table does not hold."""
    def scores(s):
        s[::2, 0] = 0.0
        s[1::3, 1, 2] = float("nan")
        s[::5, 1, 3] = float("inf")
        s[::4, 1, 4] = -float("inf")
        s[::4, 1, 5] = -2.5
        s[3] = float("nan")

    for budget, sink, recent in ((40, 0, 0), (40, 4, 20), (90, 40, 0), (110, 0, 0), (1, 0, 0)):
        case(torch.float16, 2, 64, 16, [150, 128, 111, 100, 100], budget, sink, recent, {0: [2], 1: [0], 2: [6]},
             scores=scores, lengths=[150, 128, 111, 2 ** 31 - 1, -3])


def test_captured():
    """Captured on a stream without a workspace, replayed on restored caches."""
    rng = np.random.default_rng(4)
    P = 60
    cache = xtern.KvCache.new(P, 16, 2, 64, score=True)
    for x in (cache.k, cache.v, cache.score):
        x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape))))
    first = [x.clone() for x in (cache.k, cache.v, cache.score)]
    table = torch.from_numpy(rng.permutation(P)[:50].reshape(2, 25).astype(np.int32)).cuda()
    table[0, :7] = -1
    table[1, 11] = P
    lengths = torch.tensor([390, 400], dtype=torch.int32, device="cuda")

    def reset():
        for x, y in zip((cache.k, cache.v, cache.score), first):
            x.copy_(y)

    def call():
        return xtern.kv_evict(cache, table, lengths, 100, sink=4, recent=20)

    want = [x.clone() for x in (*call(), cache.k, cache.v, cache.score)]
    assert want[0].tolist() == [7 * 16 + 100, 100]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = call()
        for _ in range(4):
            reset()
            g.replay()
            st.synchronize()
            assert all(torch.equal(a, b) for a, b in zip((*out, cache.k, cache.v, cache.score), want))
