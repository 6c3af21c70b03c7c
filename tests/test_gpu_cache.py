"""The paged cache's append, attention and eviction against plain 64-bit
forms: every element type and memory layout, head counts and sizes, lengths
from none to several thousand, pages that end anywhere.  Memory that a call
must not look at holds NaN."""
import numpy as np
import pytest
import torch

import cache_ref as ref
import xtern

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def log(msg):
    print(f"[case] {msg}", flush=True)


def same_bits(a, b):
    a, b = a.cpu().contiguous(), b.cpu().contiguous()
    t = torch.int32 if a.element_size() == 4 else torch.int16
    return torch.equal(a.view(t), b.view(t))


class Pool:
    """A pool on the host and its copy on the device."""

    def __init__(self, rng, num_pages, page, H, D, dtype, layout="page_head_slot", score=False):
        self.mem, self.view, self.score = ref.pool(rng, num_pages, page, H, D, dtype, layout, score)
        self.page, self.P = page, num_pages

    @property
    def k(self):
        return self.view[0](self.mem[0])

    @property
    def v(self):
        return self.view[1](self.mem[1])

    def fill(self, rng, table, lens, std=1.0):
        """Random keys and values at the written positions."""
        for b, n in enumerate(lens):
            for _, pg, sl in ref.positions(table[b], n, self.page, self.P):
                for x in (self.k, self.v):
                    x[pg, sl] = torch.from_numpy(rng.standard_normal(tuple(x.shape[2:])) * std).to(x.dtype)

    def upload(self):
        one = self.mem[0] is self.mem[1]
        self.dev = [self.mem[0].cuda()]
        self.dev.append(self.dev[0] if one else self.mem[1].cuda())
        self.dscore = self.score.cuda() if self.score is not None else None
        return xtern.KvCache(self.view[0](self.dev[0]), self.view[1](self.dev[1]), self.dscore)


def attention_case(dtype, hq, H, D, page, lens, layout="page_head_slot", accumulate=False, scale=None, seed=0,
                   edit=None, seq=None, lengths=None, std=1.0):
    rng = np.random.default_rng(seed)
    num = sum((n + page - 1) // page for n in lens) + 2
    pool = Pool(rng, num, page, H, D, dtype, layout, accumulate)
    table = ref.tables(rng, lens, page, num)
    pool.fill(rng, table, lens, std)
    lengths = np.asarray(lens if lengths is None else lengths, np.int32)
    if edit:
        edit(table, lengths, pool)
    q = torch.from_numpy(rng.standard_normal((len(lengths), hq, D)).astype(np.float32))
    scale = D ** -0.5 if scale is None else scale
    want = ref.attention(pool.k, pool.v, table, page, q, lengths, seq, scale, pool.score)
    cache = pool.upload()
    out, lse = xtern.paged_attention(cache, torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda(),
                                     q.cuda(), seq=None if seq is None else torch.tensor(seq, dtype=torch.int32).cuda(),
                                     scale=scale, lse=True, accumulate=accumulate)
    torch.cuda.synchronize()
    ref.close(out, want[0], want[3], "out")
    ref.close(lse, want[1], want[4], "lse")
    if accumulate:
        ref.close(pool.dscore, want[2], want[5], "score")
    for a, b in zip(pool.dev, pool.mem):
        assert same_bits(a, b), "the cache changed"


HEADS = [(1, 1, 64), (4, 4, 100), (20, 5, 128), (16, 2, 80), (8, 1, 256), (24, 2, 96), (40, 2, 33), (3, 1, 1),
         (32, 1, 192), (12, 3, 7)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_attention_heads(dtype, heads):
    log(f"attention {dtype} {heads}")
    for acc in (False, True):
        attention_case(dtype, *heads, page=16, lens=[1, 37, 0, 130], accumulate=acc)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("page", [1, 2, 3, 7, 8, 24, 33, 64, 1000])
def test_attention_pages(dtype, page):
    log(f"attention {dtype} page {page}")
    attention_case(dtype, 4, 2, 64, page, lens=[1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 129], accumulate=page % 2 == 0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("layout", ref.LAYOUTS)
@pytest.mark.parametrize("D", [64, 100, 128, 37])
def test_attention_layouts(dtype, layout, D):
    log(f"attention {dtype} {layout} {D}")
    attention_case(dtype, 6, 3, D, 16, lens=[70, 5, 259], layout=layout, accumulate=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("lens", [[4097], [1, 5000], [3000] * 3, [511, 512, 513, 1023, 1024, 1025], [20000]], ids=str)
def test_attention_long(dtype, lens):
    log(f"attention {dtype} {lens}")
    attention_case(dtype, 8, 2, 128 if dtype != torch.float32 else 100, 32, lens=lens, accumulate=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_many_rows(dtype):
    log(f"attention {dtype} many rows")
    rng = np.random.default_rng(3)
    attention_case(dtype, 4, 2, 32, 8, lens=[int(x) for x in rng.integers(0, 90, 300)], accumulate=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads", [(1, 1, 64), (2, 1, 130), (4, 2, 255), (6, 2, 200), (17, 1, 64), (10, 5, 36)], ids=str)
def test_attention_long_heads(dtype, heads):
    """Rows in many segments for one, two and more query heads of a group."""
    log(f"attention {dtype} {heads} long")
    attention_case(dtype, *heads, page=16, lens=[9000, 140], accumulate=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_row_counts(dtype):
    """More rows than a wave has lanes, some of them split; more rows than are
    split at all, several to a sequence."""
    rng = np.random.default_rng(4)
    lens = [int(x) for x in rng.integers(0, 60, 150)]
    lens[3], lens[70], lens[149] = 3000, 1500, 2500
    log(f"attention {dtype} 150 rows")
    attention_case(dtype, 4, 2, 64, 16, lens=lens, accumulate=True)
    log(f"attention {dtype} 1100 rows")
    seq = [i % 5 for i in range(1100)]
    attention_case(dtype, 4, 2, 64, 16, lens=[300, 20, 1, 150, 64], seq=seq,
                   lengths=[(37 * i) % (l + 1) for i, l in enumerate([[300, 20, 1, 150, 64][b] for b in seq])],
                   accumulate=dtype == torch.float32)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_spread(dtype):
    """Scores hundreds apart, equal scores, a scale below zero."""
    for scale, std in ((2.0, 3.0), (0.0, 1.0), (-0.3, 1.0), (1e-3, 100.0 if dtype != torch.float16 else 50.0)):
        attention_case(dtype, 8, 2, 64, 16, lens=[200, 33], scale=scale, std=std, accumulate=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_holes(dtype):
    """Entries that are no page, lengths past the table and below zero, whole
    rows without a page."""
    def edit(table, lengths, pool):
        table[0, 1] = -1
        table[0, 3] = pool.P
        table[1, :] = -7
        table[2, 0] = 2 ** 31 - 1
        table[3, 4:] = -1
        lengths[4] = -5
        lengths[5] = 2 ** 31 - 1
        lengths[6] = 10 ** 6

    attention_case(dtype, 8, 2, 64, 16, lens=[100, 40, 300, 200, 33, 64, 50], edit=edit, accumulate=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_freed_front(dtype):
    """The front pages of long sequences given back (a sliding window): whole
    segments of the split hold nothing."""
    def edit(table, lengths, pool):
        table[0, :240] = -1
        table[1, 10:100] = -1

    attention_case(dtype, 8, 2, 64, 16, lens=[4000, 2000, 30], edit=edit, accumulate=True)


def test_attention_rows_of_one_sequence():
    """A prompt: each token attends up to itself; rows that name no sequence."""
    for dtype in DTYPES:
        attention_case(dtype, 8, 2, 64, 16, lens=[50, 70], seq=[0] * 20 + [1] * 10 + [2, -1, 2 ** 31 - 1],
                       lengths=list(range(1, 21)) + list(range(61, 71)) + [5, 5, 5], accumulate=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_infinities(dtype):
    """What a formula of infinities gives, and only where a row sees them."""
    page, H, D, n = 16, 2, 64, 40
    rng = np.random.default_rng(1)
    pool = Pool(rng, 8, page, H, D, dtype)
    table = np.repeat(ref.tables(rng, [n], page, 8, spare=0), 3, 0)  # (one sequence, three rows)
    pool.fill(rng, table[:1], [n])
    q = torch.from_numpy(np.abs(rng.standard_normal((3, 4, D))).astype(np.float32))
    pg, sl = int(table[0, 20 // page]), 20 % page
    pool.k[pg, sl, 0] = float("inf")      # head 0: +inf scores -> NaN
    pool.k[pg, sl, 1] = -float("inf")     # head 1: weight 0
    lengths = np.array([20, 21, 40], np.int32)
    cache = pool.upload()
    out, lse = xtern.paged_attention(cache, torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda(),
                                     q.cuda(), lse=True)
    out, lse = out.cpu(), lse.cpu()
    assert bool(torch.isfinite(out[0]).all()) and bool(torch.isfinite(out[1:, 2:]).all())
    assert bool(torch.isnan(out[1:, :2]).all()) and not bool(torch.isfinite(lse[1:, :2]).any())
    assert bool(torch.isfinite(lse[:, 2:]).all()) and bool(torch.isfinite(lse[0]).all())
    # every score -inf: nothing is left
    pool.k[:] = torch.where(torch.isnan(pool.k), pool.k, torch.full((), -float("inf"), dtype=dtype))
    cache = pool.upload()
    out, lse = xtern.paged_attention(cache, torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda(),
                                     q.cuda(), lse=True)
    assert bool((out == 0).all()) and bool((lse == -float("inf")).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_infinities_of_a_split_row(dtype):
    """An infinite key or value far into a long row: NaN or infinity where the
    formula has them, the other heads and rows untouched by it."""
    page, H, D, n = 16, 2, 64, 3000
    rng = np.random.default_rng(8)
    pool = Pool(rng, 2 * 188 + 2, page, H, D, dtype, score=True)
    table = ref.tables(rng, [n, n], page, pool.P)
    pool.fill(rng, table, [n, n])
    q = torch.from_numpy(rng.standard_normal((2, 4, D)).astype(np.float32))
    clean = ref.attention(pool.k, pool.v, table, page, q, [n, n], None, D ** -0.5)
    pg, sl = int(table[0, 2500 // page]), 2500 % page
    pool.v[pg, sl, 0, 3] = float("inf")
    pool.k[int(table[0, 700 // page]), 700 % page, 1, :] = float("nan")
    cache = pool.upload()
    out, lse = xtern.paged_attention(cache, torch.from_numpy(table).cuda(), torch.tensor([n, n], dtype=torch.int32).cuda(),
                                     q.cuda(), lse=True)
    out, lse = out.cpu(), lse.cpu()
    ref.close(out[1], clean[0][1], clean[3][1], "the other row")
    ref.close(lse[1], clean[1][1], clean[4][1], "its lse")
    rest = [d for d in range(D) if d != 3]
    ref.close(out[0, :2][:, rest], clean[0][0, :2][:, rest], clean[3][0, :2][:, rest], "the other columns")
    assert bool((out[0, :2, 3] == float("inf")).all())
    ref.close(lse[0, :2], clean[1][0, :2], clean[4][0, :2], "lse")
    assert bool(torch.isnan(out[0, 2:]).all()) and bool(torch.isnan(lse[0, 2:]).all())


def test_attention_strided_rows():
    """q and out as parts of wider rows; the rest of out stays."""
    rng = np.random.default_rng(5)
    hq, H, D, page, lens = 4, 2, 64, 16, [30, 61]
    pool = Pool(rng, 8, page, H, D, torch.bfloat16)
    table = ref.tables(rng, lens, page, 8)
    pool.fill(rng, table, lens)
    wide = torch.from_numpy(rng.standard_normal((2, 3 * hq * D + 5)).astype(np.float32)).cuda()
    q, res = wide[:, 1:1 + hq * D], torch.full((2, hq * D + 3), 7.0, device="cuda")
    cache, dt = pool.upload(), torch.from_numpy(np.ascontiguousarray(table)).cuda()
    wide_table = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide_table[:, 2:2 + table.shape[1]] = dt
    got = xtern.paged_attention(cache, wide_table[:, 2:2 + table.shape[1]], torch.tensor(lens, dtype=torch.int32).cuda(),
                                q, out=res[:, 2:2 + hq * D])
    want = ref.attention(pool.k, pool.v, table, page, q.cpu().reshape(2, hq, D), lens, None, D ** -0.5)
    ref.close(got.reshape(2, hq, D), want[0], want[3], "out")
    assert bool((res[:, :2] == 7).all()) and bool((res[:, -1] == 7).all())


def test_attention_in_place():
    """out = q: whole rows, rows in parts, rows in plain operations (a tiny
    head; infinite values), many rows, columns of a wider tensor."""
    g = torch.Generator().manual_seed(11)
    for dtype in DTYPES:
        for hq, H, D, R, length in ((8, 2, 128, 3, 90), (20, 1, 64, 2, 9000), (4, 2, 3, 5, 300), (4, 4, 256, 300, 40)):
            pages = -(-length // 16)
            c = xtern.KvCache.new(pages, 16, H, D, dtype=dtype, score=True)
            c.k.copy_(torch.randn(c.k.shape, generator=g))
            c.v.copy_(torch.randn(c.v.shape, generator=g))
            c.v[0, 3, 0, 0] = float("inf")
            table = torch.arange(pages, dtype=torch.int32, device="cuda").reshape(1, pages)
            seq = torch.zeros(R, dtype=torch.int32, device="cuda")
            lengths = torch.randint(0, length + 1, (R,), generator=g, dtype=torch.int32).cuda()
            lengths[0] = length
            wide = torch.randn((R, hq * D + 5), generator=g).cuda()
            q = wide[:, 2:hq * D + 2]
            want, lse = xtern.paged_attention(c, table, lengths, q.clone(), seq=seq, lse=True)
            edge = wide.clone()
            got, lse2 = xtern.paged_attention(c, table, lengths, q, seq=seq, lse=True, out=q, accumulate=True)
            assert got is q and same_bits(got, want) and same_bits(lse, lse2), (dtype, D)
            edge[:, 2:hq * D + 2] = want
            assert same_bits(wide, edge)


def test_attention_empty_calls():
    cache = xtern.KvCache.new(4, 16, 2, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    out = xtern.paged_attention(cache, torch.zeros((0, 3), **i32), torch.zeros(0, **i32),
                                torch.zeros((0, 4, 64), device="cuda"))
    assert out.shape == (0, 4, 64)
    out, lse = xtern.paged_attention(cache, torch.zeros((2, 0), **i32), torch.ones(2, **i32),
                                     torch.ones((2, 4, 64), device="cuda"), lse=True)
    assert bool((out == 0).all()) and bool((lse == -float("inf")).all())


# --- append ----------------------------------------------------------------

def append_case(dtype, hq, H, D, rot, page, layout, with_q=True, seed=0, in_place=False):
    rng = np.random.default_rng(seed)
    num = 240 // page + 4
    pool = Pool(rng, num, page, H, D, dtype, layout, score=True)
    table = ref.tables(rng, [64 + page] * 2 if page > 40 else [64, 20], page, num)
    S, cap = table.shape[0], table.shape[1] * page
    slots = np.array([0, 1, 5, page, 63, -1, cap, cap - 1, 2, 0, 3, 7], np.int32)
    seq = np.array([0, 0, 0, 0, 0, 0, 0, 0, 1, 1, S, 1], np.int32)
    pos = np.array([3, 900, 0, 17, 999, 4, 4, 4, -1, 1000, 4, 5], np.int32)
    R = len(slots)
    q, k, v = (torch.from_numpy(rng.standard_normal((R, h, D)).astype(np.float32)) for h in (hq, H, H))
    half = rot // 2
    ang = np.arange(1000)[:, None] * 10000.0 ** (-np.arange(half) / max(half, 1))
    cos, sin = torch.from_numpy(np.cos(ang).astype(np.float32)), torch.from_numpy(np.sin(ang).astype(np.float32))
    cache = pool.upload()
    dq = q.cuda()
    out = dq if in_place else torch.full_like(dq, -7.0)
    before = out.cpu().clone()
    xtern.kv_append(cache, torch.from_numpy(table).cuda(), torch.from_numpy(slots).cuda(), k.cuda(), v.cuda(),
                    q=dq if with_q else None, seq=torch.from_numpy(seq).cuda(),
                    positions=torch.from_numpy(pos).cuda() if rot else None,
                    rope=(cos.cuda(), sin.cuda()) if rot else None, q_out=out if with_q else None)
    torch.cuda.synchronize()

    def turned(x, r):
        x = x.double()
        if not rot:
            return x, torch.zeros_like(x)
        c, s = cos[pos[r]].double(), sin[pos[r]].double()
        a, b = x[:, :half], x[:, half:rot]
        bound = 3 * ref.EPS * ((a * c).abs() + (b * s).abs()), 3 * ref.EPS * ((b * c).abs() + (a * s).abs())
        rest = x[:, rot:]
        return torch.cat([a * c - b * s, b * c + a * s, rest], 1), torch.cat([*bound, torch.zeros_like(rest)], 1)

    want_q, half_step = before.clone().double(), ref.HALF[dtype]
    gk, gv = pool.view[0](pool.dev[0]).cpu(), pool.view[1](pool.dev[1]).cpu()
    done = 0
    for r in range(R):
        ok = (0 <= slots[r] < cap and 0 <= seq[r] < S and (not rot or 0 <= pos[r] < 1000)
              and 0 <= table[seq[r] % S][min(max(slots[r], 0), cap - 1) // page] < num)
        got_q = out[r].cpu()
        if not ok:
            assert same_bits(got_q, before[r]), f"row {r} is not there, its q was written"
            continue
        done += 1
        pg, sl = int(table[seq[r], slots[r] // page]), slots[r] % page
        if with_q:
            w, tol = turned(q[r], r)
            ref.close(got_q, w, tol, f"q row {r}")
        w, tol = turned(k[r], r)
        # (the rounding to the cache's type: half a step of the value, or of
        # the type's smallest step)
        tiny = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dtype]
        ref.close(gk[pg, sl], w, tol * (1 + half_step) + half_step * w.abs() + tiny, f"k row {r}")
        assert same_bits(gv[pg, sl], v[r].to(dtype)), f"v row {r}"
        pool.k[pg, sl], pool.v[pg, sl] = gk[pg, sl], gv[pg, sl]
        pool.score[pg, :, sl] = 0.0
    assert done >= 5
    for a, b in zip(pool.dev, pool.mem):
        assert same_bits(a, b), "other memory changed"
    assert same_bits(pool.dscore, pool.score)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("layout", ref.LAYOUTS)
@pytest.mark.parametrize("shape", [(20, 5, 128, 128), (4, 4, 100, 100), (4, 2, 64, 32), (3, 1, 7, 2), (2, 1, 1, 0),
                                   (8, 1, 256, 0)], ids=str)
def test_append(dtype, layout, shape):
    log(f"append {dtype} {layout} {shape}")
    append_case(dtype, *shape, page=16, layout=layout)


@pytest.mark.parametrize("page", [1, 3, 24, 64])
def test_append_forms(page):
    for dtype in DTYPES:
        append_case(dtype, 4, 2, 64, 64, page if page > 1 else 8, "page_head_slot", in_place=True, seed=page)
        append_case(dtype, 4, 2, 64, 64, page if page > 1 else 8, "joint", with_q=False, seed=page)


def test_append_parts_of_wider_rows():
    """q, k and v as columns of one fused tensor, q rotated where it lies."""
    rng = np.random.default_rng(9)
    hq, H, D, page = 4, 2, 64, 16
    for dtype in DTYPES:
        fused = torch.from_numpy(rng.standard_normal((5, (hq + 2 * H) * D + 3)).astype(np.float32)).cuda()
        q, k, v = (fused[:, a * D + 1:b * D + 1] for a, b in ((0, hq), (hq, hq + H), (hq + H, hq + 2 * H)))
        table = torch.arange(10, dtype=torch.int32, device="cuda").reshape(5, 2)
        slots = torch.tensor([0, 31, 16, 15, -1], dtype=torch.int32, device="cuda")
        ang = torch.rand((40, D // 2), device="cuda")
        rope = (ang.cos().contiguous(), ang.sin().contiguous())
        a, b = (xtern.KvCache.new(10, page, H, D, dtype=dtype) for _ in range(2))
        want = xtern.kv_append(a, table, slots, k.contiguous(), v.contiguous(), q=q.contiguous(), rope=rope,
                               q_out=q.contiguous().clone())
        before = fused.clone()
        xtern.kv_append(b, table, slots, k, v, q=q, rope=rope, q_out=q)
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(q, want)
        before[:, 1:hq * D + 1] = q
        assert torch.equal(before, fused)


def test_append_special_values():
    """Overflow to infinity, subnormals, ties to even, NaN."""
    vals = torch.tensor([65519.0, 65520.0, 1e38, -1e38, 3.4e38, 1e-8, -6e-8, 5.9e-8, 1 + 2 ** -8, 1 + 3 * 2 ** -8,
                         1 + 2 ** -11, float("nan"), float("inf"), -0.0, 1e-45, 2 ** -133.0])
    i32 = dict(dtype=torch.int32, device="cuda")
    for dtype in DTYPES:
        cache = xtern.KvCache.new(1, 4, 1, 16, dtype=dtype)
        kv = vals.reshape(1, 1, 16).cuda()
        xtern.kv_append(cache, torch.zeros((1, 1), **i32), torch.tensor([2], **i32), kv, kv)
        want = vals.to(dtype)
        for got in (cache.k[0, 2, 0], cache.v[0, 2, 0]):
            got = got.cpu()
            nan = torch.isnan(want)
            assert torch.equal(torch.isnan(got), nan) and same_bits(got[~nan], want[~nan])


def test_append_no_rows():
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = xtern.KvCache.new(2, 16, 2, 64)
    e = torch.zeros((0, 2, 64), device="cuda")
    assert xtern.kv_append(cache, torch.zeros((1, 2), **i32), torch.zeros(0, **i32), e, e) is None


# --- eviction --------------------------------------------------------------

def evict_case(dtype, H, D, page, lens, budget, sink, recent, layout="page_head_slot", seed=0, edit=None):
    rng = np.random.default_rng(seed)
    num = sum((n + page - 1) // page for n in lens) + 2
    pool = Pool(rng, num, page, H, D, dtype, layout, score=True)
    table = ref.tables(rng, lens, page, num)
    pool.fill(rng, table, lens)
    pool.score = torch.from_numpy(rng.choice([0.0, -0.0, 0.25, 0.5, 1.0, 3.0], pool.score.shape).astype(np.float32)
                                  * rng.integers(1, 40, pool.score.shape).astype(np.float32))
    lengths = np.asarray(lens, np.int32)
    if edit:
        edit(table, lengths, pool)
    cache = pool.upload()
    new, kept = xtern.kv_evict(cache, torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda(), budget,
                               sink=sink, recent=recent)
    torch.cuda.synchronize()
    wnew, wkept = ref.evict(pool.k, pool.v, pool.score, table, page, lengths, budget, sink, recent)
    assert np.array_equal(new.cpu().numpy(), wnew)
    assert np.array_equal(kept.cpu().numpy(), wkept)
    assert same_bits(pool.dscore, pool.score)
    for a, b in zip(pool.dev, pool.mem):
        assert same_bits(a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("layout", ref.LAYOUTS)
def test_evict_layouts(dtype, layout):
    for D in (64, 100, 37):
        evict_case(dtype, 3, D, 16, [100, 33, 50, 51, 200], 50, 4, 8, layout=layout)


@pytest.mark.parametrize("page", [1, 3, 16, 100])
@pytest.mark.parametrize("rule", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (20, 10, 10), (20, 20, 0), (20, 0, 20), (20, 0, 0),
                                  (63, 3, 7), (64, 0, 1), (65, 1, 0), (299, 0, 0), (299, 4, 5)], ids=str)
def test_evict_rules(page, rule):
    log(f"evict page {page} {rule}")
    evict_case(torch.bfloat16, 2, 32, page, [300, 64, 1, 0, 65, 21], *rule, seed=page)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_evict_long(dtype):
    for n, budget in ((5000, 1), (5000, 4999), (9000, 2500), (20011, 7000), (16384 + 4, 16380), (16385 + 4, 16000)):
        log(f"evict {dtype} {n} {budget}")
        evict_case(dtype, 1, 64, 32, [n], budget, min(4, budget), 0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D,layout", [(64, "page_head_slot"), (100, "odd"), (37, "joint"), (256, "head_first")])
def test_evict_many_rows_of_few_heads(dtype, D, layout):
    """Thousands of kept rows: moved through a workspace where heads are few,
    in place where they are many."""
    log(f"evict {dtype} {D} {layout}")
    evict_case(dtype, 1, D, 16, [6000, 4500, 4300], 4400, 7, 100, layout=layout)
    evict_case(dtype, 2, D, 48, [5000], 4096 + 3, 3, 0, layout=layout)


def test_evict_budgets_and_lengths():
    """Budgets above the table's capacity; several long sequences whose keys
    go through the workspace."""
    evict_case(torch.bfloat16, 2, 32, 16, [100, 50], 5000, 3, 4)
    evict_case(torch.float16, 2, 8, 16, [17000, 20000, 300], 400, 2, 5)
    evict_case(torch.float16, 1, 4, 16, [17000, 20000], 16700, 0, 5)  # (rows below one piece)


def test_evict_largest_budget():
    """A list of 2^31 - 1 entries, none of it past its end."""
    c = xtern.KvCache.new(4, 16, 1, 8, score=True)
    c.k.copy_(torch.randn(c.k.shape))
    before = c.k.clone()
    table = torch.arange(4, dtype=torch.int32, device="cuda").reshape(1, 4)
    lengths = torch.tensor([50], dtype=torch.int32, device="cuda")
    new, kept = xtern.kv_evict(c, table, lengths, 2 ** 31 - 1, sink=2 ** 30, recent=2 ** 30 - 1)
    assert new.tolist() == [50] and kept[0, 0, :50].tolist() == list(range(50))
    assert int(kept[0, 0, 50:].max()) == -1 and int(kept[0, 0, 50:].min()) == -1
    assert torch.equal(c.k, before)
    del kept
    torch.cuda.empty_cache()


def test_evict_more_sequences_than_a_grid_side():
    """70000 sequences, the last one long: as in a call of its own."""
    S, page = 70000, 16500
    k, v = (torch.randn((2, page, 1, 8)).half().cuda() for _ in range(2))
    score = torch.rand((2, 1, page)).cuda()
    one, many = (xtern.KvCache(k.clone(), v.clone(), score.clone()) for _ in range(2))
    table = torch.full((S, 1), -1, dtype=torch.int32, device="cuda")
    table[-1] = 1
    lengths = torch.arange(S, dtype=torch.int32, device="cuda") % 9
    lengths[-1] = page
    new, kept = xtern.kv_evict(many, table, lengths, 40, sink=2, recent=3)
    new1, kept1 = xtern.kv_evict(one, table[-1:], lengths[-1:], 40, sink=2, recent=3)
    assert torch.equal(new[:-1], lengths[:-1]) and int(new[-1]) == int(new1[0]) == 40
    assert torch.equal(kept[-1:], kept1) and int(kept1.min()) == 0
    assert torch.equal(one.k, many.k) and torch.equal(one.v, many.v) and torch.equal(one.score, many.score)
    want = torch.where(torch.arange(40, device="cuda") < lengths[:-1, None], torch.arange(40, device="cuda"), -1)
    assert torch.equal(kept[:-1, 0], want.int())


def test_evict_scores():
    """Equal scores, NaN, infinities, negative ones, holes in the table,
    lengths that the table does not hold."""
    def edit(table, lengths, pool):
        table[0, 2] = -1
        table[1, 0] = pool.P + 3
        table[2, -2] = -1
        pool.score[::2, 0] = 0.0
        pool.score[1::3, 1, 2] = float("nan")
        pool.score[::5, 1, 3] = float("inf")
        pool.score[::4, 1, 4] = -float("inf")
        pool.score[::4, 1, 5] = -2.5
        lengths[3] = 2 ** 31 - 1
        lengths[4] = -3

    for budget, sink, recent in ((40, 0, 0), (40, 4, 20), (90, 40, 0)):
        evict_case(torch.float16, 2, 64, 16, [150, 128, 111, 100, 100], budget, sink, recent, edit=edit)


def test_evict_no_sequences():
    cache = xtern.KvCache.new(2, 16, 2, 64, score=True)
    i32 = dict(dtype=torch.int32, device="cuda")
    new, kept = xtern.kv_evict(cache, torch.zeros((0, 2), **i32), torch.zeros(0, **i32), 4)
    assert new.shape == (0,) and kept.shape == (0, 2, 4)
