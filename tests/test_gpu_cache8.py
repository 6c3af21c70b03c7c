"""The 8-bit cache: norms, rotation and codes as they are written, positions
read back, attention over the codes; and windows and several tokens of a
sequence over every type of cache, against plain 64-bit forms.  Memory that a
call must not look at holds what would show."""
import threading

import numpy as np
import pytest
import torch

import cache8_ref as ref
import xtern
from cache_ref import LAYOUTS, close, tables
from test_gpu_cache import log

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")
TYPES = [torch.int8, torch.float32, torch.float16, torch.bfloat16]
NAN = float("nan")


class Pool:
    """A pool on the host, every element and scale a poison (NaN, or codes of
    -128 with scales of NaN), and its copy on the device."""

    def __init__(self, num_pages, page, H, D, dtype, layout="page_head_slot", score=None):
        codes = dtype == torch.int8
        fill = -128 if codes else NAN
        shapes = {"page_head_slot": ((num_pages, H, page, D), lambda m: m.transpose(1, 2)),
                  "page_slot_head": ((num_pages, page, H, D), lambda m: m),
                  "head_first": ((H, num_pages, page, D), lambda m: m.permute(1, 2, 0, 3)),
                  "odd": ((num_pages, page, H, D + 1), lambda m: m[..., 1:])}
        if layout == "joint":  # k and v of a page side by side
            m = torch.full((num_pages, 2, page, H, D), fill, dtype=dtype)
            self.mem, self.view = [m, m], [lambda m: m[:, 0], lambda m: m[:, 1]]
        else:
            shape, view = shapes[layout]
            self.mem = [torch.full(shape, fill, dtype=dtype) for _ in range(2)]
            self.view = [view, view]
        self.scales = [torch.full((num_pages, H, page), NAN) for _ in range(2)] if codes else [None, None]
        self.score, self.page, self.P, self.dtype = score, page, num_pages, dtype
        self.k, self.v = (f(m) for f, m in zip(self.view, self.mem))

    def fill(self, rng, table, lens, std=1.0):
        for b, n in enumerate(lens):
            for _, pg, sl in ref.visible(table[b], n, self.page, self.P, 0, 0):
                for x, s in zip((self.k, self.v), self.scales):
                    y = torch.from_numpy(rng.standard_normal(tuple(x.shape[2:])) * std)
                    if s is None:
                        x[pg, sl] = y.to(x.dtype)
                    else:
                        x[pg, sl], s[pg, :, sl] = ref.codes(y)

    def upload(self):
        one = self.mem[0] is self.mem[1]
        self.dev = [self.mem[0].cuda()]
        self.dev.append(self.dev[0] if one else self.mem[1].cuda())
        self.dscales = [s.cuda() if s is not None else None for s in self.scales]
        self.dscore = self.score.cuda() if self.score is not None else None
        return xtern.KvCache(self.view[0](self.dev[0]), self.view[1](self.dev[1]), self.dscore, *self.dscales)

    def unchanged(self):
        for a, b in zip(self.dev + self.dscales, self.mem + self.scales):
            if a is not None:
                a = a.cpu()
                assert torch.equal(a[a == a], b[b == b]) and torch.equal(a == a, b == b), "the cache changed"


def same(a, b):
    """Equal values, NaN in the same places."""
    nan = torch.isnan(a.float()), torch.isnan(b.float())
    return bool(torch.equal(*nan) and torch.equal(a[~nan[0]], b[~nan[1]]))


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


# --- attention -------------------------------------------------------------

def attention_case(dtype, hq, H, D, page, lens, window=0, sink=0, tokens=1, lengths=None, seq=None, layout="page_head_slot",
                   accumulate=False, scale=None, std=1.0, seed=0, edit=None, q=None):
    """tokens > 1: the last `tokens` positions of each sequence, unless lengths
    are given."""
    rng = np.random.default_rng(seed)
    num = sum((n + page - 1) // page for n in lens) + 2
    pool = Pool(num, page, H, D, dtype, layout,
                torch.from_numpy(rng.random((num, H, page)).astype(np.float32)) if accumulate else None)
    table = tables(rng, lens, page, num)
    pool.fill(rng, table, lens, std)
    if lengths is None:
        lengths = [max(0, n - tokens + 1 + t) for n in lens for t in range(tokens)]
    lengths = np.asarray(lengths, np.int32)
    if edit:
        edit(table, lengths, pool)
    if q is None:
        q = torch.from_numpy(rng.standard_normal((len(lengths), hq, D)).astype(np.float32))
    scale = D ** -0.5 if scale is None else scale
    want = ref.attention(pool.k, pool.v, table, page, q, lengths, seq, scale, *pool.scales, window, sink, tokens, pool.score)
    cache = pool.upload()
    out, lse = xtern.paged_attention(cache, dev(table), dev(lengths), q.cuda(), scale=scale, lse=True,
                                     seq=None if seq is None else torch.tensor(seq, **I32), accumulate=accumulate,
                                     window=window or None, sink=sink, tokens=tokens)
    torch.cuda.synchronize()
    close(out, want[0], want[3], "out")
    close(lse, want[1], want[4], "lse")
    if accumulate:
        close(pool.dscore, want[2], want[5], "score")
    pool.unchanged()


HEADS = [(1, 1, 64), (4, 4, 100), (20, 5, 128), (16, 2, 80), (8, 1, 256), (24, 2, 96), (40, 2, 33), (3, 1, 1), (32, 1, 192),
         (12, 3, 7), (34, 2, 16), (5, 5, 17), (6, 2, 15), (7, 1, 250), (17, 1, 129)]


@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_codes_heads(heads):
    log(f"attention8 {heads}")
    attention_case(torch.int8, *heads, page=16, lens=[1, 37, 0, 130])
    attention_case(torch.int8, *heads, page=16, lens=[3, 90, 260], tokens=3)


@pytest.mark.parametrize("page", [1, 2, 3, 7, 8, 24, 33, 64, 1000])
def test_codes_pages(page):
    log(f"attention8 page {page}")
    attention_case(torch.int8, 4, 2, 64, page, lens=[1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 257])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("D", [64, 100, 128, 37])
def test_codes_layouts(layout, D):
    log(f"attention8 {layout} {D}")
    attention_case(torch.int8, 6, 3, D, 16, lens=[70, 5, 259], layout=layout)


@pytest.mark.parametrize("lens", [[4097], [1, 5000], [3000] * 3, [511, 512, 513, 1023, 1024, 1025], [20000]], ids=str)
@pytest.mark.parametrize("tokens", [1, 3])
def test_codes_long(lens, tokens):
    log(f"attention8 {lens} {tokens}")
    attention_case(torch.int8, 8, 2, 128, 32, lens=lens, tokens=tokens)


@pytest.mark.parametrize("heads", [(1, 1, 64), (2, 1, 130), (4, 2, 255), (6, 2, 200), (17, 1, 64), (10, 5, 36)], ids=str)
def test_codes_long_heads(heads):
    """Rows in many segments for one, two and more columns."""
    log(f"attention8 {heads} long")
    attention_case(torch.int8, *heads, page=16, lens=[9000, 140])


def test_codes_row_counts():
    """More units than a wave has lanes, some of them split; more than are
    split at all."""
    rng = np.random.default_rng(4)
    lens = [int(x) for x in rng.integers(0, 60, 150)]
    lens[3], lens[70], lens[149] = 3000, 1500, 2500
    attention_case(torch.int8, 4, 2, 64, 16, lens=lens)
    attention_case(torch.int8, 32, 2, 64, 16, lens=lens[:90], tokens=2)
    long = [300, 20, 1, 150, 64]
    seq = [i // 4 % 5 for i in range(1200)]
    lengths = [(37 * i) % (long[b] + 1) for i, b in enumerate(seq)]
    attention_case(torch.int8, 4, 2, 64, 16, lens=long, seq=seq, lengths=lengths)
    attention_case(torch.int8, 20, 2, 64, 16, lens=long, seq=seq, lengths=lengths, tokens=4, window=40, sink=3)


def test_codes_spread():
    """Scores hundreds apart, equal scores, a scale below zero, queries and
    keys of very different sizes."""
    for scale, std in ((2.0, 3.0), (0.0, 1.0), (-0.3, 1.0), (1e-3, 100.0), (1e20, 1e-20), (1e-25, 1e25)):
        attention_case(torch.int8, 8, 2, 64, 16, lens=[200, 33], scale=scale, std=std)


def test_codes_tiny_values():
    """Value scales that the weights' digits have no room for."""
    for std in (1e-25, 1e-30, 1e-33):
        attention_case(torch.int8, 8, 2, 64, 16, lens=[200, 33], std=std)


def test_codes_one_large_query_element():
    rng = np.random.default_rng(6)
    q = torch.from_numpy(rng.standard_normal((2, 8, 64)).astype(np.float32))
    q[0, :, 5] = 3000.0
    q[1, 3] = 0.0
    q[1, 4] = 1e-30
    attention_case(torch.int8, 8, 2, 64, 16, lens=[200, 33], q=q, scale=1e-3)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("window,sink", [(1, 0), (1, 4), (16, 0), (100, 4), (128, 64), (129, 1), (1000, 3), (2 ** 30, 2 ** 30)])
def test_windows(dtype, window, sink):
    """Shorter, equal and longer sequences; several tokens, empty rows."""
    log(f"window {dtype} {window} {sink}")
    lens = [0, 1, 5, 16, window % 4096, window % 4096 + sink % 4096, window % 4096 + sink % 4096 + 1, 300, 1500]
    acc = dtype != torch.int8
    attention_case(dtype, 8, 2, 64, 16, lens=lens, window=window, sink=sink, accumulate=acc)
    attention_case(dtype, 8, 2, 64, 16, lens=[max(3, n) for n in lens], window=window, sink=sink, tokens=3, accumulate=acc)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads", [(20, 5, 128), (12, 3, 100), (7, 1, 256), (40, 2, 33), (6, 2, 5)], ids=str)
def test_windows_heads(dtype, heads):
    log(f"window {dtype} {heads}")
    attention_case(dtype, *heads, page=24, lens=[5000, 77, 400], window=300, sink=5, tokens=2, accumulate=dtype != torch.int8)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens", [1, 2, 5, 16, 33])
def test_tokens(dtype, tokens):
    """Groups of tokens, with padded rows and rows in any order of lengths;
    a group belongs to the sequence of its first row."""
    log(f"tokens {dtype} {tokens}")
    lens = [700, 90, 40, 2000]
    for hq, H in ((4, 4), (10, 2), (32, 1)):
        attention_case(dtype, hq, H, 64, 16, lens=lens, tokens=tokens)
        seq = [s for b in (2, 0, 3, 9, -1) for s in [b] + [0] * (tokens - 1)]
        rng = np.random.default_rng(tokens)
        lengths = rng.integers(0, 41, len(seq))
        lengths[::3] = 0
        lengths[2 * tokens] = 1999
        attention_case(dtype, hq, H, 64, 16, lens=lens, tokens=tokens, seq=seq, lengths=lengths)
        attention_case(dtype, hq, H, 64, 16, lens=lens, tokens=tokens, seq=seq, lengths=lengths, window=15, sink=2)


def test_prompt():
    """A prompt of 300 tokens in one group."""
    for dtype in TYPES:
        attention_case(dtype, 4, 2, 64, 16, lens=[300], tokens=300, lengths=range(1, 301))
        attention_case(dtype, 4, 2, 64, 16, lens=[300], tokens=300, lengths=range(1, 301), window=20, sink=1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_holes(dtype):
    """Entries that are no page, lengths past the table and below zero, whole
    rows without a page, windows that lie in the holes."""
    def edit(table, lengths, pool):
        table[0, 1] = -1
        table[0, 3] = pool.P
        table[1, :] = -7
        table[2, 0] = 2 ** 31 - 1
        table[3, 4:] = -1
        lengths[4] = -5
        lengths[5] = 2 ** 31 - 1
        lengths[6] = 10 ** 6

    for window, sink in ((0, 0), (50, 3), (10, 70)):
        attention_case(dtype, 8, 2, 64, 16, lens=[100, 40, 300, 200, 33, 64, 50], edit=edit, window=window, sink=sink)

    def front(table, lengths, pool):
        table[0, :240] = -1
        table[1, 10:100] = -1

    for window, sink in ((0, 0), (200, 4)):
        attention_case(dtype, 8, 2, 64, 16, lens=[4000, 2000, 30], edit=front, window=window, sink=sink)


def test_not_a_number():
    """A key or value that is no number shows where a row sees it, and only
    there: other heads, rows, tokens of the same pass and positions outside the
    window stay."""
    page, H, D, n = 16, 2, 64, 200
    rng = np.random.default_rng(1)
    pool = Pool(16, page, H, D, torch.int8)
    table = tables(rng, [n], page, 16, spare=0)
    pool.fill(rng, table, [n])
    q = torch.from_numpy(rng.standard_normal((4, 4, D)).astype(np.float32))
    lengths = np.array([50, 51, 150, 200], np.int32)
    clean = ref.attention(pool.k, pool.v, table, page, q, lengths, None, 0.1, *pool.scales, 0, 0, 4)
    windowed = ref.attention(pool.k, pool.v, table, page, q, lengths, None, 0.1, *pool.scales, 60, 2, 4)
    at = int(table[0, 50 // page]), 50 % page
    for which, bad in ((0, NAN), (1, NAN), (0, float("inf")), (1, float("inf"))):
        scales = [s.clone() for s in pool.scales]
        scales[which][at[0], 1, at[1]] = bad
        c = xtern.KvCache(pool.k.cuda(), pool.v.cuda(), None, *(s.cuda() for s in scales))
        got = xtern.paged_attention(c, dev(table), dev(lengths), q.cuda(), scale=0.1, tokens=4).cpu()
        close(got[0], clean[0][0], clean[3][0], "before it")
        close(got[:, :2], clean[0][:, :2], clean[3][:, :2], "the other head")
        assert not bool(torch.isfinite(got[1:, 2:]).all(-1).any()), which
        got = xtern.paged_attention(c, dev(table), dev(lengths), q.cuda(), scale=0.1, tokens=4, window=60, sink=2).cpu()
        close(got[[0, 2, 3]], windowed[0][[0, 2, 3]], windowed[3][[0, 2, 3]], "outside the window")
        assert not bool(torch.isfinite(got[1, 2:]).all(-1).any())
    # a query that is no number: its own head alone
    c = pool.upload()
    q[2, 1, 7] = float("inf")
    q[3, 2, 0] = NAN
    got = xtern.paged_attention(c, dev(table), dev(lengths), q.cuda(), scale=0.1, tokens=4).cpu()
    bad = torch.zeros((4, 4), dtype=torch.bool)
    bad[2, 1] = bad[3, 2] = True
    close(got[~bad], clean[0][~bad], clean[3][~bad], "the other rows and heads")
    assert not bool(torch.isfinite(got[bad]).all(-1).any())


def test_scales_of_any_sign():
    """Scales that no append writes: negative ones, zeros."""
    def edit(table, lengths, pool):
        for s in pool.scales:
            s[::2] *= -1.0
            s[1::3, 0] = torch.where(torch.isnan(s[1::3, 0]), s[1::3, 0], 0.0)

    attention_case(torch.int8, 8, 2, 64, 16, lens=[200, 33, 1000], edit=edit)


def test_strided_and_in_place():
    """q and out as parts of wider rows, out = q, a table that is part of a
    wider one."""
    rng = np.random.default_rng(5)
    hq, H, D, page, lens, T = 4, 2, 64, 16, [30, 61], 3
    pool = Pool(8, page, H, D, torch.int8)
    table = tables(rng, lens, page, 8)
    pool.fill(rng, table, lens)
    lengths = np.array([n - T + 1 + t for n in lens for t in range(T)], np.int32)
    wide = torch.from_numpy(rng.standard_normal((2 * T, 3 * hq * D + 5)).astype(np.float32)).cuda()
    q, res = wide[:, 1:1 + hq * D], torch.full((2 * T, hq * D + 3), 7.0, device="cuda")
    want = ref.attention(pool.k, pool.v, table, page, q.cpu().reshape(2 * T, hq, D), lengths, None, D ** -0.5,
                         *pool.scales, 20, 1, T)
    cache = pool.upload()
    wide_table = torch.full((2, table.shape[1] + 5), -1, **I32)
    wide_table[:, 2:2 + table.shape[1]] = dev(table)
    args = dict(window=20, sink=1, tokens=T)
    got = xtern.paged_attention(cache, wide_table[:, 2:2 + table.shape[1]], dev(lengths), q, out=res[:, 2:2 + hq * D], **args)
    close(got.reshape(2 * T, hq, D), want[0], want[3], "out")
    assert bool((res[:, :2] == 7).all()) and bool((res[:, -1] == 7).all())
    same = xtern.paged_attention(cache, wide_table[:, 2:2 + table.shape[1]], dev(lengths), q, out=q, **args)
    assert same is q and torch.equal(same, got)


def test_offsets_past_32_bits():
    """A pool of 6 GB: the last pages hold the sequence."""
    page, H, D, n = 64, 2, 128, 500
    pages = 190000  # x 64 x 2 x 128 bytes, k and v each 3.1 GB
    k, v = (torch.zeros((pages, H, page, D), dtype=torch.int8, device="cuda").transpose(1, 2) for _ in range(2))
    ks, vs = (torch.zeros((pages, H, page), device="cuda") for _ in range(2))
    c = xtern.KvCache(k, v, None, ks, vs)
    rng = np.random.default_rng(2)
    table = (pages - 1 - np.arange(8))[None].astype(np.int32)
    x, y = (torch.from_numpy(rng.standard_normal((n, H, D)).astype(np.float32)) for _ in range(2))
    slots = torch.arange(n, **I32)
    xtern.kv_append(c, dev(table), slots, x.cuda(), y.cuda(), seq=torch.zeros(n, **I32))
    got = xtern.kv_read(c, dev(table), slots, seq=torch.zeros(n, **I32))
    for a, b in zip(got, (x, y)):
        code, s = ref.codes(b.double())
        assert torch.equal(a.cpu(), code.float() * s[..., None])
    q = torch.from_numpy(rng.standard_normal((1, 4, D)).astype(np.float32))
    out = xtern.paged_attention(c, dev(table), torch.tensor([n], **I32), q.cuda())
    where = dev(table).long()[0]
    want = ref.attention(k[where].cpu(), v[where].cpu(), np.arange(8, dtype=np.int32)[None], page, q, [n], None,
                         D ** -0.5, ks[where].cpu(), vs[where].cpu())
    close(out, want[0], want[3], "out")
    del c, k, v, ks, vs
    torch.cuda.empty_cache()


# --- store and read --------------------------------------------------------

def store_case(dtype, hq, H, D, rot, page, layout="page_head_slot", norm=True, with_q=True, in_place=False, seed=0, rows=None,
               edit=None):
    rng = np.random.default_rng(seed)
    num = 240 // page + 4
    score = torch.from_numpy(rng.random((num, H, page)).astype(np.float32)) if dtype != torch.int8 else None
    pool = Pool(num, page, H, D, dtype, layout, score)
    table = tables(rng, [64 + page] * 2 if page > 40 else [64, 20], page, num)
    S, cap = table.shape[0], table.shape[1] * page
    if rows is None:
        slots = np.array([0, 1, 5, page, 63, -1, cap, cap - 1, 2, 0, 3, 7], np.int32)
        seq = np.array([0, 0, 0, 0, 0, 0, 0, 0, 1, 1, S, 1], np.int32)
        pos = np.array([3, 900, 0, 17, 999, 4, 4, 4, -1, 1000, 4, 5], np.int32)
    else:
        slots, seq = np.arange(rows, dtype=np.int32), np.zeros(rows, np.int32)
        table = rng.permutation(num).astype(np.int32)[None]
        pos = rng.integers(0, 1000, rows).astype(np.int32)
        S, cap = 1, num * page
    R = len(slots)
    q, k, v = (torch.from_numpy((rng.standard_normal((R, h, D)) * np.exp(rng.standard_normal((R, 1, 1)) * 3)).astype(np.float32))
               for h in (hq, H, H))
    if edit:
        edit(q, k, v)
    half = rot // 2
    ang = np.arange(1000)[:, None] * 10000.0 ** (-np.arange(half) / max(half, 1))
    cos, sin = torch.from_numpy(np.cos(ang).astype(np.float32)), torch.from_numpy(np.sin(ang).astype(np.float32))
    wq, wk = (torch.from_numpy((1 + 0.3 * rng.standard_normal(D)).astype(np.float32)) for _ in range(2))
    eps = 1e-6
    cache = pool.upload()
    dq = q.cuda()
    out = dq if in_place else torch.full_like(dq, -7.0)
    before = out.cpu().clone()
    lengths = torch.full((R,), -9, **I32)
    res = xtern.kv_append(cache, dev(table), dev(slots), k.cuda(), v.cuda(), q=dq if with_q else None, seq=dev(seq),
                          positions=dev(pos) if rot else None, rope=(cos.cuda(), sin.cuda()) if rot else None,
                          q_out=out if with_q else None, lengths=lengths,
                          norm=(wq.cuda() if with_q else None, wk.cuda(), eps) if norm else None)
    torch.cuda.synchronize()
    assert res is (out if with_q else None)
    wantq, qtol = before.double(), torch.zeros_like(before, dtype=torch.float64)
    want = [x.clone() for x in (pool.k, pool.v)]
    wants = [s.clone() if s is not None else None for s in pool.scales]
    wscore = pool.score.clone() if score is not None else None
    wlen = np.zeros(R, np.int32)
    for r in range(R):
        if not (0 <= slots[r] < cap and 0 <= seq[r] < S) or (rot and not 0 <= pos[r] < 1000):
            continue
        pg, sl = int(table[seq[r], slots[r] // page]), int(slots[r]) % page
        if not 0 <= pg < num:
            continue
        wlen[r] = slots[r] + 1
        turn = (cos[pos[r]], sin[pos[r]]) if rot else (None, None)
        if with_q:
            wantq[r] = ref.heads(q[r], wq if norm else None, eps, *turn)
            qtol[r] = wantq[r].abs() * ref.EPS * (1 + 1e-6) + 2.0 ** -149
        for i, (x, w) in enumerate(((k, wk), (v, None))):
            y = ref.heads(x[r], w if norm else None, eps, *(turn if i == 0 else (None, None)))
            if dtype == torch.int8:
                want[i][pg, sl], wants[i][pg, :, sl] = ref.codes(y)
            else:
                want[i][pg, sl] = y.float().to(dtype)
        if wscore is not None:
            wscore[pg, :, sl] = 0.0
    close(out, wantq, qtol, "q")
    assert np.array_equal(lengths.cpu().numpy(), wlen)
    for f, m, x in zip(pool.view, pool.dev, want):
        assert same(f(m).cpu(), x), "the cache"
    for got, s in zip(pool.dscales, wants):
        assert s is None or same(got.cpu(), s), "the scales"
    if wscore is not None:
        assert torch.equal(pool.dscore.cpu(), wscore)
    # read back, the rows that were skipped as zeros where they name nothing
    for rd in (torch.float32, torch.float16, torch.bfloat16):
        got = xtern.kv_read(cache, dev(table), dev(slots), seq=dev(seq), dtype=rd)
        for y, x, s in zip(got, want, wants):
            w = torch.zeros((R, H, D), dtype=rd)
            for r in range(R):
                if 0 <= slots[r] < cap and 0 <= seq[r] < S:
                    pg, sl = int(table[seq[r], slots[r] // page]), int(slots[r]) % page
                    if 0 <= pg < num:
                        w[r] = (x[pg, sl].float() * s[pg, :, sl][:, None] if s is not None else x[pg, sl].float()).to(rd)
            assert same(y.cpu(), w), rd


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads", [(4, 2, 64, 64), (20, 5, 128, 128), (6, 3, 100, 50), (8, 2, 256, 256), (5, 5, 33, 32),
                                   (2, 1, 80, 40), (3, 1, 2, 2), (12, 4, 192, 96), (4, 2, 7, 0), (4, 1, 1, 0),
                                   (4, 2, 130, 64), (4, 2, 66, 66), (4, 2, 96, 8)], ids=str)
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
def test_store(dtype, heads, norm):
    """(16- and 32-bit caches without norms have another kernel, in 32 bits:
    test_gpu_cache.py.)"""
    if not norm and dtype != torch.int8:
        pytest.skip("the append of 32 bits")
    log(f"store {dtype} {heads} {norm}")
    store_case(dtype, *heads, page=16, norm=norm)
    store_case(dtype, *heads, page=50, norm=norm, in_place=True, seed=1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("D", [64, 37])
def test_store_layouts(dtype, layout, D):
    store_case(dtype, 4, 2, D, D // 4 * 2, 16, layout=layout)
    store_case(dtype, 4, 2, D, 0, 9, layout=layout, with_q=False)
    store_case(dtype, 4, 2, D, 0, 9, layout=layout, norm=False)  # (nothing to rotate: exact by either kernel)


@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16], ids=str)
@pytest.mark.parametrize("D,rot", [(100, 100), (64, 36), (64, 50), (256, 12), (192, 90), (36, 34), (252, 26), (128, 2), (4, 2)])
def test_store_rotations(dtype, D, rot):
    """Halves of every remainder by four, in place and not.  (16-bit caches without
    norms: the append of 32 bits.)"""
    store_case(dtype, 4, 2, D, rot, 16)
    store_case(dtype, 4, 2, D, rot, 16, in_place=True, norm=dtype != torch.int8)


def test_store_many_rows():
    for dtype in TYPES:
        for D, norm in ((64, True), (100, dtype != torch.int8), (37, True)):
            store_case(dtype, 8, 2, D, D // 4 * 2, 16, rows=250, norm=norm, seed=3)


def test_store_special_values():
    """Infinities and NaN, a head of zeros, the least and the largest
    magnitudes, codes at the borders."""
    def edit(q, k, v):
        k[0, 0, 3] = float("inf")
        v[0, 1, 0] = NAN
        k[1] = 0.0
        v[1] = 2.0 ** -120
        k[2] = 1e-45
        v[2, 0] = 3e38
        v[2, 1] = torch.tensor([127.0, 126.5, 125.5, -0.5, 0.5, 1.5, -126.5] + [0.0] * 57)
        v[3, 0] = -0.0
        v[3, 1, :] = 2.0 ** -119
        q[4, 0] = 0.0

    store_case(torch.int8, 4, 2, 64, 64, 16, edit=edit)
    store_case(torch.int8, 4, 2, 64, 0, 16, edit=edit, norm=False)


def test_read_many_rows():
    """Every position, several times and in any order; rows of wide heads."""
    rng = np.random.default_rng(9)
    for dtype in TYPES:
        for H, D, n in ((2, 64, 5000), (1, 4, 30000), (3, 37, 3000), (40, 128, 700)):
            c = xtern.KvCache.new(20, 24, H, D, dtype=dtype)
            if dtype == torch.int8:
                for x, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
                    x.copy_(torch.randint(-127, 128, x.shape, dtype=torch.int8))
                    s.copy_(torch.rand(s.shape))
            else:
                c.k.copy_(torch.randn(c.k.shape))
                c.v.copy_(torch.randn(c.v.shape))
            table = torch.from_numpy(rng.permutation(20).astype(np.int32)).cuda().reshape(2, 10)
            seq, slots = (torch.from_numpy(rng.integers(0, m, n).astype(np.int32)).cuda() for m in (2, 240))
            for rd in (torch.float32, torch.bfloat16):
                pg = table[seq.long(), slots.long() // 24].long()
                for got, x, s in zip(xtern.kv_read(c, table, slots, seq=seq, dtype=rd), (c.k, c.v), (c.k_scale, c.v_scale)):
                    w = x[pg, slots.long() % 24].float()
                    w = w if s is None else w * s[pg, :, slots.long() % 24][..., None]
                    assert torch.equal(got, w.to(rd))


def test_no_rows():
    c = xtern.KvCache.new(2, 16, 2, 64, dtype=torch.int8)
    e, t, none = torch.zeros((0, 2, 64), device="cuda"), torch.zeros((1, 2), **I32), torch.zeros(0, **I32)
    assert xtern.kv_append(c, t, none, e, e) is None
    k, v = xtern.kv_read(c, t, none)
    assert k.shape == v.shape == (0, 2, 64)
    assert xtern.paged_attention(c, t, none, torch.zeros((0, 4, 64), device="cuda"), tokens=5).shape == (0, 4, 64)
    out, lse = xtern.paged_attention(c, torch.zeros((2, 0), **I32), torch.ones(2, **I32), torch.ones((2, 4, 64), device="cuda"),
                                     lse=True)
    assert bool((out == 0).all()) and bool((lse == -float("inf")).all())


# --- streams and graphs ----------------------------------------------------

def decode_state(dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = xtern.KvCache.new(200, 16, 2, 64, dtype=dtype)
    table = torch.randperm(200, generator=g, device="cuda").to(torch.int32).reshape(2, 100)
    n = 1500
    k, v = (torch.randn((2 * n, 2, 64), generator=g, device="cuda") for _ in range(2))
    seq = torch.arange(2, device="cuda").repeat_interleave(n).to(torch.int32)
    slots = torch.arange(n, device="cuda").repeat(2).to(torch.int32)
    ones = torch.ones(64, device="cuda")
    xtern.kv_append(c, table, slots, k, v, seq=seq, norm=(None, ones, 1e-6))
    return c, table, ones, g


@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16], ids=str)
def test_graph(dtype):
    """A step of drafts, captured and replayed with other tokens between eager
    steps of the same cache: as without a graph."""
    c, table, ones, g = decode_state(dtype)
    one, _, _, _ = decode_state(dtype)
    T = 3
    seq = torch.arange(2, device="cuda").repeat_interleave(T).to(torch.int32)
    q, k, v = (torch.empty((2 * T, h, 64), device="cuda") for h in (8, 2, 2))
    slots = torch.empty(2 * T, **I32)

    def step(cache):
        lengths = torch.empty(2 * T, **I32)
        out = xtern.kv_append(cache, table, slots, k, v, q=q, seq=seq, lengths=lengths, norm=(ones, ones, 1e-6))
        y, lse = xtern.paged_attention(cache, table, lengths, out, seq=seq, lse=True, tokens=T, window=700, sink=4)
        return (y, lse) + xtern.kv_read(cache, table, slots, seq=seq)

    def fill(i):
        for x in (q, k, v):
            x.normal_(generator=g)
        slots.copy_((torch.arange(2 * T, device="cuda") % T + 1490 + i).to(torch.int32))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step(c)
    for i in range(4):
        fill(i)
        graph.replay()
        want = step(one)
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
        fill(i)  # (an eager step between)
        for a, b in zip(step(c), step(one)):
            assert torch.equal(a, b)


def test_two_graphs_of_one_workspace():
    """Graphs of a stream share its workspace and counters: replayed in turn on it,
    with an eager call between, each gives what its calls give by themselves."""
    c, table, ones, g = decode_state(torch.int8)
    V = 5000
    seq = torch.tensor([0, 0, 0, 1, 1, 1], **I32)
    lengths = torch.tensor([1400, 900, 3, 1500, 0, 1200], **I32)
    q = torch.randn((6, 8, 64), generator=g, device="cuda")
    target, draft = (3 * torch.randn((4, n, V), generator=g, device="cuda") for n in (4, 3))
    drafted = draft.argmax(2).to(torch.int32)
    uniforms = torch.rand((4, 4), generator=g, device="cuda")

    def one():
        return (xtern.paged_attention(c, table, lengths, q, seq=seq, tokens=3),) + \
            xtern.verify_drafts(target, drafted, uniforms, draft=draft)

    def other():
        return (xtern.paged_attention(c, table, lengths, q, seq=seq, tokens=1, window=600, sink=5),) + \
            xtern.verify_drafts(target[:2], drafted[:2], uniforms[:2])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [[x.clone() for x in f()] for f in (one, other)]
        graphs = []
        for f in (one, other):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = f()
            graphs.append((graph, out))
        for i in (0, 1, 1, 0, 1, 0, 0):
            graph, out = graphs[i]
            for x in out:
                x.fill_(77)
            graph.replay()
            eager = (one, other)[1 - i]()
            for a, b in zip(out + eager, want[i] + want[1 - i], strict=True):
                assert torch.equal(a, b)
    torch.cuda.synchronize()


def test_threads():
    """Four host threads at once, on one stream and on their own."""
    c, table, _, g = decode_state(torch.int8)
    seq = torch.tensor([0, 0, 0, 1, 1, 1], **I32)
    lengths = [torch.tensor(n, **I32) for n in ([1400, 900, 3, 1500, 0, 1200], [7, 1, 1300, 64, 1100, 1490])]
    q = torch.randn((6, 8, 64), generator=g, device="cuda")
    target, draft = (3 * torch.randn((4, n, 5000), generator=g, device="cuda") for n in (4, 3))
    drafted = draft.argmax(2).to(torch.int32)
    uniforms = torch.rand((4, 4), generator=g, device="cuda")

    def call(i):
        n = lengths[i % 2]
        return (xtern.paged_attention(c, table, n, q, seq=seq, tokens=3),
                *xtern.kv_read(c, table, n - 1, seq=seq),
                *xtern.verify_drafts(target[i % 2:], drafted[i % 2:], uniforms[i % 2:], draft=draft[i % 2:]))

    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    for own in (False, True):
        got, streams = [[] for _ in range(4)], [torch.cuda.Stream() for _ in range(4)]

        def work(i):
            with torch.cuda.stream(streams[i if own else 0]):
                for _ in range(20):
                    got[i].append(call(i))

        threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        for i in range(4):
            assert len(got[i]) == 20
            for x in got[i]:
                for a, b in zip(x, want[i % 2], strict=True):
                    assert torch.equal(a, b)


def test_most_rows():
    """As many rows as a call takes: 2^21, two of which are no padding."""
    R, D = 1 << 21, 4
    c = xtern.KvCache.new(2, 8, 1, D, dtype=torch.int8)
    table = torch.tensor([[1]], **I32)
    slots = torch.full((R,), -1, **I32)
    slots[0], slots[R - 1] = 3, 5
    seq = torch.zeros(R, **I32)
    k = torch.zeros((R, 1, D), device="cuda")
    k[0, 0], k[R - 1, 0] = torch.tensor([127.0, 1, 2, 3], device="cuda"), torch.tensor([-127.0, 4, 5, 6], device="cuda")
    lengths = torch.empty(R, **I32)
    xtern.kv_append(c, table, slots, k, 2 * k, seq=seq, lengths=lengths)
    assert int(lengths[0]) == 4 and int(lengths[R - 1]) == 6 and int(lengths.sum()) == 10
    a, b = xtern.kv_read(c, table, slots, seq=seq)
    assert torch.equal(a, k) and torch.equal(b, 2 * k)
    # (scores beyond f32's exponents apart: one position has all of it)
    q = torch.zeros((R, 1, D), device="cuda")
    q[R - 1, 0, 0] = -10.0
    out = xtern.paged_attention(c, table, lengths, q, seq=seq)
    assert torch.equal(out[R - 1], 2 * k[R - 1]) and torch.equal(out[0], k[0] / 2)
    assert float(out[1:R - 1].abs().max()) == 0.0


def test_streams():
    """Two streams at once, each with its own workspace; a stream argument."""
    c, table, ones, g = decode_state(torch.int8)
    q = torch.randn((6, 8, 64), generator=g, device="cuda")
    lengths = torch.tensor([1400, 900, 3, 1500, 1000, 1200], **I32)
    seq = torch.tensor([0, 0, 0, 1, 1, 1], **I32)
    want = xtern.paged_attention(c, table, lengths, q, seq=seq, tokens=3)
    read = xtern.kv_read(c, table, lengths - 1, seq=seq)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for s in streams:
            got.append(xtern.paged_attention(c, table, lengths, q, seq=seq, tokens=3, stream=s))
            got.append(xtern.kv_read(c, table, lengths - 1, seq=seq, stream=s))
    torch.cuda.synchronize()
    for x in got:
        for a, b in zip(x if isinstance(x, tuple) else (x,), read if isinstance(x, tuple) else (want,)):
            assert torch.equal(a, b)


# --- the layer -------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layer(dtype):
    """CausalSelfAttention with norms of the heads, a window and drafts: its
    parts one after the other."""
    rng = np.random.default_rng(12)
    hidden, hq, H, D, T, S = 256, 8, 2, 64, 3, 2
    lin = lambda o, i: xtern.TernaryLinear.new(i, o, rng.integers(-1, 2, (o, i)).astype(np.float32),  # noqa: E731
                                               xtern.TernaryPackType.Pack4, 0.05)
    ql, kl, vl, ol = lin(hq * D, hidden), lin(H * D, hidden), lin(H * D, hidden), lin(hidden, hq * D)
    norms = [xtern.FastRmsNorm(torch.from_numpy((1 + 0.1 * rng.standard_normal(D)).astype(np.float32)).cuda(), 1e-5)
             for _ in range(2)]
    attn = xtern.CausalSelfAttention(ql, kl, vl, ol, D, q_norm=norms[0], k_norm=norms[1], window=20, sink=2)
    ang = np.arange(100)[:, None] * 10000.0 ** (-np.arange(D // 2) / (D // 2))
    rope = dev(np.cos(ang).astype(np.float32)), dev(np.sin(ang).astype(np.float32))
    table = torch.arange(14, **I32).reshape(2, 7)
    a, b = (xtern.KvCache.new(14, 8, H, D, dtype=dtype) for _ in range(2))
    seq = torch.arange(S, device="cuda").repeat_interleave(T).to(torch.int32)
    for step in range(14):
        x = dev(rng.standard_normal((S * T, hidden)).astype(np.float32))
        slots = (torch.arange(S * T, device="cuda") % T + step * T).to(torch.int32)
        if step % 4 == 3:
            slots[T - 1] = -1  # (one draft fewer)
        y = attn.forward(x, a, table, slots, seq=seq, rope=rope, tokens=T)
        q, k, v = xtern.linear_multi_f32([l.weights for l in (ql, kl, vl)], x)
        lengths = torch.empty(S * T, **I32)
        q = xtern.kv_append(b, table, slots, k, v, q=q, seq=seq, rope=rope, lengths=lengths,
                            norm=(norms[0].weight, norms[1].weight, 1e-5))
        z, lse = xtern.paged_attention(b, table, lengths, q, seq=seq, lse=True, window=20, sink=2, tokens=T)
        assert torch.equal(y, xtern.linear_f32(ol.weights, z))
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
        scales = (b.k_scale.cpu(), b.v_scale.cpu()) if dtype == torch.int8 else (None, None)
        want = ref.attention(b.k.cpu(), b.v.cpu(), table.cpu().numpy(), 8, q.cpu().view(S * T, hq, D), lengths.cpu().numpy(),
                             seq.tolist(), D ** -0.5, *scales, 20, 2, T)
        close(z.view(S * T, hq, D), want[0], want[3], "attention")
        close(lse, want[1], want[4], "lse")
