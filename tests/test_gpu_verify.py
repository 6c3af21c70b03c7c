"""Verification of drafted tokens against its plain 64-bit form: every type,
vocabularies of any size, counts, temperatures, masks and what is no
probability; and a decode loop with drafts over an 8-bit cache."""
import numpy as np
import pytest
import torch

import cache8_ref as ref
import xtern
from test_gpu_cache import log

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
INF, NAN = float("inf"), float("nan")


def inputs(rng, S, T, V, dtype, draft, masked=0.0, near=1.0, spread=2.5):
    x = rng.standard_normal((S, T + 1, V)).astype(np.float32) * spread
    hot = rng.integers(0, V, (S, T + 1))
    np.put_along_axis(x, hot[..., None], 6.0, -1)
    y = 0.9 * x[:, :T] + near * rng.standard_normal((S, T, V)).astype(np.float32)
    if masked:
        gone = rng.random((S, 1, V)) < masked
        gone[:, 0, 0] = False
        x[np.broadcast_to(gone, x.shape)] = -INF
        y[np.broadcast_to(gone, y.shape)] = -INF
    target, source = torch.from_numpy(x).to(dtype), torch.from_numpy(y).to(dtype)
    drafted = np.zeros((S, T), np.int32)
    for b in range(S):
        for t in range(T):
            p = ref.chances(source[b, t], 1.0)
            drafted[b, t] = rng.choice(V, p=p)
    uniforms = torch.from_numpy(rng.random((S, T + 1)).astype(np.float32))
    return target, source if draft else None, torch.from_numpy(drafted), uniforms


def check(target, draft, drafted, uniforms, counts=None, temperature=1.0, wide=False):
    d = lambda x: None if x is None else x.cuda()  # noqa: E731
    want = ref.verify(target, drafted, uniforms, draft, counts, temperature)
    tt = temperature if np.isscalar(temperature) else torch.from_numpy(np.asarray(temperature, np.float32)).cuda()
    gt, gd = d(target), d(draft)
    if wide:  # rows of a wider tensor, sequences apart
        S, n, V = target.shape
        gt = torch.full((S + 1, n + 2, V + 3), NAN, dtype=target.dtype, device="cuda")[1:, 1:n + 1, 1:V + 1]
        gt.copy_(target)
        if draft is not None:
            gd = torch.full((n, S, V + 1), NAN, dtype=target.dtype, device="cuda")[:n - 1, :, :V].transpose(0, 1)
            gd.copy_(draft)
    got = xtern.verify_drafts(gt, d(drafted), d(uniforms), draft=gd,
                              counts=None if counts is None else torch.tensor(counts, **I32), temperature=tt)
    torch.cuda.synchronize()
    accepted, tokens, lp = (x.cpu().numpy() for x in got)
    assert np.array_equal(accepted, want[0]), (accepted, want[0])
    assert np.array_equal(tokens, want[1]), (tokens, want[1])
    # (the logit's difference is exact in 64 bits up to 2^-52 of both; rounded once)
    tol = np.abs(want[2]) * 2.0 ** -24 * (1 + 1e-6) + 1e-12
    assert bool((np.abs(lp - want[2]) <= tol).all()), np.abs(lp - want[2]).max()
    return got


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 1023, 1024, 1025, 4097, 32003])
@pytest.mark.parametrize("draft", [False, True], ids=["certain", "draft"])
def test_vocabularies(dtype, V, draft):
    log(f"verify {dtype} {V} {draft}")
    rng = np.random.default_rng(V)
    for T in (0, 1, 4):
        check(*inputs(rng, 5, T, V, dtype, draft))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("masked", [0.5, 0.99])
def test_masks(dtype, masked):
    rng = np.random.default_rng(2)
    for draft in (False, True):
        for V in (300, 5000):
            check(*inputs(rng, 9, 3, V, dtype, draft, masked=masked))


@pytest.mark.parametrize("T", [0, 1, 2, 8, 33, 63, 64])
def test_drafts(T):
    """Every number of drafts, many of them accepted."""
    log(f"verify T {T}")
    rng = np.random.default_rng(T)
    counts = rng.integers(-1, T + 3, 7).tolist()
    for draft in (False, True):
        x = inputs(rng, 7, T, 257, torch.float32, draft, near=0.05)
        check(*x)
        check(*x, counts=counts)
        check(*x, wide=True)


@pytest.mark.parametrize("S", [1, 3, 64, 300, 2000])
def test_sequences(S):
    log(f"verify S {S}")
    rng = np.random.default_rng(S)
    x = inputs(rng, S, 2, 211 if S > 300 else 2111, torch.bfloat16, True)
    check(*x, wide=S == 3)


def test_long_rows():
    """Rows in many slices and tiles."""
    rng = np.random.default_rng(5)
    for dtype in DTYPES:
        for S, T in ((1, 0), (1, 4), (6, 2)):
            log(f"verify {dtype} {S} {T} x 200003")
            check(*inputs(rng, S, T, 200003, dtype, True, near=0.3))


def test_temperatures():
    rng = np.random.default_rng(6)
    for dtype in DTYPES:
        for draft in (False, True):
            x = inputs(rng, 12, 3, 700, dtype, draft, near=0.3)
            for temp in (0, 0.0, 0.01, 0.7, 1.0, 3.0, 1e6):
                check(*x, temperature=temp)
            check(*x, temperature=[0.0, 0.5, 1.0, 2.0, NAN, -1.0, INF, 0.0, 1e-30, 1e30, 1.0, 0.3])


def test_equal_logits_without_temperature():
    """The lowest of equals, across lanes, tiles and slices."""
    for at in ([3, 5], [5000, 70], [1023, 1024], [9999, 0], [4096, 8192, 100]):
        x = torch.zeros((2, 2, 10000))
        x[:, :, at] = 2.0
        drafted = torch.tensor([[min(at)], [max(at)]], dtype=torch.int32)
        got = check(x, None, drafted, torch.full((2, 2), 0.5), temperature=0.0)
        assert got[1].tolist() == [[min(at), min(at)], [min(at), -1]]


def test_uniforms_at_the_ends():
    rng = np.random.default_rng(7)
    top = float(np.nextafter(np.float32(1), np.float32(0)))
    for u in (0.0, top, 1.0, 2.0, NAN):
        for draft in (False, True):
            t, d, x, _ = inputs(rng, 6, 2, 3000, torch.float32, draft, masked=0.3)
            check(t, d, x, torch.full((6, 3), u))
    # all of p on the drafted token, refused all the same: drawn from p
    t = torch.full((1, 2, 50), -INF)
    t[:, :, 7] = 1.0
    check(t, None, torch.tensor([[7]], dtype=torch.int32), torch.tensor([[1.0, 0.3]]))
    check(t, t[:, :1], torch.tensor([[7]], dtype=torch.int32), torch.tensor([[1.0, 0.3]]))


def test_impossible_drafts():
    """Drafts that the target masks, that the draft model masks, ids outside
    the vocabulary."""
    rng = np.random.default_rng(8)
    t, d, x, u = inputs(rng, 6, 3, 500, torch.float32, True, near=0.1)
    for b in range(6):
        if b < 2:
            t[b, 1, x[b, 1]] = -INF
        elif b < 4:
            d[b, 1, x[b, 1]] = -INF
    x[4, 1], x[5, 0] = -3, 500
    u[:, 0] = 0.0
    check(t, d, x, u)
    check(t, None, x, u)


def test_rows_that_are_no_probabilities():
    """NaN, +inf and nothing but -inf, in rows that count and in rows that
    do not."""
    rng = np.random.default_rng(9)
    for bad in (NAN, INF, None):
        for place in range(3):
            for which in range(2):
                for temp in (1.0, 0.0):
                    t, d, x, u = inputs(rng, 3, 2, 3000, torch.float32, True, near=0.05)
                    row = (t if which == 0 or place == 2 else d)[:, place]
                    if bad is None:
                        row[1] = -INF
                    else:
                        row[1, 2345] = bad
                    u[:, 0] = 0.0
                    check(t, d, x, u, temperature=temp)
                    check(t, d, x, u, temperature=temp, counts=[2, 0, 1])


def test_large_logits():
    """Logits of 1e38, differences beyond exp's range."""
    x = torch.full((2, 2, 3000), -3e38)
    x[0, :, 17] = 3e38
    x[1, :, 18] = x[1, :, 2900] = 1e30
    check(x, x[:, :1] * 0.5, torch.tensor([[17], [18]], dtype=torch.int32), torch.tensor([[0.3, 0.6], [0.3, 0.6]]))
    check(x, None, torch.tensor([[16], [2900]], dtype=torch.int32), torch.tensor([[0.3, 0.4], [0.3, 0.6]]))


def test_shared_row():
    """One row of logits shown to several sequences, by a stride of 0."""
    rng = np.random.default_rng(10)
    row = torch.from_numpy(rng.standard_normal((1, 1, 900)).astype(np.float32)).expand(40, 1, 900)
    u = torch.from_numpy(rng.random((40, 1)).astype(np.float32))
    want = ref.verify(row, torch.zeros((40, 0), dtype=torch.int32), u)
    got = xtern.verify_drafts(row[:1].cuda().expand(40, 1, 900), torch.zeros((40, 0), **I32), u.cuda())
    assert np.array_equal(got[1].cpu().numpy(), want[1])


def test_no_sequences():
    got = xtern.verify_drafts(torch.zeros((0, 3, 10), device="cuda"), torch.zeros((0, 2), **I32), torch.zeros((0, 3), device="cuda"))
    assert [tuple(x.shape) for x in got] == [(0,), (0, 3), (0, 3)]


def test_most_sequences():
    """2^21 of them, one row each: the most likely token, and one that is certain."""
    S = 1 << 21
    target = torch.zeros((S, 1, 3), device="cuda")
    target[:, 0, 1] = 200.0
    target[S - 1, 0, 2] = 400.0
    uniforms = torch.full((S, 1), 0.5, device="cuda")
    drafted = torch.empty((S, 0), dtype=torch.int32, device="cuda")
    for temperature in (0.0, 1.0):
        accepted, tokens, logprobs = xtern.verify_drafts(target, drafted, uniforms, temperature=temperature)
        assert int(accepted.abs().max()) == 0 and int(tokens[S - 1]) == 2
        assert bool((tokens[:S - 1] == 1).all()) and float(logprobs.abs().max()) == 0.0


def test_graph_and_streams():
    """Replayed several times with other inputs, eager calls between; two
    streams at once."""
    rng = np.random.default_rng(11)
    cases = [inputs(rng, 4, 3, 20000, torch.float32, True, near=0.2) for _ in range(3)]
    state = [torch.empty_like(x, device="cuda") for x in cases[0]]
    call = lambda s: xtern.verify_drafts(s[0], s[2], s[3], draft=s[1])  # noqa: E731
    side = torch.cuda.Stream()
    for a, b in zip(state, cases[0]):
        a.copy_(b)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = call(state)
    eager = [[x.cuda() for x in c] for c in cases]
    want = [[x.cpu() for x in call(e)] for e in eager]
    for i in (0, 1, 2, 1, 0):
        for a, b in zip(state, eager[i]):
            a.copy_(b)
        graph.replay()
        again = call(eager[(i + 1) % 3])
        torch.cuda.synchronize()
        for a, b in zip(captured, want[i]):
            assert torch.equal(a.cpu(), b)
        for a, b in zip(again, want[(i + 1) % 3]):
            assert torch.equal(a.cpu(), b)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for k, s in enumerate(streams):
            e = eager[k]
            got.append((k, xtern.verify_drafts(e[0], e[2], e[3], draft=e[1], stream=s)))
    torch.cuda.synchronize()
    for k, g in got:
        for a, b in zip(g, want[k]):
            assert torch.equal(a.cpu(), b)


def test_decode_loop_with_drafts():
    """Drafts through the layer over an 8-bit cache, verified, the cache taken
    back to the last accepted token: the greedy text is the one that decoding
    token by token over the same kind of cache gives."""
    rng = np.random.default_rng(13)
    hidden, hq, H, D, V, T, S = 256, 4, 2, 64, 320, 3, 3
    lin = lambda o, i: xtern.TernaryLinear.new(i, o, rng.integers(-1, 2, (o, i)).astype(np.float32),  # noqa: E731
                                               xtern.TernaryPackType.Pack4, 0.05)
    ones = xtern.FastRmsNorm(torch.ones(D, device="cuda"), 1e-6)
    attn = xtern.CausalSelfAttention(lin(hq * D, hidden), lin(H * D, hidden), lin(H * D, hidden), lin(hidden, hq * D), D,
                                     q_norm=ones, k_norm=ones, window=24, sink=2)
    head = lin(V, hidden)
    embed = torch.from_numpy(rng.standard_normal((V, hidden)).astype(np.float32)).cuda()
    ang = np.arange(200)[:, None] * 10000.0 ** (-np.arange(D // 2) / (D // 2))
    rope = tuple(torch.from_numpy(f(ang).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    table = torch.arange(S * 8, **I32).reshape(S, 8)

    def logits(cache, ids, at, seq, tokens):
        x = embed[ids.long()]
        return head.forward(x + attn.forward(x, cache, table, at, seq=seq, rope=rope, tokens=tokens))

    # token by token
    steps = 40
    one = xtern.KvCache.new(S * 8, 8, H, D, dtype=torch.int8)
    text = [torch.tensor([1, 2, 3], **I32)]
    seq1 = torch.arange(S, **I32)
    for i in range(steps):
        lg = logits(one, text[-1], torch.full((S,), i, **I32), seq1, 1)
        _, tok, _ = xtern.verify_drafts(lg.view(S, 1, V), torch.zeros((S, 0), **I32), torch.full((S, 1), 0.5, device="cuda"),
                                        temperature=0.0)
        text.append(tok[:, 0].contiguous())
    text = torch.stack(text, 1).cpu().numpy()
    # with drafts, some of them wrong
    c = xtern.KvCache.new(S * 8, 8, H, D, dtype=torch.int8)
    done = [[int(text[b, 0])] for b in range(S)]
    seq = torch.arange(S, device="cuda").repeat_interleave(T + 1).to(torch.int32)
    calls = 0
    while max(len(d) for d in done) + T <= steps:
        drafts = np.array([[text[b, len(done[b]) + t] for t in range(T)] for b in range(S)], np.int32)
        drafts[calls % S, calls % T] = (drafts[calls % S, calls % T] + 1) % V
        n = [len(d) for d in done]
        ids = np.concatenate([np.array([[d[-1]] for d in done], np.int32), drafts], 1)
        at = np.array([[n[b] - 1 + t for t in range(T + 1)] for b in range(S)], np.int32)
        lg = logits(c, torch.from_numpy(ids.reshape(-1)).cuda(), torch.from_numpy(at.reshape(-1)).cuda(), seq, T + 1)
        acc, tok, _ = xtern.verify_drafts(lg.view(S, T + 1, V), torch.from_numpy(drafts).cuda(),
                                          torch.full((S, T + 1), 0.5, device="cuda"), temperature=0.0)
        acc, tok = acc.tolist(), tok.tolist()
        for b in range(S):
            assert acc[b] == (calls % T if b == calls % S else T)
            done[b] += tok[b][:acc[b] + 1]
        calls += 1
    for b in range(S):
        m = min(len(done[b]), steps + 1)
        assert done[b][:m] == text[b, :m].tolist()
