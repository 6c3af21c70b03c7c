"""The cache and probability calls as a serving loop makes them: a prompt and
decoded tokens through CausalSelfAttention, eviction, more tokens, the head's
logits; on other streams, from several threads, captured into graphs and
replayed, with outputs of earlier calls still in use."""
import threading

import numpy as np
import pytest
import torch

import cache_ref as ref
import xtern

pytestmark = pytest.mark.gpu

HID, HQ, H, D, PAGE = 256, 8, 2, 64, 16
I32 = dict(dtype=torch.int32, device="cuda")


def linear(rng, i, o, pack=xtern.TernaryPackType.Pack4):
    return xtern.TernaryLinear.new(i, o, rng.integers(-1, 2, (o, i)).astype(np.float32), pack, 0.05)


def rope(n):
    ang = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    return torch.from_numpy(np.cos(ang).astype(np.float32)).cuda(), torch.from_numpy(np.sin(ang).astype(np.float32)).cuda()


def layer(rng, norm=True):
    n = xtern.FastRmsNorm(torch.from_numpy(rng.random(HQ * D).astype(np.float32)).cuda(), 1e-5) if norm else None
    return xtern.CausalSelfAttention(linear(rng, HID, HQ * D), linear(rng, HID, H * D), linear(rng, HID, H * D),
                                     linear(rng, HQ * D, HID), D, attn_sub_norm=n)


def tensor(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_serving_loop(dtype):
    """Two sequences: prompts of 50 and 21 tokens in one call, 30 decoded
    tokens, an eviction to 40 positions, 10 more tokens.  A copy of the cache
    on the host is appended to and evicted from by the plain forms; every
    attention is held to the plain form over it."""
    rng = np.random.default_rng(0)
    attn, (cos, sin) = layer(rng), rope(256)
    head = xtern.Int8Linear.new(rng.standard_normal((1000, HID)).astype(np.float32), 1000, HID)
    cache = xtern.KvCache.new(24, PAGE, H, D, dtype=dtype, score=True)
    table = torch.from_numpy(rng.permutation(24)[:16].reshape(2, 8).astype(np.int32)).cuda()
    htab = table.cpu().numpy()
    lens, pos = [0, 0], [0, 0]

    def step(seq_rows):
        """One call for the given tokens per sequence."""
        seq = [b for b, n in enumerate(seq_rows) for _ in range(n)]
        slots = [lens[b] + i for b, n in enumerate(seq_rows) for i in range(n)]
        at = [pos[b] + i for b, n in enumerate(seq_rows) for i in range(n)]
        x = tensor(rng, len(seq), HID)
        dseq, dslots, dpos = (torch.tensor(v, **I32) for v in (seq, slots, at))
        before = cache.score.clone()
        y = attn.forward(x, cache, table, dslots, seq=dseq, positions=dpos, rope=(cos, sin), accumulate=True)
        # the same, call by call
        q, k, v = xtern.linear_multi_f32([l.weights for l in (attn.q_proj, attn.k_proj, attn.v_proj)], x)
        kh, vh = cache.k.cpu(), cache.v.cpu()  # (appended by the layer)
        for r, (b, s, p) in enumerate(zip(seq, slots, at)):
            pg, sl = htab[b][s // PAGE], s % PAGE
            assert torch.equal(vh[pg, sl], v[r].cpu().reshape(H, D).to(dtype))
            kr = k[r].cpu().double().reshape(H, D)
            c, sn = cos[p].cpu().double(), sin[p].cpu().double()
            a, e = kr[:, :D // 2], kr[:, D // 2:]
            want = torch.cat([a * c - e * sn, e * c + a * sn], 1)
            mag = torch.cat([(a * c).abs() + (e * sn).abs(), (e * c).abs() + (a * sn).abs()], 1)
            ref.close(kh[pg, sl], want, 3 * ref.EPS * mag * 1.01 + ref.HALF[dtype] * want.abs(), "k")
            before[int(pg), :, sl] = 0.0
        rot = torch.empty_like(q)
        scratch = xtern.KvCache.new(24, PAGE, H, D, dtype=dtype)
        xtern.kv_append(scratch, table, dslots, k, v, q=q, seq=dseq, positions=dpos, rope=(cos, sin), q_out=rot)
        o = xtern.paged_attention(cache, table, dslots + 1, rot, seq=dseq)
        assert torch.equal(y, xtern.linear_f32(attn.o_proj.weights, attn.attn_sub_norm.forward(o)))
        w = ref.attention(kh, vh, htab, PAGE, rot.cpu().reshape(-1, HQ, D), [s + 1 for s in slots], seq, D ** -0.5,
                          before.cpu())
        ref.close(o.reshape(-1, HQ, D), w[0], w[3], "attention")
        # (rows of one sequence add to a score one after the other)
        ref.close(cache.score, w[2], w[5] + len(seq) * ref.EPS * w[2].abs(), "score")
        for b, n in enumerate(seq_rows):
            lens[b] += n
            pos[b] += n
        return y

    step([50, 21])
    for i in range(30):
        y = step([1, 1] if i % 3 else [1, 0])
    k, v, score = cache.k.cpu().clone(), cache.v.cpu().clone(), cache.score.cpu().clone()
    new, kept = xtern.kv_evict(cache, table, torch.tensor(lens, **I32), 40, sink=2, recent=8)
    wnew, wkept = ref.evict(k, v, score, htab, PAGE, lens, 40, 2, 8)
    assert new.tolist() == wnew.tolist() and np.array_equal(kept.cpu().numpy(), wkept)
    assert torch.equal(cache.k.cpu(), k) and torch.equal(cache.v.cpu(), v) and torch.equal(cache.score.cpu(), score)
    lens[:] = new.tolist()
    for i in range(10):
        y = step([1, 1])
    logits = head.forward(y)
    lp, ent, ids, tlp = xtern.token_logprobs(logits, torch.tensor([3, 999], **I32), top=5)
    w = ref.logprobs(logits.cpu(), torch.tensor([[3], [999]]), 5)
    ref.close(lp[:, None], w[0], w[4], "lp")
    ref.close(ent, w[1], w[5], "entropy")
    assert torch.equal(ids.cpu().long(), w[2])
    ref.close(tlp, w[3], w[6], "alternatives")


def state(seed, n=700, R=3, dtype=torch.bfloat16, score=True):
    """A cache of R sequences of up to n positions and the inputs of a step."""
    rng = np.random.default_rng(seed)
    per = (n + PAGE) // PAGE + 1
    cache = xtern.KvCache.new(R * per, PAGE, H, D, dtype=dtype, score=score)
    cache.k.copy_(tensor(rng, *cache.k.shape))
    cache.v.copy_(tensor(rng, *cache.v.shape))
    table = torch.from_numpy(rng.permutation(R * per).reshape(R, per).astype(np.int32)).cuda()
    lens = torch.tensor([n - 37 * i for i in range(R)], **I32)
    return dict(cache=cache, table=table, slots=lens, lens=lens + 1, q=tensor(rng, R, HQ, D), k=tensor(rng, R, H, D),
                v=tensor(rng, R, H, D), logits=tensor(rng, R, 20000), tokens=torch.tensor([[5], [6], [7]][:R], **I32))


def step(s, rp, stream=None):
    """Append, attend with scores, probabilities: (out, lse, lp, entropy, ids, top)."""
    q = xtern.kv_append(s["cache"], s["table"], s["slots"], s["k"], s["v"], q=s["q"], rope=rp, stream=stream)
    o, lse = xtern.paged_attention(s["cache"], s["table"], s["lens"], q, lse=True, accumulate=True, stream=stream)
    return (o, lse) + xtern.token_logprobs(s["logits"], s["tokens"], top=8, stream=stream)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_calls_repeat_bit_for_bit():
    rp = rope(1024)
    s = state(1)
    first = [x.clone() for x in step(s, rp)]
    for _ in range(5):
        assert same(first, step(s, rp))


def test_graph_of_a_step():
    """Captured once, replayed with eager calls of other shapes and a growing
    workspace between; every replay equals the eager result, scores add up."""
    rp, s, other = rope(4096), state(2), state(3, n=3000)
    st = torch.cuda.Stream()
    want = None
    with torch.cuda.stream(st):
        step(s, rp)  # (workspaces of this stream)
        s["cache"].score.zero_()
        want = [x.clone() for x in step(s, rp)]
        one = s["cache"].score.clone()
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = step(s, rp)
        s["cache"].score.zero_()
        for i in range(6):
            for x in out:
                x.fill_(7)
            g.replay()
            st.synchronize()
            assert same(out, want), i
            # (the appended position's score starts at 0 in every replay)
            there = one > 0
            again = s["cache"].score.clone()
            step(other, rp)
            torch.cuda.synchronize()
            assert bool((again[there] >= one[there]).all()) and bool(torch.isfinite(again).all())
        # new inputs in place
        fresh = state(4)
        for k in ("q", "k", "v", "logits"):
            s[k].copy_(fresh[k])
        eager = [x.clone() for x in step(s, rp)]
        for _ in range(3):
            g.replay()
            st.synchronize()
            assert same(out, eager)


def test_graph_of_an_eviction():
    s = state(5, n=600)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    s["cache"].score.uniform_(generator=gen)
    k0, v0, s0 = s["cache"].k.clone(), s["cache"].v.clone(), s["cache"].score.clone()

    def reset():
        s["cache"].k.copy_(k0)
        s["cache"].v.copy_(v0)
        s["cache"].score.copy_(s0)

    def call():
        return xtern.kv_evict(s["cache"], s["table"], s["slots"], 200, sink=4, recent=20)

    want = [x.clone() for x in call()] + [x.clone() for x in (s["cache"].k, s["cache"].v, s["cache"].score)]
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
            assert same(list(out) + [s["cache"].k, s["cache"].v, s["cache"].score], want)


def test_capture_without_a_workspace_is_refused():
    rp, s = rope(1024), state(6)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        with torch.cuda.graph(g, stream=st):
            with pytest.raises(xtern.XternError, match="capture"):
                xtern.paged_attention(s["cache"], s["table"], s["lens"], s["q"])
    want = xtern.paged_attention(s["cache"], s["table"], s["lens"], s["q"])
    with torch.cuda.stream(st):
        assert torch.equal(want, xtern.paged_attention(s["cache"], s["table"], s["lens"], s["q"]))
    st.synchronize()


def test_stream_argument():
    """Results belong to the given stream; inputs may be dropped at once."""
    rp, st = rope(1024), torch.cuda.Stream()
    want = [x.clone() for x in step(state(7), rp)]
    for _ in range(4):
        s = state(7)
        st.wait_stream(torch.cuda.current_stream())
        got = step(s, rp, stream=st)
        del s
        junk = [torch.full((3, HQ, D), 9.0, device="cuda") for _ in range(20)]  # (freed memory comes back)
        st.synchronize()
        assert same(got, want)
        del junk


def test_threads_on_one_stream():
    """Workspaces and counters are a thread's own."""
    rp, states = rope(4096), [state(10 + i, n=300 + 500 * i) for i in range(4)]
    want = [[x.clone() for x in step(s, rp)] for s in states]
    torch.cuda.synchronize()
    st, errors, go = torch.cuda.Stream(), [], threading.Barrier(4)
    st.wait_stream(torch.cuda.current_stream())
    got = [[] for _ in states]

    def body(i):
        try:
            go.wait()
            for _ in range(10):
                got[i].append(step(states[i], rp, stream=st))
        except Exception as e:  # reported below
            errors.append(e)

    threads = [threading.Thread(target=body, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    st.synchronize()
    assert not errors, errors
    for w, g in zip(want, got):
        assert len(g) == 10 and all(same(w, x) for x in g)


def test_far_positions_of_a_large_cache():
    """Element offsets past 2^31 and byte offsets past 2^32: the same pages at
    the far end of a 6 GiB pool give the same bits."""
    P = (3 << 30) // (PAGE * 2 * 128)  # elements: 3 * 2^30 in each of k and v
    big = xtern.KvCache.new(P, PAGE, 2, 128, dtype=torch.bfloat16, score=True)
    small = xtern.KvCache.new(8, PAGE, 2, 128, dtype=torch.bfloat16, score=True)
    rng = np.random.default_rng(20)
    near = torch.arange(8, **I32).reshape(1, 8)
    far = near + (P - 8)
    n = torch.tensor([100], **I32)
    out = []
    for cache, table in ((small, near), (big, far)):
        r = np.random.default_rng(21)
        for p in range(0, 120, 40):
            m = 40
            xtern.kv_append(cache, table, torch.arange(p, p + m, **I32), tensor(r, m, 2, 128), tensor(r, m, 2, 128),
                            seq=torch.zeros(m, **I32))
        o, l = xtern.paged_attention(cache, table, n, tensor(r, 1, 8, 128), lse=True, accumulate=True)
        kept = xtern.kv_evict(cache, table, n, 50, sink=2, recent=3)
        pages = table[0].long()
        out.append([o, l, *kept, cache.k[pages], cache.v[pages], cache.score[pages]])
    assert same(*out)
    assert not bool(big.k[:8].any()) and not bool(big.score[:8].any())


def test_python_refusals():
    """What the Python calls refuse beyond the C ABI's checks."""
    s = state(30)
    c, t, n, q = s["cache"], s["table"], s["lens"], s["q"]
    E = xtern.XternError
    att = xtern.paged_attention
    bad = [lambda: att(c, t.long(), n, q), lambda: att(c, t[0], n, q), lambda: att(c, t.t(), n, q),
           lambda: att(c, t, n.long(), q), lambda: att(c, t, n[:2], q), lambda: att(c, t, n.cpu(), q),
           lambda: att(c, t, n, q.half()), lambda: att(c, t, n, q[..., :63]), lambda: att(c, t, n, q.transpose(0, 1)),
           lambda: att(c, t, n, q[..., ::2]), lambda: att(c, t, n, q[0]), lambda: att(c, t[:2], n, q),
           lambda: att(c, t, n, q, seq=n[:1]), lambda: att(c, t, n, q, out=q[:2]), lambda: att(c, t, n, q, out=q.half()),
           lambda: att(c, t, n, q.cpu()), lambda: att(c, t, n, q.numpy) if False else att(c, t, n, None),
           lambda: att(c, t, n, q, scale=float("nan")),
           lambda: att(xtern.KvCache(c.k, c.v), t, n, q, accumulate=True),
           lambda: xtern.KvCache(c.k, c.v[:3]), lambda: xtern.KvCache(c.k, c.v.float()),
           lambda: xtern.KvCache(c.k, c.v.contiguous()), lambda: xtern.KvCache(c.k[0], c.v[0]),
           lambda: xtern.KvCache(c.k.transpose(2, 3), c.v.transpose(2, 3)), lambda: xtern.KvCache(c.k.double(), c.v),
           lambda: xtern.KvCache(c.k, c.v, c.score.transpose(1, 2)), lambda: xtern.KvCache(c.k, c.v, c.score.cpu()),
           lambda: xtern.KvCache(c.k.expand(c.k.shape) * 1, c.v, c.score[:1]),
           lambda: xtern.kv_append(c, t, s["slots"], s["k"], s["v"][:2]),
           lambda: xtern.kv_append(c, t, s["slots"], s["k"][:, :1], s["v"]),
           lambda: xtern.kv_append(c, t, s["slots"], s["k"], s["v"], q_out=q),
           lambda: xtern.kv_append(c, t, s["slots"], s["k"], s["v"], q=q, q_out=q[:, :4]),
           lambda: xtern.kv_append(c, t, s["slots"], s["k"], s["v"], rope=(q[0], q[0][:1])),
           lambda: xtern.kv_append(c, t, s["slots"], s["k"], s["v"], rope=(rope(4)[0][:, :0],) * 2),
           lambda: xtern.kv_evict(c, t, n[:1], 5), lambda: xtern.kv_evict(c, t, n, 0),
           lambda: xtern.kv_evict(c, t, n, 5, sink=3, recent=3), lambda: xtern.kv_evict(xtern.KvCache(c.k, c.v), t, n, 5),
           lambda: xtern.token_logprobs(s["logits"].t()), lambda: xtern.token_logprobs(s["logits"][0]),
           lambda: xtern.token_logprobs(s["logits"], s["tokens"].long()),
           lambda: xtern.token_logprobs(s["logits"], s["tokens"][:2]), lambda: xtern.token_logprobs(s["logits"], top=65),
           lambda: xtern.token_logprobs(s["logits"][:, :3], top=4), lambda: xtern.token_logprobs(s["logits"].int())]
    k0, s0 = c.k.clone(), c.score.clone()
    for i, f in enumerate(bad):
        with pytest.raises(E):
            f()
            print("call", i, "was not refused")
    assert torch.equal(c.k, k0) and torch.equal(c.score, s0)
