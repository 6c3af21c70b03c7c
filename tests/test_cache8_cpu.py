"""What the calls of the 8-bit cache, of windows and of verification refuse, on
the CPU: every check comes before the first HIP call, so no GPU is needed.  And
the plain forms of the GPU tests against hand-worked values and planted
mistakes."""
import ctypes

import numpy as np
import pytest
import torch

import cache8_ref as ref
import xtern
from test_cache_cpu import BUF, CACHE_FAULTS, P, TABLE_FAULTS, FakeLinear, cache, ref_, rope, table  # noqa: F401
from xtern.cache import _HeadNorm, _KvScales

L = xtern.lib()


def codes(**kw):
    return cache(**{**dict(dtype=3, score=None), **kw})


def scales(**kw):
    return _KvScales(**{**dict(k=P, v=P), **kw})


def norm(**kw):
    return _HeadNorm(**{**dict(q=P, k=P, eps=1e-6), **kw})


def store(c=None, s="own", t=None, r=None, nm=None, seq=P, slots=P, pos=P, q=P, ldq=256, hq=4, qo=P, ldqo=256, k=P,
          ldk=128, v=P, ldv=128, R=2, lengths=None):
    return L.xt_kv_store(ref_(c or codes()), ref_(scales() if s == "own" else s), ref_(t or table()), seq, slots, pos,
                         ref_(r or rope()), ref_(nm), q, ldq, hq, qo, ldqo, k, ldk, v, ldv, R, lengths, None)


def read(c=None, s="own", t=None, seq=P, slots=P, R=2, out=0, k=P, ldk=128, v=P, ldv=128):
    return L.xt_kv_read(ref_(c or codes()), ref_(scales() if s == "own" else s), ref_(t or table()), seq, slots, R, out, k,
                        ldk, v, ldv, None)


def attend(c=None, s="own", t=None, seq=P, lengths=P, tokens=1, window=0, sink=0, q=P, ldq=256, hq=4, scale=1.0, R=2,
           out=P, ldo=256, lse=P, acc=0):
    return L.xt_paged_attention_window(ref_(c or codes()), ref_(scales() if s == "own" else s), ref_(t or table()), seq,
                                       lengths, tokens, window, sink, q, ldq, hq, scale, R, out, ldo, lse, acc, None)


def verify(dtype=0, x=P, ls=300, lr=100, y=P, ds=200, dr=100, S=2, T=2, V=100, drafted=P, counts=P, u=P, temp=1.0,
           temps=None, acc=P, tok=P, lp=P):
    return L.xt_verify_drafts(dtype, x, ls, lr, y, ds, dr, S, T, V, drafted, counts, u, temp, temps, acc, tok, lp, None)


@pytest.mark.parametrize("call", [store, read, attend], ids=lambda f: f.__name__)
def test_bad_caches_scales_and_tables(call):
    for f in CACHE_FAULTS:
        if f.get("dtype") not in (3, 0) and "score" not in f and not {f.get("k"), f.get("v")} & {P + 1}:
            assert call(c=codes(**f)) == xtern.XT_ERR_INVALID, f
        assert call(c=cache(**f), s=None) == xtern.XT_ERR_INVALID, f
    for f in TABLE_FAULTS:
        assert call(t=table(**f)) == xtern.XT_ERR_INVALID, f
    for f in (dict(s=None), dict(s=scales(k=None)), dict(s=scales(v=None)), dict(s=scales(k=P + 2)),
              dict(s=scales(v=P + 1)), dict(c=codes(score=P)), dict(c=cache()), dict(c=cache(dtype=4), s=None),
              dict(c=codes(dtype=4))):
        assert call(**f) == xtern.XT_ERR_INVALID, f
        assert L.xt_last_error()


FAULTS = [
    (store, dict(R=-1)), (store, dict(R=(1 << 21) + 1)), (store, dict(slots=None)), (store, dict(k=None)),
    (store, dict(v=None)), (store, dict(qo=None)), (store, dict(ldk=127)), (store, dict(ldqo=255)), (store, dict(hq=3)),
    (store, dict(ldqo=257)), (store, dict(r=rope(dim=63))), (store, dict(r=rope(cos=None))),
    (store, dict(nm=norm(k=None))), (store, dict(nm=norm(q=None))), (store, dict(nm=norm(eps=-1e-9))),
    (store, dict(nm=norm(eps=float("nan")))), (store, dict(nm=norm(eps=float("inf")))), (store, dict(nm=norm(q=P + 2))),
    (store, dict(nm=norm(k=P + 1))), (store, dict(lengths=P)), (store, dict(lengths=P + 2)),
    (read, dict(R=-1)), (read, dict(slots=None)), (read, dict(out=3)), (read, dict(out=-1)), (read, dict(k=None)),
    (read, dict(v=None)), (read, dict(ldk=127)), (read, dict(ldv=127)), (read, dict(k=P + 2)),
    (read, dict(out=1, v=P + 1)), (read, dict(ldk=1 << 60)),
    (attend, dict(tokens=0)), (attend, dict(tokens=-1)), (attend, dict(tokens=3)), (attend, dict(tokens=65537, R=65537)),
    (attend, dict(window=-1)), (attend, dict(window=(1 << 30) + 1)), (attend, dict(window=5, sink=-1)),
    (attend, dict(window=5, sink=(1 << 30) + 1)), (attend, dict(sink=1)), (attend, dict(acc=1)), (attend, dict(hq=5)),
    (attend, dict(lengths=None)), (attend, dict(q=None)), (attend, dict(out=None)), (attend, dict(ldo=257)),
    (attend, dict(scale=float("nan"))), (attend, dict(lse=P + 2)),
    (verify, dict(dtype=3)), (verify, dict(T=-1)), (verify, dict(T=65)), (verify, dict(S=-1)), (verify, dict(S=1 << 21)),
    (verify, dict(S=1 << 62)), (verify, dict(V=0)), (verify, dict(V=(1 << 30) + 1)), (verify, dict(x=None)),
    (verify, dict(drafted=None)), (verify, dict(u=None)), (verify, dict(acc=None)), (verify, dict(tok=None)),
    (verify, dict(lp=None)), (verify, dict(temp=-0.5)), (verify, dict(temp=float("nan"))),
    (verify, dict(temp=float("inf"))), (verify, dict(ls=-1)), (verify, dict(lr=-1)), (verify, dict(ds=-1)),
    (verify, dict(dr=-1)), (verify, dict(ls=1 << 62)), (verify, dict(dr=1 << 62)), (verify, dict(x=P + 2)),
    (verify, dict(dtype=1, y=P + 1)), (verify, dict(u=P + 2)), (verify, dict(temps=P + 2)), (verify, dict(counts=P + 1)),
]


@pytest.mark.parametrize("i", range(len(FAULTS)))
def test_bad_arguments(i):
    call, f = FAULTS[i]
    assert call(**f) == xtern.XT_ERR_INVALID, (call.__name__, f)
    assert L.xt_last_error()


def test_calls_without_codes_refuse_them():
    """The calls that take no scales say that codes need them."""
    c, t = ref_(codes()), ref_(table())
    assert L.xt_kv_append(c, t, P, P, P, None, None, 0, 0, None, 0, P, 128, P, 128, 1, None) == xtern.XT_ERR_INVALID
    assert L.xt_paged_attention(c, t, P, P, P, 256, 4, 1.0, 1, P, 256, None, 0, None) == xtern.XT_ERR_INVALID
    assert b"scales" in L.xt_last_error()
    assert L.xt_kv_evict(c, t, P, 8, 0, 0, P + 64, P, None) == xtern.XT_ERR_INVALID


def test_rows_times_heads():
    """One int numbers the workgroups of a call over codes, a row's heads each."""
    wide = lambda h: codes(kv_heads=h, head_dim=1, stride_slot=h, stride_page=16 * h, stride_head=1)  # noqa: E731
    big = dict(ldq=1 << 16, ldo=1 << 16)
    assert attend(c=wide(65535), R=32769, hq=65535, **big) == xtern.XT_ERR_INVALID
    assert b"below 2^31" in L.xt_last_error()
    assert attend(c=wide(16), R=1 << 21, hq=16 * 1024, **big) == xtern.XT_ERR_INVALID
    assert b"below 2^31" in L.xt_last_error()


def test_verify_outputs_are_arrays_of_their_own():
    """(2 sequences of 2 drafts: arrays of 4, 2, 6 and 2 words, then 2, 6 and 6)"""
    at = dict(drafted=P, counts=P + 16, u=P + 24, temps=P + 48, acc=P + 56, tok=P + 64, lp=P + 88)
    for out, n in (("acc", 2), ("tok", 6), ("lp", 6)):
        for other, size in (("drafted", 4), ("counts", 2), ("u", 6), ("temps", 2), ("acc", 2), ("tok", 6), ("lp", 6)):
            if other == out:
                continue
            for where in (at[other], at[other] + 4 * size - 4, at[other] - 4 * n + 4):
                assert verify(**{**at, out: where}) == xtern.XT_ERR_INVALID, (out, other, where)
                assert b"overlaps" in L.xt_last_error()


def test_no_rows_is_no_work():
    assert store(R=0, slots=None, k=None) == xtern.XT_OK
    assert read(R=0, slots=None, k=None) == xtern.XT_OK
    assert attend(R=0, lengths=None, q=None, tokens=7) == xtern.XT_OK
    assert verify(S=0, x=None, u=None) == xtern.XT_OK


def test_workspaces_beyond_any_device():
    t = table(seqs=1 << 21, max_pages=1 << 26, stride=1 << 26)
    assert attend(c=cache(), s=None, t=t, R=1 << 21, hq=2048, ldq=1 << 17, ldo=1 << 17, acc=1, tokens=1 << 16,
                  window=4) == xtern.XT_ERR_NOMEM


# --- the Python calls ------------------------------------------------------

def test_python_refuses():
    k = torch.zeros((4, 16, 2, 64), dtype=torch.int8)
    with pytest.raises(xtern.XternError, match="must be a CUDA"):
        xtern.KvCache(k, k)
    for x in (torch.zeros((2, 3, 10)), torch.zeros((2, 3, 10), dtype=torch.int32), np.zeros((2, 3, 10))):
        with pytest.raises(xtern.XternError, match="must be a"):
            xtern.verify_drafts(x, torch.zeros((2, 2), dtype=torch.int32), torch.zeros((2, 3)))
    for x in (torch.zeros((2, 10)), torch.zeros((2, 0, 10))):
        with pytest.raises(xtern.XternError, match="drafts \\+ 1"):
            xtern.verify_drafts(x, torch.zeros((2, 2), dtype=torch.int32), torch.zeros((2, 3)))


class Norm:
    def __init__(self, n, eps=1e-6):
        self.weight, self.eps = torch.ones(n), eps


def test_layer_refuses():
    args = [FakeLinear(32, 256), FakeLinear(32, 128), FakeLinear(32, 128), FakeLinear(256, 32), 64]
    for kw, what in ((dict(q_norm=Norm(64)), "together"), (dict(k_norm=Norm(64)), "together"),
                     (dict(q_norm=Norm(64), k_norm=Norm(128)), "head_dim"),
                     (dict(q_norm=Norm(64), k_norm=Norm(64, 1e-5)), "one eps")):
        with pytest.raises(xtern.XternError, match=what):
            xtern.CausalSelfAttention(*args, **kw)
    layer = xtern.CausalSelfAttention(*args, q_norm=Norm(64), k_norm=Norm(64), window=8, sink=1)

    class Cache:
        head_dim, kv_heads = 64, 2

    with pytest.raises(xtern.XternError, match="need seq"):
        layer.forward(torch.zeros(4, 32), Cache, None, None, tokens=2)


# --- the plain forms -------------------------------------------------------

def test_codes_by_hand():
    y = torch.tensor([[127.0, 1.5, 2.5, -126.5, 0.0], [2.0 ** -120] * 5, [0.0] * 5, [float("inf"), 1, 2, 3, 4],
                      [float("nan"), 1, 2, 3, 4], [-3e38, 3e38, 0, 0, 1e38]], dtype=torch.float64)
    c, s = ref.codes(y)
    assert c[0].tolist() == [127, 2, 2, -126, 0] and float(s[0]) == 1.0
    assert c[1:5].abs().max() == 0 and s[1:3].tolist() == [0.0, 0.0] and bool(torch.isnan(s[3:5]).all())
    assert c[5].tolist() == [-127, 127, 0, 0, 42]


def test_heads_by_hand():
    x = torch.tensor([3.0, 4.0, 12.0], dtype=torch.float64)
    w = torch.tensor([1.0, 2.0, 0.5])
    r = (169 / 3) ** 0.5
    want = [3 / r, 8 / r, 6 / r]
    assert ref.heads(x, w, 0.0).tolist() == pytest.approx(want)
    turned = ref.heads(x, w, 0.0, torch.tensor([0.0]), torch.tensor([1.0]))
    assert turned.tolist() == pytest.approx([-want[1], want[0], want[2]])


def test_visible_by_hand():
    row = [3, -1, 0, 9]
    see = lambda *a: [p for p, _, _ in ref.visible(row, *a)]  # noqa: E731
    assert see(8, 2, 4, 0, 0) == [0, 1, 4, 5]
    assert see(6, 2, 4, 1, 0) == [5] and see(6, 2, 4, 1, 1) == [0, 5] and see(6, 2, 4, 3, 2) == [0, 1, 4, 5]
    assert see(0, 2, 4, 1, 1) == [] and see(-3, 2, 4, 0, 0) == [] and see(100, 2, 20, 0, 0) == [0, 1, 4, 5, 6, 7]


def test_attention_bounds_see_mistakes():
    """One position too many or too few at the edge of the window, a scale of
    the neighbour, a code off by one: beyond the bounds."""
    rng = np.random.default_rng(0)
    page, H, D, n = 8, 1, 32, 40
    y = torch.from_numpy(rng.standard_normal((2, 5, page, H, D)))
    (kc, ks), (vc, vs) = ref.codes(y[0]), ref.codes(y[1])
    ks, vs = ks.transpose(1, 2).contiguous(), vs.transpose(1, 2).contiguous()
    q = torch.from_numpy(rng.standard_normal((1, 2, D)).astype(np.float32))
    t = np.arange(5, dtype=np.int32)[None]
    run = lambda n=n, w=20, s=2, k=kc, ks=ks, v=vc: ref.attention(k, v, t, page, q, [n], None, D ** -0.5, ks, vs, w, s)  # noqa: E731
    out, _, _, tol, _, _ = run()
    assert float(tol.max()) < 1e-4 * float(out.abs().max())
    off = vc.clone()
    off[3, 0, 0, :] += 1
    near = ks.clone()
    near[4] = ks[4].roll(1, -1)
    for bad in (run(w=21), run(w=19), run(s=1), run(s=3), run(n=n - 1), run(v=off), run(ks=near)):
        assert bool(((bad[0] - out).abs() > tol).any())


def test_verify_by_hand():
    ln = lambda *p: torch.tensor(p, dtype=torch.float64).log().to(torch.float32)  # noqa: E731
    p = torch.stack([ln(0.5, 0.25, 0.25, 1e-30), ln(0.125, 0.125, 0.25, 0.5)])[None]
    q = ln(0.25, 0.5, 0.25, 1e-30)[None, None]
    x = torch.tensor([[1]], dtype=torch.int32)
    run = lambda u, **kw: ref.verify(p, x, torch.tensor([u]), **kw)  # noqa: E731
    # accepted while u q < p: u < 0.5
    a, tok, lp = run([0.499, 0.3], draft=q)
    assert a.tolist() == [1] and tok.tolist() == [[1, 2]] and lp[0].tolist() == pytest.approx(np.log([0.25, 0.25]).tolist())
    a, tok, lp = run([0.501, 0.99], draft=q)  # what is left: all on token 0
    assert a.tolist() == [0] and tok.tolist() == [[0, -1]]
    a, tok, _ = run([0.3, 0.6])  # a certain draft: accepted below 0.25, else p without it
    assert a.tolist() == [0] and tok.tolist() == [[0, -1]]
    a, tok, _ = run([0.3, 0.7])
    assert tok.tolist() == [[2, -1]]
    a, tok, _ = run([0.2, 0.1], counts=[0])
    assert a.tolist() == [0] and tok.tolist() == [[0, -1]]
    a, tok, lp = run([0.2, 0.1], counts=[-1])
    assert a.tolist() == [0] and tok.tolist() == [[-1, -1]] and lp.tolist() == [[0, 0]]
    a, tok, _ = run([0.9, 0.1], temperature=0.0)
    assert a.tolist() == [0] and tok.tolist() == [[0, -1]]


def test_verify_gives_the_targets_distribution():
    """The tokens after a refused or accepted draft are distributed as p: over
    a grid of uniforms, to the grid's step."""
    rng = np.random.default_rng(3)
    V, n = 5, 60
    p, q = (torch.from_numpy(rng.standard_normal((1, 2, V)).astype(np.float32)) for _ in range(2))
    want, src = ref.chances(p[0, 0], 1.0), ref.chances(q[0, 0], 1.0)
    got = np.zeros(V)
    grid = (np.arange(n) + 0.5) / n
    for x in range(V):
        for u in grid:
            if u * src[x] < want[x]:
                got[x] += src[x] / n
                continue
            for w in grid:
                _, tok, _ = ref.verify(p, torch.tensor([[x]], dtype=torch.int32), torch.tensor([[u, w]]), q[:, :1])
                got[tok[0, 0]] += src[x] / n / n
    assert np.abs(got - want).max() < 2.0 / n
