"""What the cache and probability entry points refuse, on the CPU: every check
comes before the first HIP call, so no GPU is needed.  And the oracle of the
GPU tests against hand-worked values and planted mistakes."""
import ctypes

import numpy as np
import pytest
import torch

import cache_ref as ref
import xtern
from xtern.cache import _KvCache, _KvTable, _Rope

L = xtern.lib()
BUF = ctypes.create_string_buffer(1 << 12)
P = (ctypes.addressof(BUF) + 63) // 64 * 64


def cache(**kw):
    d = dict(k=P, v=P, score=P, dtype=2, kv_heads=2, head_dim=64, page_size=16, num_pages=4, stride_page=2048,
             stride_slot=64, stride_head=1024)
    return _KvCache(**{**d, **kw})


def table(**kw):
    return _KvTable(**{**dict(pages=P, stride=3, seqs=2, max_pages=3), **kw})


def rope(**kw):
    return _Rope(**{**dict(cos=P, sin=P, rows=10, dim=64), **kw})


def ref_(x):
    return ctypes.byref(x) if x is not None else None


def append(c=None, t=None, r=None, seq=P, slots=P, pos=P, q=P, ldq=256, hq=4, qo=P, ldqo=256, k=P, ldk=128, v=P,
           ldv=128, R=2):
    return L.xt_kv_append(ref_(c or cache()), ref_(t or table()), seq, slots, pos, ref_(r or rope()), q, ldq, hq, qo,
                          ldqo, k, ldk, v, ldv, R, None)


def attend(c=None, t=None, seq=P, lengths=P, q=P, ldq=256, hq=4, scale=1.0, R=2, out=P, ldo=256, lse=P, acc=0):
    return L.xt_paged_attention(ref_(c or cache()), ref_(t or table()), seq, lengths, q, ldq, hq, scale, R, out, ldo,
                                lse, acc, None)


def evict(c=None, t=None, lengths=P, budget=8, sink=1, recent=1, new=P + 64, kept=P):
    return L.xt_kv_evict(ref_(c or cache()), ref_(t or table()), lengths, budget, sink, recent, new, kept, None)


def probs(dtype=0, x=P, ld=100, M=2, V=100, tokens=P, T=1, lp=P, H=P, top=3, ids=P, tlp=P):
    return L.xt_token_logprobs(dtype, x, ld, M, V, tokens, T, lp, H, top, ids, tlp, None)


CACHE_FAULTS = [dict(dtype=3), dict(dtype=-1), dict(kv_heads=0), dict(kv_heads=1 << 17), dict(head_dim=0),
                dict(head_dim=257), dict(page_size=0), dict(page_size=65537), dict(num_pages=0),
                dict(num_pages=1 << 31), dict(k=None), dict(v=None), dict(k=P + 1), dict(v=P + 1), dict(score=P + 2),
                dict(dtype=0, k=P + 2), dict(stride_slot=63), dict(stride_head=1023), dict(stride_page=2047),
                dict(stride_page=0), dict(stride_head=0), dict(stride_page=-2048), dict(stride_page=1 << 61)]
TABLE_FAULTS = [dict(seqs=-1), dict(seqs=1 << 31), dict(seqs=(1 << 21) + 1), dict(max_pages=-1), dict(max_pages=1 << 27, stride=1 << 27),
                dict(max_pages=1 << 62, stride=1 << 62), dict(pages=None), dict(stride=2), dict(pages=P + 1)]


@pytest.mark.parametrize("call", [append, attend, evict], ids=lambda f: f.__name__)
def test_bad_caches_and_tables(call):
    for f in CACHE_FAULTS:
        assert call(c=cache(**f)) == xtern.XT_ERR_INVALID, f
    for f in TABLE_FAULTS:
        assert call(t=table(**f)) == xtern.XT_ERR_INVALID, f
        assert L.xt_last_error()


FAULTS = [
    (append, dict(R=-1)), (append, dict(R=1 << 31)), (attend, dict(R=(1 << 21) + 1)), (probs, dict(M=(1 << 21) + 1)), (append, dict(slots=None)), (append, dict(k=None)),
    (append, dict(v=None)), (append, dict(qo=None)), (append, dict(ldk=127)), (append, dict(ldv=127)),
    (append, dict(ldq=255)), (append, dict(ldqo=255)), (append, dict(hq=3)), (append, dict(hq=0)),
    (append, dict(hq=1 << 16)), (append, dict(ldqo=257)), (append, dict(k=P + 2)), (append, dict(ldk=1 << 60)),
    (append, dict(r=rope(dim=63))), (append, dict(r=rope(dim=66))), (append, dict(r=rope(dim=0))),
    (append, dict(r=rope(cos=None))), (append, dict(r=rope(sin=None))), (append, dict(r=rope(rows=-1))),
    (append, dict(r=rope(cos=P + 2))),
    (attend, dict(R=-1)), (attend, dict(lengths=None)), (attend, dict(q=None)), (attend, dict(out=None)),
    (attend, dict(hq=5)), (attend, dict(hq=2050, ldq=1 << 20, ldo=1 << 20)), (attend, dict(hq=0)), (attend, dict(hq=-2)), (attend, dict(ldq=255)),
    (attend, dict(ldo=255)), (attend, dict(scale=float("nan"))), (attend, dict(scale=float("inf"))),
    (attend, dict(c=cache(score=None), acc=1)), (attend, dict(lse=P + 2)), (attend, dict(q=P + 1)),
    (evict, dict(c=cache(score=None))), (evict, dict(budget=0)), (evict, dict(budget=1 << 31)),
    (evict, dict(sink=-1)), (evict, dict(recent=-1)), (evict, dict(sink=5, recent=4)), (evict, dict(sink=9)),
    (evict, dict(recent=1 << 62)), (evict, dict(lengths=None)), (evict, dict(new=None)), (evict, dict(kept=None)),
    (evict, dict(new=P)),
    (probs, dict(dtype=3)), (probs, dict(M=-1)), (probs, dict(V=0)), (probs, dict(V=(1 << 30) + 1, ld=1 << 40)),
    (probs, dict(T=-1)), (probs, dict(T=1 << 21)), (probs, dict(top=-1)), (probs, dict(top=65)),
    (probs, dict(V=2, top=3)), (probs, dict(x=None)), (probs, dict(H=None)), (probs, dict(tokens=None)),
    (probs, dict(lp=None)), (probs, dict(ids=None)), (probs, dict(tlp=None)), (probs, dict(ld=99)),
    (probs, dict(ld=1 << 62)), (probs, dict(x=P + 2)), (probs, dict(dtype=1, x=P + 1)), (attend, dict(ldo=257)),
]


@pytest.mark.parametrize("i", range(len(FAULTS)))
def test_bad_arguments(i):
    call, f = FAULTS[i]
    assert call(**f) == xtern.XT_ERR_INVALID, (call.__name__, f)
    assert L.xt_last_error()


def test_workspaces_beyond_any_device():
    """Sizes that a size_t would wrap."""
    t = table(seqs=1 << 21, max_pages=1 << 26, stride=1 << 26)
    assert attend(t=t, R=1 << 21, hq=2048, ldq=1 << 17, ldo=1 << 17, acc=1) == xtern.XT_ERR_NOMEM
    assert evict(t=t) == xtern.XT_ERR_NOMEM


def test_null_structs():
    assert L.xt_kv_append(None, ref_(table()), P, P, P, None, None, 0, 0, None, 0, P, 128, P, 128, 1,
                          None) == xtern.XT_ERR_INVALID
    assert L.xt_paged_attention(ref_(cache()), None, P, P, P, 256, 4, 1.0, 1, P, 256, None, 0,
                                None) == xtern.XT_ERR_INVALID
    assert L.xt_kv_evict(None, None, P, 8, 0, 0, P + 64, P, None) == xtern.XT_ERR_INVALID


def test_no_rows_is_no_work():
    assert append(R=0, slots=None, k=None) == xtern.XT_OK
    assert attend(R=0, lengths=None, q=None) == xtern.XT_OK
    assert evict(t=table(seqs=0, pages=None), lengths=None) == xtern.XT_OK
    assert probs(M=0, x=None) == xtern.XT_OK


# --- the Python calls ------------------------------------------------------

H = torch.zeros(2, 2, 64)
I = torch.zeros(2, dtype=torch.int32)


def test_python_refuses_host_tensors():
    k = torch.zeros(4, 16, 2, 64)
    with pytest.raises(xtern.XternError, match="must be a CUDA"):
        xtern.KvCache(k, k)
    with pytest.raises(xtern.XternError, match="must be a CUDA"):
        xtern.KvCache(np.zeros((4, 16, 2, 64)), k)
    with pytest.raises(xtern.XternError, match="must be a CUDA"):
        xtern.token_logprobs(torch.zeros(2, 10))
    with pytest.raises(xtern.XternError, match="must be a CUDA"):
        xtern.token_logprobs(np.zeros((2, 10)))


class FakeLinear:
    def __init__(self, i, o):
        self.in_dim, self.out_dim, self.weights = i, o, None


def test_attention_layer_refuses():
    f = FakeLinear
    ok = xtern.CausalSelfAttention(f(256, 512), f(256, 128), f(256, 128), f(512, 256), 64)
    for bad in ((f(256, 500), f(256, 128), f(256, 128), f(500, 256)), (f(256, 512), f(256, 128), f(256, 64),
                                                                       f(512, 256)),
                (f(256, 512), f(256, 128), f(256, 128), f(256, 256))):
        with pytest.raises(xtern.XternError):
            xtern.CausalSelfAttention(*bad, 64)

    class C:
        head_dim, kv_heads = 64, 2

    with pytest.raises(xtern.XternError, match="rows, hidden"):
        ok.forward(torch.zeros(256), C, None, None)
    with pytest.raises(xtern.XternError, match="Input dimension mismatch"):
        ok.forward(torch.zeros(2, 255), C, None, None)
    C.kv_heads = 1
    with pytest.raises(xtern.XternError, match="heads"):
        ok.forward(torch.zeros(2, 256), C, None, None)


# --- the plain forms that the GPU tests hold the kernels to ------------------

def small(seed=0, n=40, H=2, D=8, page=4):
    rng = np.random.default_rng(seed)
    num = n // page + 3
    mem, view, score = ref.pool(rng, num, page, H, D, torch.float32, "page_head_slot", True)
    k, v = view[0](mem[0]), view[1](mem[1])
    t = ref.tables(rng, [n], page, num)
    for _, pg, sl in ref.positions(t[0], n, page, num):
        k[pg, sl] = torch.from_numpy(rng.standard_normal((H, D)))
        v[pg, sl] = torch.from_numpy(rng.standard_normal((H, D)))
    return rng, k, v, score, t, page, n


def test_reference_attention():
    rng, k, v, score, t, page, n = small()
    q = torch.from_numpy(rng.standard_normal((1, 4, 8)).astype(np.float32))
    out, lse, new, tol, ltol, stol = ref.attention(k, v, t, page, q, [n], None, 0.3, score)
    at = ref.positions(t[0], n, page, k.shape[0])
    for h in range(4):
        s = [0.3 * float(sum(float(q[0, h, d]) * float(k[pg, sl, h // 2, d]) for d in range(8))) for _, pg, sl in at]
        z = sum(np.exp(s))
        assert abs(float(lse[0, h]) - np.log(z)) < 1e-12
        for d in range(8):
            o = sum(np.exp(x) / z * float(v[pg, sl, h // 2, d]) for x, (_, pg, sl) in zip(s, at))
            assert abs(float(out[0, h, d]) - o) < 1e-12
    assert abs(float((new - score.double()).sum()) - 4) < 1e-9  # each head gives a weight of one
    # the bounds are a few hundred float32 steps, far below a mistake
    assert float(tol.max()) < 1e-4 and float(ltol.max()) < 1e-4
    for wrong in (lambda: ref.attention(k, v, t, page, q, [n - 1], None, 0.3)[0],
                  lambda: ref.attention(k, v, t, page, q, [n], None, 0.301)[0],
                  lambda: ref.attention(k, v, t, page, q.to(torch.bfloat16).float(), [n], None, 0.3)[0],
                  lambda: ref.attention(k, v.to(torch.bfloat16), t, page, q, [n], None, 0.3)[0]):
        with pytest.raises(AssertionError):
            ref.close(wrong(), out, tol, "planted")


def test_reference_eviction():
    _, k, v, score, t, page, n = small(1)
    k0, s0 = k.clone(), score.clone()
    new, kept = ref.evict(k, v, score, t, page, [n], 12, 2, 3)
    assert new[0] == 12
    for h in range(2):
        s = np.array([float(s0[pg, h, sl]) for _, pg, sl in ref.positions(t[0], n, page, k.shape[0])])
        s[:2] = s[-3:] = 9.0
        want = np.sort(np.argsort(-s, kind="stable")[:12])
        assert kept[0, h].tolist() == want.tolist()
        for j, p in enumerate(want):
            to, fr = (t[0, j // page], j % page), (t[0, p // page], p % page)
            assert torch.equal(k[to[0], to[1], h], k0[fr[0], fr[1], h])


def test_reference_logprobs():
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.standard_normal((3, 300)) * 4)
    x[1, ::2] = -np.inf
    x[2] = -np.inf
    t = torch.tensor([[0, 5], [1, 2], [3, -1]])
    lp, H, ids, tlp, ltol, htol, _ = ref.logprobs(x, t, 3)
    ls = torch.log_softmax(x[:2], -1)
    assert torch.allclose(lp[:2], ls.gather(1, t[:2]), atol=1e-12)
    assert torch.allclose(H[:2], -(ls.exp() * torch.where(ls.isfinite(), ls, torch.zeros((), dtype=ls.dtype))).sum(-1), atol=1e-12)
    assert lp[2, 0] == -np.inf and lp[2, 1] == 0 and H[2] == 0 and ids[2].tolist() == [0, 1, 2]
    assert ids[0].tolist() == torch.argsort(x[0], descending=True)[:3].tolist()
    assert float(ltol.max()) < 1e-4 and float(htol.max()) < 1e-3
    with pytest.raises(AssertionError):
        ref.close(lp + 1e-3, lp, ltol, "planted")
