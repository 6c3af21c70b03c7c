"""Rows of CausalSelfAttention that the append skips (a slot below zero or past
the table, a sequence or a page that is not there, a rotary position without a
row in the tables): they see nothing, add nothing to the scores, and the other
rows are as if they were not there."""
import numpy as np
import pytest
import torch

import xtern
from test_gpu_decode import D, H, HID, HQ, I32, PAGE, layer, rope, tensor

pytestmark = pytest.mark.gpu


def filled(rng, P, dtype):
    """A pool whose every slot holds something."""
    c = xtern.KvCache.new(P, PAGE, H, D, dtype=dtype, score=True)
    for x in (c.k, c.v, c.score):
        x.copy_(tensor(rng, *x.shape))
    return c


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("norm", [False, True])
def test_skipped_rows_see_nothing(dtype, norm):
    rng = np.random.default_rng(3)
    attn, rp = layer(rng, norm), rope(100)  # (rotary positions 0..99)
    first = filled(rng, 12, dtype)
    table = torch.from_numpy(rng.permutation(12)[:10].reshape(2, 5).astype(np.int32)).cuda()  # 80 positions each
    table[1, 2] = -1
    #        fine  past the rope    below   past the table  hole  no sequence  fine
    seq = [0, 0, 0, 1, 0, 0, 1, 1, 1, 2, -1, 1]
    slots = [20, 30, 31, 50, -1, 80, 2 ** 31 - 1, 35, 47, 5, 5, 70]
    pos = [99, 100, 2 ** 31 - 1, -1, 3, 4, 5, 6, 7, 8, 9, 0]
    there = [0, 11]
    x = tensor(rng, len(seq), HID)

    def run(rows, mark):
        cache = xtern.KvCache(first.k.clone(), first.v.clone(), first.score.clone())
        a, b, c = (torch.tensor([v[r] for r in rows], **I32) for v in (seq, slots, pos))
        y = attn.forward(x[rows], cache, table, b, seq=a, positions=c, rope=rp, accumulate=mark)
        return y, cache

    y, cache = run(list(range(len(seq))), True)
    want, cache2 = run(there, True)
    assert torch.equal(y[there], want)
    assert torch.equal(cache.k, cache2.k) and torch.equal(cache.v, cache2.v)
    assert torch.equal(cache.score, cache2.score)
    nothing = torch.zeros((1, HQ * D), device="cuda")
    if norm:
        nothing = attn.attn_sub_norm.forward(nothing)
    nothing = xtern.linear_f32(attn.o_proj.weights, nothing)
    for r in range(len(seq)):
        if r not in there:
            assert torch.equal(y[r], nothing[0]), r


def test_a_chat_behind_its_rope_tables():
    """Slots that stay low while positions grow past the tables: the row gives
    nothing instead of attending with a query that was not rotated."""
    rng = np.random.default_rng(5)
    attn, rp = layer(rng, False), rope(64)
    cache = filled(rng, 5, torch.bfloat16)
    table = torch.arange(5, **I32).reshape(1, 5)
    for p in range(60, 68):
        slot = torch.tensor([10 + p - 60], **I32)
        y = attn.forward(tensor(rng, 1, HID), cache, table, slot, positions=torch.tensor([p], **I32), rope=rp)
        assert bool(y.any()) == (p < 64), p


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rotated", [False, True])
def test_lengths_of_the_append(dtype, rotated):
    """slots + 1 of the rows that were written, 0 of the others; everything
    else as without them."""
    rng = np.random.default_rng(9)
    table = torch.tensor([[3, -1, 2, 9], [1, 0, 8, 4]], **I32)  # 64 positions each, pages 0..7 exist
    slots = torch.tensor([0, 15, 16, 40, 48, 63, 64, -1, 2 ** 31 - 1, -2 ** 31, 20, 33, 5, 5], **I32)
    seq = torch.tensor([0, 0, 0, 0, 0, 1, 1, 1, 1, 1, 1, 1, 2, -1], **I32)
    pos = torch.tensor([5, 64, 0, 63, 0, 63, 0, 0, 0, 0, -1, 0, 0, 0], **I32)
    want = [1, 16, 0, 41, 0, 64, 0, 0, 0, 0, 21, 0, 0, 0]
    if rotated:
        want[1] = want[10] = 0
    a, b = (xtern.KvCache.new(8, PAGE, H, D, dtype=dtype) for _ in range(2))
    R = len(want)
    q, k, v = (tensor(rng, R, h, D) for h in (HQ, H, H))
    args = dict(seq=seq, positions=pos if rotated else None, rope=rope(64) if rotated else None)
    lengths = torch.full((R,), 7, **I32)
    qa = xtern.kv_append(a, table, slots, k, v, q=q, q_out=q.clone(), lengths=lengths, **args)
    qb = xtern.kv_append(b, table, slots, k, v, q=q, q_out=q.clone(), **args)
    assert lengths.tolist() == want
    assert torch.equal(qa, qb) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    # rows of their own sequences, no q, another stream
    lengths.fill_(7)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    xtern.kv_append(a, table, slots[:2], k[:2], v[:2], lengths=lengths[:2], stream=st)
    st.synchronize()
    assert lengths.tolist() == [1, 16] + [7] * (R - 2)
    xtern.kv_append(a, table, slots[:0], k[:0], v[:0], lengths=lengths[:0])
    for bad in (lengths[:3], lengths.long(), lengths.cpu(), slots):
        with pytest.raises(xtern.XternError):
            xtern.kv_append(a, table, slots, k, v, seq=seq, lengths=bad)
