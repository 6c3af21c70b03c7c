"""Prompts as rows of one sequence, more of them than are split by their
length: through the attention against the plain form, and through the layer
in one call and in several."""
import numpy as np
import pytest
import torch

import cache_ref as ref
import xtern
from test_gpu_cache import DTYPES, attention_case, log
from test_gpu_decode import D, H, HID, HQ, I32, PAGE, layer, rope, tensor

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("R", [700, 1300])
def test_rows_of_growing_lengths(dtype, R):
    """A prompt of R tokens, a few rows of another, longer sequence among it."""
    log(f"prompt rows {dtype} {R}")
    seq = [1 if r % 150 == 77 else 0 for r in range(R)]
    lengths = [2500 - r if b else r + 1 for r, b in enumerate(seq)]
    attention_case(dtype, 4, 1, 64, 16, lens=[R, 2500], seq=seq, lengths=lengths)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("cuts", [[], [1, 8, 308, 608, 908]], ids=["whole", "cut"])
def test_a_prompt_through_the_layer(dtype, cuts):
    """1100 tokens of two sequences in one call, and in calls of 1, 7 and 300:
    the layer is its calls to the bit, and the attention the plain form's."""
    rng = np.random.default_rng(11)
    attn, rp = layer(rng), rope(800)
    lens = [700, 400]
    x = tensor(rng, sum(lens), HID)
    seq = [b for b, n in enumerate(lens) for _ in range(n)]
    slots = [i for n in lens for i in range(n)]
    host = rng.permutation(100)[:2 * 44].reshape(2, 44).astype(np.int32)
    table = torch.from_numpy(host).cuda()
    cache = xtern.KvCache.new(100, PAGE, H, D, dtype=dtype, score=True)
    other = xtern.KvCache.new(100, PAGE, H, D, dtype=dtype)
    rows, outs, queries = [], [], []
    for a, b in zip([0] + cuts, cuts + [len(seq)]):
        s, p = (torch.tensor(v[a:b], **I32) for v in (seq, slots))
        y = attn.forward(x[a:b], cache, table, p, seq=s, rope=rp, accumulate=True)
        q, k, v = xtern.linear_multi_f32([l.weights for l in (attn.q_proj, attn.k_proj, attn.v_proj)], x[a:b])
        q = xtern.kv_append(other, table, p, k, v, q=q, seq=s, rope=rp)
        o = xtern.paged_attention(other, table, p + 1, q, seq=s)
        assert torch.equal(y, xtern.linear_f32(attn.o_proj.weights, attn.attn_sub_norm.forward(o)))
        for r in range(a, b, 1 + (b - a) // 13):
            rows.append(r)
            outs.append(o[r - a].cpu().reshape(HQ, D))
            queries.append(q[r - a].cpu().reshape(HQ, D))
    assert torch.equal(cache.k, other.k) and torch.equal(cache.v, other.v)
    want = ref.attention(cache.k.cpu(), cache.v.cpu(), host, PAGE, torch.stack(queries), [slots[r] + 1 for r in rows],
                         [seq[r] for r in rows], D ** -0.5)
    ref.close(torch.stack(outs), want[0], want[3], "attention")
    # every token's query heads give a weight of one each: 700 weights a row at
    # most, each off by a few steps and by its row's sum (700 terms), added to a
    # score behind 700 others at most
    assert abs(float(cache.score.double().sum()) - len(seq) * HQ) <= (3 * 700 + 64) * ref.EPS * len(seq) * HQ
