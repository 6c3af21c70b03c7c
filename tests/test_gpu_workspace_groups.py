"""Scores of several tokens of a sequence: the workspace stays within its bound
whatever the groups, and rows in any part of a call belong to their group's
sequence."""
import numpy as np
import pytest
import torch

import xtern
from test_gpu_cache import log
from test_gpu_cache_workspaces import BOUND, cache_of, tables, used

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("window,sink", [(None, 0), (40, 3), (1 << 19, 3)], ids=["all", "window", "wide window"])
@pytest.mark.parametrize("named", [False, True], ids=["rows", "seq"])
@pytest.mark.parametrize("dtype,R,tokens", [(torch.float32, 40, 8), (torch.bfloat16, 42, 42), (torch.float16, 1105, 13)],
                         ids=str)
def test_scores_of_groups(dtype, R, tokens, named, window, sink):
    """Rows of 64 query heads over a table for 2^20 positions, 4 rows to a part
    without a window, 7 with the wide one: as over the narrow table, and as each row by itself."""
    log(f"accumulate {dtype} {R} {tokens} {named} {window}")
    # (torch hands out its streams again after 32: one with a workspace of almost
    # this size from an earlier test would have it doubled here)
    xtern.workspace_release()
    rng = np.random.default_rng(R)
    hq, H, D = 64, 2, 64
    groups = R // tokens
    lens = [int(x) for x in rng.integers(100, 128, groups)]
    P, narrow, wide = tables(rng, lens, groups)
    first = cache_of(rng, P, H, D, dtype)
    q = torch.from_numpy(rng.standard_normal((R, hq, D)).astype(np.float32)).cuda()
    order = rng.permutation(groups) if named else np.arange(groups)
    seq = order.repeat(tokens)  # (only the group's first entry counts)
    named_seq = seq.copy()
    named_seq[np.arange(R) % tokens > 0] = -1
    lengths = rng.integers(0, 100, R).astype(np.int32)
    lengths[::5] = 0
    lengths[tokens - 1::tokens] = [lens[b] for b in order]
    lengths = torch.from_numpy(lengths).cuda()

    def call(small, each=False):
        c = xtern.KvCache(first.k, first.v, first.score.clone())
        at = torch.from_numpy((seq if each else named_seq).astype(np.int32)).cuda() if named or each else None
        out, lse = xtern.paged_attention(c, narrow if small else wide, lengths, q, seq=at, lse=True, accumulate=True,
                                         window=window, sink=sink, tokens=1 if each else tokens)
        return out, lse, c.score

    (out, lse, score), took = used(call)
    log(f"took {took / 2 ** 20:.0f} MiB")
    assert took < BOUND
    # (a row is split by the table's and the call's size: sums of segments in other
    # orders; 128 positions are one segment.  Scores add up in any order: half a step
    # of each of 64 / 2 + tokens additions of at most `tokens` times 32.)
    for each in (False, True):
        want = call(small=True, each=each)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        top = float(score.abs().max())
        assert float((score - want[2]).abs().max()) <= (tokens + 2) * 2.0 ** -24 * 2 * top
    assert bool(out.any())
