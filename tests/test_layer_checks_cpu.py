"""What the attention layer refuses, it refuses before its append has written
into the cache: no projection, no kernel runs, so no GPU is needed."""
import pytest
import torch

import xtern
from test_cache_cpu import FakeLinear


class Cache:
    """(no tensors: a call that goes on fails with another error)"""
    head_dim, kv_heads, score = 64, 2, None


def layer(**kw):
    return xtern.CausalSelfAttention(FakeLinear(32, 256), FakeLinear(32, 128), FakeLinear(32, 128), FakeLinear(256, 32), 64,
                                     **kw)


@pytest.mark.parametrize("rows,kw,what", [
    (4, dict(tokens=3), "divisor"), (4, dict(tokens=8), "divisor"), (4, dict(tokens=0), "tokens must be"),
    (4, dict(tokens=-2), "tokens must be"), (65537, dict(tokens=65537), "tokens must be"),
    (4, dict(accumulate=True), "cache with scores"), (4, dict(tokens=2, accumulate=True), "cache with scores")], ids=str)
def test_refused_before_the_append(rows, kw, what):
    with pytest.raises(xtern.XternError, match=what):
        layer(window=8, sink=1).forward(torch.zeros(rows, 32), Cache, None, None, seq=torch.zeros(rows), **kw)


@pytest.mark.parametrize("kw,what", [
    (dict(window=0), "window must be"), (dict(window=-1), "window must be"), (dict(window=2 ** 30 + 1), "window must be"),
    (dict(sink=1), "sink must be"), (dict(window=4, sink=-1), "sink must be"),
    (dict(window=4, sink=2 ** 30 + 1), "sink must be")], ids=str)
def test_windows_that_no_call_takes(kw, what):
    with pytest.raises(xtern.XternError, match=what):
        layer(**kw)
