"""What xt_kv_append_lengths refuses, on the CPU: as xt_kv_append, and lengths
that are another argument or not aligned.  And scales whose multiple in base 2
is infinite."""
import pytest

import xtern
from test_cache_cpu import CACHE_FAULTS, L, P, TABLE_FAULTS, attend, cache, ref_, rope, table


def append(c=None, t=None, slots=P, seq=P, pos=P, lengths=P + 64, R=2, k=P):
    return L.xt_kv_append_lengths(ref_(c or cache()), ref_(t or table()), seq, slots, pos, ref_(rope()), P, 256, 4, P,
                                  256, k, 128, P, 128, R, lengths, None)


@pytest.mark.parametrize("i", range(len(CACHE_FAULTS) + len(TABLE_FAULTS)))
def test_bad_caches_and_tables(i):
    f = (CACHE_FAULTS + TABLE_FAULTS)[i]
    kw = dict(c=cache(**f)) if i < len(CACHE_FAULTS) else dict(t=table(**f))
    assert append(**kw) == xtern.XT_ERR_INVALID


@pytest.mark.parametrize("f", [dict(lengths=P + 2), dict(slots=P + 64, lengths=P + 64), dict(seq=P + 64),
                               dict(pos=P + 64), dict(k=None), dict(slots=None), dict(R=-1)], ids=str)
def test_bad_arguments(f):
    assert append(**f) == xtern.XT_ERR_INVALID
    assert L.xt_last_error()


def test_no_rows():
    assert append(R=0) == xtern.XT_OK


@pytest.mark.parametrize("scale", [3e38, -3e38, 2.36e38, float("inf"), float("nan")])
def test_scales(scale):
    assert attend(scale=scale) == xtern.XT_ERR_INVALID
    assert attend(scale=scale / 10, R=0) == (xtern.XT_OK if abs(scale) < float("inf") else xtern.XT_ERR_INVALID)
