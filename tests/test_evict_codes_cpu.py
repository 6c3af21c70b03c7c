"""Eviction over 8-bit codes is refused for what is missing: the scores."""
import xtern
from test_cache_cpu import P, ref_, table
from test_cache8_cpu import codes

L = xtern.lib()


def test_codes_keep_no_scores():
    for c in (codes(), codes(score=P)):
        assert L.xt_kv_evict(ref_(c), ref_(table()), P, 8, 0, 0, P + 64, P, None) == xtern.XT_ERR_INVALID
        assert b"scores" in L.xt_last_error() and b"scales" not in L.xt_last_error()
