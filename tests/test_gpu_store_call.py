"""xt_kv_store without norms into 16- and 32-bit caches: in Python those appends
take xt_kv_append, in C both calls do them."""
import ctypes

import pytest
import torch

import xtern
from test_gpu_cache import log
from test_gpu_cache8 import store_case
from xtern import cache as C

pytestmark = pytest.mark.gpu


def store(cache, table, slots, k, v, q=None, seq=None, positions=None, rope=None, q_out=None, lengths=None, norm=None):
    """kv_append by the C call alone."""
    assert norm is None
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    here, D = C._here(), cache.head_dim
    t, _ = C._table(table, here)
    r = ctypes.byref(C._Rope(at(rope[0]), at(rope[1]), rope[0].shape[0], 2 * rope[0].shape[1])) if rope is not None else None
    R, H = k.shape[:2]
    hq = q.shape[1] if q is not None else 0
    assert xtern.lib().xt_kv_store(cache._ref, cache._sref, t, at(seq), at(slots), at(positions), r, None, at(q), hq * D, hq,
                                   at(q_out), hq * D, at(k), H * D, at(v), H * D, R, at(lengths),
                                   torch.cuda.current_stream().cuda_stream) == xtern.XT_OK
    return q_out


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("heads", [(4, 2, 64, 64), (20, 5, 128, 128), (6, 3, 100, 50), (8, 2, 256, 256), (5, 5, 33, 32),
                                   (2, 1, 80, 40), (3, 1, 2, 2), (12, 4, 192, 96), (4, 2, 7, 0), (4, 1, 1, 0),
                                   (4, 2, 130, 64), (4, 2, 66, 66), (4, 2, 96, 8)], ids=str)
def test_store_without_norms(dtype, heads, monkeypatch):
    log(f"store call {dtype} {heads}")
    monkeypatch.setattr(xtern, "kv_append", store)
    store_case(dtype, *heads, page=16, norm=False)
    store_case(dtype, *heads, page=50, norm=False, in_place=True, seed=1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_many_rows_without_norms(dtype, monkeypatch):
    monkeypatch.setattr(xtern, "kv_append", store)
    for D in (64, 100, 37):
        store_case(dtype, 8, 2, D, D // 4 * 2, 16, rows=250, norm=False, seed=3)
        store_case(dtype, 8, 2, D, 0, 16, rows=250, norm=False, with_q=False, seed=4)
