"""The outputs of xt_verify_drafts are memory of their own, beside the logits as
well: refused before the first HIP call, so no GPU is needed.  (Every call here
has something to refuse.)"""
import ctypes

import pytest

import xtern

L = xtern.lib()
BUF = ctypes.create_string_buffer(1 << 16)
P = (ctypes.addressof(BUF) + 63) // 64 * 64
WORDS = P + (1 << 15)  # arrays of words, none of which overlap
S, T, V = 3, 2, 100
OUTS = {"acc": (S, "accepted"), "tok": (S * (T + 1), "tokens"), "lp": (S * (T + 1), "logprobs")}


def verify(dtype=0, x=P, ls=3 * 120, lr=120, y=None, ds=0, dr=0, **at):
    w = {n: WORDS + 256 * i for i, n in enumerate(("drafted", "counts", "u", "acc", "tok", "lp"))}
    w.update(at)
    rc = L.xt_verify_drafts(dtype, x, ls, lr, y, ds, dr, S, T, V, w["drafted"], w["counts"], w["u"], 1.0, None, w["acc"],
                            w["tok"], w["lp"], None)
    return rc, L.xt_last_error().decode()


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
@pytest.mark.parametrize("out", OUTS)
def test_logits_are_no_place_for_results(out, dtype, size):
    n, name = OUTS[out]
    for what, rows, ls, lr in (("target", T + 1, 3 * 120, 120), ("draft", T, 120, 3 * 120), ("target", T + 1, 0, 120),
                               ("draft", T, 2 * 120, 0)):
        place = dict(x=P, ls=ls, lr=lr) if what == "target" else dict(x=P + (1 << 14), y=P, ds=ls, dr=lr)
        for b in range(S):
            for t in range(rows):
                first = P + (b * ls + t * lr) * size
                for at in (first, first + V * size - 4, first + 4 - 4 * n):
                    if at < P - 4 * n:
                        continue
                    rc, error = verify(dtype, **{**place, out: at})
                    assert rc == xtern.XT_ERR_INVALID and error == f"{name} overlaps {what}", (what, b, t, at - P, error)


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2)])
def test_gaps_between_rows_are_free(dtype, size):
    """accepted between the rows of target, or behind them: what is refused is the
    next output."""
    for gap in (P + V * size, P + 120 * size - 4 * S, P + (2 * 120 + V) * size, P + (3 * 120 + V) * size,
                P + (8 * 120 + V) * size):
        gap = (gap + 3) // 4 * 4
        rc, error = verify(dtype, acc=gap, tok=P + 120 * size)
        assert rc == xtern.XT_ERR_INVALID and error == "tokens overlaps target", (gap - P, error)
