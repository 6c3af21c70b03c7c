"""Token log probabilities, entropy and alternatives against a plain 64-bit
form: element types, vocabularies from one token to 200000, masked tokens,
ties, rows that leave nothing."""
import numpy as np
import pytest
import torch

import cache_ref as ref
import xtern

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")


def log(msg):
    print(f"[case] {msg}", flush=True)


def case(x, tokens, top):
    """x [M, V] on the device (any row stride)."""
    lp, H, ids, tlp = xtern.token_logprobs(x, tokens.cuda() if tokens is not None else None, top=top)
    torch.cuda.synchronize()
    w = ref.logprobs(x.cpu(), tokens, top)
    ref.close(H, w[1], w[5], "entropy")
    if tokens is not None:
        ref.close(lp, w[0], w[4], "logprobs")
    else:
        assert lp is None
    if top:
        assert torch.equal(ids.cpu().long(), w[2]), "alternatives"
        ref.close(tlp, w[3], w[6], "their log probabilities")
    else:
        assert ids is None and tlp is None


def rows(rng, M, V, dtype, std=2.5, masked=0.0):
    x = torch.from_numpy(rng.standard_normal((M, V)) * std)
    if masked:
        x[torch.from_numpy(rng.random((M, V)) < masked)] = -INF
    return x.to(dtype).cuda()


def toks(rng, M, T, V):
    return torch.from_numpy(rng.integers(0, V, (M, T)).astype(np.int32))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 1023, 4097, 32003, 128256, 200001])
def test_vocabularies(dtype, V):
    rng = np.random.default_rng(V)
    for M, T, top in ((1, 1, min(20, V)), (3, 4, min(64, V)), (5, 2, 1)):
        log(f"logprobs {dtype} V={V} M={M} T={T} top={top}")
        case(rows(rng, M, V, dtype), toks(rng, M, T, V), top)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M", [2, 17, 300, 1100])
def test_row_counts(dtype, M):
    rng = np.random.default_rng(M)
    log(f"logprobs {dtype} M={M}")
    case(rows(rng, M, 5003, dtype), toks(rng, M, 1, 5003), 7)
    case(rows(rng, M, 5003, dtype), None, 0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_slices_of_several_tiles(dtype):
    """Enough rows that a row has few slices, each of several tiles."""
    rng = np.random.default_rng(5)
    for M, V, top in ((400, 40000, 20), (130, 70001, 64), (1030, 17000, 1)):
        log(f"logprobs {dtype} M={M} V={V} top={top}")
        case(rows(rng, M, V, dtype), toks(rng, M, 2, V), top)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("std", [0.0, 1e-3, 30.0, 3000.0])
def test_spread(dtype, std):
    """All logits equal (every alternative a tie), almost equal, far apart."""
    rng = np.random.default_rng(7)
    for top in (1, 20, 64):
        case(rows(rng, 3, 40000, dtype, std=std), toks(rng, 3, 3, 40000), top)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("masked", [0.5, 0.99, 0.9999, 1.0])
def test_masked(dtype, masked):
    rng = np.random.default_rng(11)
    for V in (70, 9000, 33333):
        case(rows(rng, 4, V, dtype, masked=masked), toks(rng, 4, 5, V), min(64, V))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_lowest_value_masks(dtype):
    """Masks of the type's lowest value: p is 0, not NaN."""
    rng = np.random.default_rng(12)
    x = rows(rng, 3, 7001, dtype)
    x[:, ::3] = torch.finfo(dtype).min
    x[2] = torch.finfo(dtype).min
    case(x, toks(rng, 3, 6, 7001), 30)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("order", ["rising", "falling", "blocks", "few"])
def test_orders(dtype, order):
    """Rows whose largest values lie together: at the end, at the start, in
    one stretch, and rows of few distinct values."""
    V = 50021
    base = torch.arange(V, dtype=torch.float64) / V * 20 - 10
    if order == "falling":
        base = base.flip(0)
    elif order == "blocks":
        base = torch.where((torch.arange(V) // 700) % 9 == 4, base + 5, base - 5)
    elif order == "few":
        base = (torch.arange(V) * 7919 % 5).double()
    x = base.to(dtype).repeat(2, 1)
    x[1] = x[1].roll(1234)
    rng = np.random.default_rng(13)
    for top in (1, 5, 33, 64):
        case(x.cuda(), toks(rng, 2, 2, V), top)


def test_certain_token():
    """ln p of an almost certain token keeps its relative precision."""
    x = torch.full((4, 3000), -20.0)
    for r, gap in enumerate((5.0, 20.0, 40.0, 80.0)):
        x[r, 1717] = -20.0 + gap + 8.0
    case(x.cuda(), torch.full((4, 1), 1717, dtype=torch.int32), 3)


def test_strided_rows_and_alignment():
    rng = np.random.default_rng(14)
    for dtype in DTYPES:
        wide = rows(rng, 6, 5100, dtype)
        for off, V, step in ((0, 5001, 1), (1, 5000, 1), (3, 4097, 2), (5, 77, 3)):
            x = wide[::step, off:off + V]
            case(x, toks(rng, x.shape[0], 2, V), 9)


def test_token_ids():
    """Ids below zero give 0, ids past the vocabulary NaN; nothing else is
    touched by them."""
    rng = np.random.default_rng(15)
    t = toks(rng, 2, 6, 900)
    t[0, 1], t[0, 3], t[1, 0], t[1, 5] = -1, 900, 2 ** 31 - 1, -2 ** 31
    case(rows(rng, 2, 900, torch.float32), t, 2)


def test_nan_and_infinity():
    rng = np.random.default_rng(16)
    for dtype in DTYPES:
        x = rows(rng, 5, 3000, dtype)
        x[0, 7] = float("nan")
        x[1, 9] = INF
        x[2, 9], x[2, 11] = INF, INF
        x[3] = -INF
        x[3, 8] = float("nan")
        t = torch.tensor([[7, 9, 100]] * 5, dtype=torch.int32)
        lp, H, ids, tlp = (v.cpu() for v in xtern.token_logprobs(x, t.cuda(), top=2))
        for r in range(4):
            assert bool(torch.isnan(lp[r]).all()) and bool(torch.isnan(H[r])), r
        assert bool(torch.isfinite(lp[4]).all())
        want = torch.sort(torch.where(torch.isnan(x), -INF, x.float()).cpu(), dim=-1, descending=True,
                          stable=True).indices
        for r in (0, 1, 2, 4):
            assert torch.equal(ids[r].long(), want[r, :2]), r
        # NaN stands behind -inf
        assert ids[3].tolist() == [0, 1]
        y = torch.full((1, 3), float("nan"), dtype=dtype, device="cuda")
        assert xtern.token_logprobs(y, top=3)[2].tolist() == [[0, 1, 2]]


def test_no_tokens():
    x = torch.zeros((2, 64), device="cuda")
    lp, H, ids, tlp = xtern.token_logprobs(x, torch.zeros((2, 0), dtype=torch.int32, device="cuda"), top=64)
    assert lp.shape == (2, 0) and ids.tolist() == [list(range(64))] * 2
    ref.close(tlp, torch.full((2, 64), -np.log(64.0), dtype=torch.float64), torch.full((2, 64), 8 * ref.EPS * np.log(64.0)), "uniform")


def test_no_rows():
    lp, H, ids, tlp = xtern.token_logprobs(torch.zeros((0, 10), device="cuda"),
                                           torch.zeros((0, 1), dtype=torch.int32, device="cuda"), top=2)
    assert lp.shape == (0, 1) and H.shape == (0,) and ids.shape == (0, 2) and tlp.shape == (0, 2)
