"""The paged key-value cache, token probabilities and the verification of
drafted tokens over the C ABI: append, read-back, attention, eviction (xt_kv_*,
xt_paged_attention), xt_token_logprobs and xt_verify_drafts.

Tensors are on the current device; a call runs on torch's current stream or
on `stream`.  With a `stream` of its own, results are allocated on that
stream and the inputs are marked as used there.
"""
import ctypes

from . import XT_ERR_INVALID, XternError, _check, _cur_device, _i64, _lib, _stream_ptr, _torch, _torch_mod, _vp

XT_F32, XT_F16, XT_BF16 = 0, 1, 2
XT_I8 = 3  # of a cache alone


class _KvCache(ctypes.Structure):
    """struct xt_kv_cache (include/xtern.h)."""
    _fields_ = [("k", _vp), ("v", _vp), ("score", _vp), ("dtype", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("page_size", ctypes.c_int), ("num_pages", _i64),
                ("stride_page", _i64), ("stride_slot", _i64), ("stride_head", _i64)]


class _KvTable(ctypes.Structure):
    """struct xt_kv_table."""
    _fields_ = [("pages", _vp), ("stride", _i64), ("seqs", _i64), ("max_pages", _i64)]


class _Rope(ctypes.Structure):
    """struct xt_rope."""
    _fields_ = [("cos", _vp), ("sin", _vp), ("rows", _i64), ("dim", ctypes.c_int)]


class _KvScales(ctypes.Structure):
    """struct xt_kv_scales."""
    _fields_ = [("k", _vp), ("v", _vp)]


class _HeadNorm(ctypes.Structure):
    """struct xt_head_norm."""
    _fields_ = [("q", _vp), ("k", _vp), ("eps", ctypes.c_double)]


_cache_p, _table_p, _rope_p, _scales_p, _norm_p = (ctypes.POINTER(t) for t in (_KvCache, _KvTable, _Rope, _KvScales,
                                                                               _HeadNorm))
_lib.xt_kv_append.argtypes = [_cache_p, _table_p, _vp, _vp, _vp, _rope_p, _vp, _i64, ctypes.c_int, _vp, _i64,
                              _vp, _i64, _vp, _i64, _i64, _vp]
_lib.xt_kv_append_lengths.argtypes = _lib.xt_kv_append.argtypes[:-1] + [_vp, _vp]
_lib.xt_kv_store.argtypes = [_cache_p, _scales_p, _table_p, _vp, _vp, _vp, _rope_p, _norm_p, _vp, _i64, ctypes.c_int,
                             _vp, _i64, _vp, _i64, _vp, _i64, _i64, _vp, _vp]
_lib.xt_kv_read.argtypes = [_cache_p, _scales_p, _table_p, _vp, _vp, _i64, ctypes.c_int, _vp, _i64, _vp, _i64, _vp]
_lib.xt_paged_attention_window.argtypes = [_cache_p, _scales_p, _table_p, _vp, _vp, _i64, _i64, _i64, _vp, _i64,
                                           ctypes.c_int, ctypes.c_float, _i64, _vp, _i64, _vp, ctypes.c_int, _vp]
_lib.xt_verify_drafts.argtypes = [ctypes.c_int, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _i64, _i64, _vp, _vp, _vp,
                                  ctypes.c_float, _vp, _vp, _vp, _vp, _vp]
_lib.xt_paged_attention.argtypes = [_cache_p, _table_p, _vp, _vp, _vp, _i64, ctypes.c_int, ctypes.c_float, _i64,
                                    _vp, _i64, _vp, ctypes.c_int, _vp]
_lib.xt_kv_evict.argtypes = [_cache_p, _table_p, _vp, _i64, _i64, _i64, _vp, _vp, _vp]
_lib.xt_token_logprobs.argtypes = [ctypes.c_int, _vp, _i64, _i64, _i64, _vp, _i64, _vp, _vp, ctypes.c_int, _vp,
                                   _vp, _vp]


def _invalid(msg):
    return XternError(XT_ERR_INVALID, msg)


def _torch_types():
    torch = _torch()
    return (torch.int32, torch.float32, torch.int8,
            {torch.float32: XT_F32, torch.float16: XT_F16, torch.bfloat16: XT_BF16})


_I32, _F32, _I8, _DTYPES = _torch_types() if _torch_mod is not None else (None, None, None, {})
_empty_strided = _torch_mod.empty_strided if _torch_mod is not None else None


# The checks of one call's tensors cost as much as a small kernel: each makes
# its sure case in few attribute reads and leaves the message to _refuse.

def _here():
    """The current device's index; -2 (no tensor's) without one."""
    try:
        return _cur_device() if _cur_device is not None else _torch().cuda.current_device()
    except RuntimeError:
        return -2


def _refuse(t, dtype, what, shape, here):
    if not isinstance(t, _torch().Tensor) or not t.is_cuda:
        raise _invalid(f"{what} must be a CUDA (HIP) tensor")
    if t.dtype != dtype:
        raise _invalid(f"{what} must be {dtype}, got {t.dtype}")
    if t.get_device() != here:
        raise _invalid(f"{what} is on {t.device}, the current device is cuda:{here}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise _invalid(f"{what} must be {list(shape)}, got {list(t.shape)}")
    raise _invalid(f"{what} must be contiguous")


def _ptr(t, dtype, what, here):
    """Address of a tensor of this type on the current device."""
    try:
        if t.dtype is dtype and t.get_device() == here:
            return t.data_ptr()
    except AttributeError:
        pass
    _refuse(t, dtype, what, None, here)


def _vec(t, dtype, what, shape, here):
    """Address of a contiguous tensor of this type and shape."""
    try:
        if t.dtype is dtype and t.get_device() == here and t.shape == shape and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _refuse(t, dtype, what, shape, here)


def _head_rows(t, what, D, here, R=None, heads=None):
    """(address, row stride, heads) of float32 rows [R, heads * D] or [R,
    heads, D] whose elements lie side by side; rows may be any distance
    apart."""
    try:
        if t.dtype is _F32 and t.get_device() == here and t.is_contiguous():
            s = t.shape
            n = s[1] if len(s) == 3 and s[2] == D else (s[1] // D if len(s) == 2 and not s[1] % D else 0)
            if n and (R is None or s[0] == R) and (heads is None or n == heads):
                return t.data_ptr(), n * D, n
    except AttributeError:
        pass
    p = _ptr(t, _F32, what, here)
    s = t.shape
    if len(s) == 3:
        n = s[1]
        ok = s[2] == D and n > 0 and (t.stride(2) == 1 or D == 1) and (t.stride(1) == D or n == 1)
    else:
        n = s[1] // D if len(s) == 2 else 0
        ok = n > 0 and n * D == s[1] and (t.stride(1) == 1 or s[1] == 1)
    if not ok or (heads is not None and n != heads):
        if len(s) in (2, 3) and (s[1:] == (heads or n, D) or s[1:] == ((heads or n) * D,)) and n > 0:
            raise _invalid(f"{what} must be contiguous within a row")
        h = "heads" if heads is None else heads
        raise _invalid(f"{what} must be [rows, {h} * {D}] or [rows, {h}, {D}], got {list(s)}")
    if R is not None and s[0] != R:
        raise _invalid(f"{what} must have {R} rows, got {s[0]}")
    return p, t.stride(0), n


def _mark(stream, *inputs):
    """Keeps the inputs allocated until the stream's work so far is done."""
    for t in inputs:
        if t is not None:
            t.record_stream(stream)


def _empty(stream, dtype, device, *shape):
    """A contiguous output, on the allocator's side of the stream that writes
    it.  (Given strides, torch allocates in two thirds of the time.)"""
    strides = (1,) if len(shape) == 1 else ((shape[1], 1) if len(shape) == 2 else (shape[1] * shape[2], shape[2], 1))
    if stream is None:
        return _empty_strided(shape, strides, dtype=dtype, device=device)
    with _torch().cuda.stream(stream):
        return _empty_strided(shape, strides, dtype=dtype, device=device)


class KvCache:
    """A pool of pages (xt_kv_cache): k and v [num_pages, page_size, kv_heads,
    head_dim] of one type (float32, float16, bfloat16, int8) and of equal
    strides (any order; head_dim contiguous), score None or [num_pages,
    kv_heads, page_size] float32, the attention weight each position has
    received.  int8 codes need k_scale and v_scale, shaped as score: a code
    stands for itself times its position's and head's scale; they keep no
    score."""

    def __init__(self, k, v, score=None, k_scale=None, v_scale=None):
        torch = _torch()
        for t, what in ((k, "k"), (v, "v")):
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise _invalid(f"{what} must be a CUDA (HIP) tensor")
            if t.dim() != 4:
                raise _invalid(f"{what} must be [num_pages, page_size, kv_heads, head_dim], got {list(t.shape)}")
        codes = k.dtype == torch.int8
        if not codes and k.dtype not in _DTYPES:
            raise _invalid(f"k must be float32, float16, bfloat16 or int8, got {k.dtype}")
        if v.dtype != k.dtype or v.shape != k.shape or v.device != k.device:
            raise _invalid("k and v must have one type, shape and device")
        P, page, H, D = k.shape
        if D > 1 and (k.stride(3) != 1 or v.stride(3) != 1):
            raise _invalid("head_dim must be contiguous")
        if any(n > 1 and a != b for n, a, b in zip(k.shape, k.stride(), v.stride())):
            raise _invalid("k and v must have equal strides")
        if codes and score is not None:
            raise _invalid("a cache of 8-bit codes keeps no score")
        if codes != (k_scale is not None) or codes != (v_scale is not None):
            raise _invalid("k_scale and v_scale are needed for int8 codes, and only there")
        for t, what in ((score, "score"), (k_scale, "k_scale"), (v_scale, "v_scale")):
            if t is None:
                continue
            if not isinstance(t, torch.Tensor) or t.device != k.device:
                raise _invalid(f"{what} must be on the device of k")
            if t.dtype != torch.float32 or tuple(t.shape) != (P, H, page) or not t.is_contiguous():
                raise _invalid(f"{what} must be contiguous float32 [{P}, {H}, {page}]")
        self.k, self.v, self.score, self.k_scale, self.v_scale = k, v, score, k_scale, v_scale
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = P, page, H, D
        self._c = _KvCache(k.data_ptr(), v.data_ptr(), score.data_ptr() if score is not None else None,
                           XT_I8 if codes else _DTYPES[k.dtype], H, D, page, P, k.stride(0), k.stride(1), k.stride(2))
        self._scales = _KvScales(k_scale.data_ptr(), v_scale.data_ptr()) if codes else None
        self._sref = ctypes.byref(self._scales) if codes else None
        self._device, self._ref = k.get_device(), ctypes.byref(self._c)

    @classmethod
    def new(cls, num_pages, page_size, kv_heads, head_dim, dtype=None, score=False, device="cuda"):
        """A pool of zeros; the slots of a head lie side by side in a page."""
        torch = _torch()
        dtype = torch.bfloat16 if dtype is None else dtype
        k, v = (torch.zeros((num_pages, kv_heads, page_size, head_dim), dtype=dtype,
                            device=device).transpose(1, 2) for _ in range(2))
        more = lambda want: (torch.zeros((num_pages, kv_heads, page_size), dtype=torch.float32, device=device)  # noqa: E731
                             if want else None)
        codes = dtype == torch.int8
        return cls(k, v, more(score), more(codes), more(codes))

    def _tensors(self):
        return self.k, self.v, self.score, self.k_scale, self.v_scale

    def _on(self, here):
        if self._device != here:
            raise _invalid(f"the cache is on cuda:{self._device}, the current device is cuda:{here}")
        return self._ref


def _table(table, here):
    """xt_kv_table of an int32 tensor [seqs, max_pages]."""
    p = _ptr(table, _I32, "table", here)
    s = table.shape
    if len(s) != 2 or (s[1] > 1 and table.stride(1) != 1):
        raise _invalid("table must be [seqs, max_pages], contiguous within a row")
    return ctypes.byref(_KvTable(p, table.stride(0), s[0], s[1])), s[0]


def kv_append(cache, table, slots, k, v, q=None, seq=None, positions=None, rope=None, q_out=None, stream=None,
              lengths=None, norm=None):
    """xt_kv_append: R new tokens' k and v (float32 [R, kv_heads, head_dim] or
    [R, kv_heads * head_dim]) into position slots[r] (int32 [R]; -1 skips the
    row) of sequence seq[r] (default r) of table (int32 [seqs, max_pages]).
    rope = (cos, sin), float32 [rows, dim / 2] each, rotates k and q by row
    positions[r] (default slots[r]).  lengths (int32 [R], if given) receives
    what each token sees, slots[r] + 1, or 0 for a row that was skipped.
    norm = (q weight, k weight, eps), float32 [head_dim] each, norms q's and
    k's heads before the rotation (xt_kv_store, as for an int8 cache, which gets
    codes and a scale for each token and head; in 64 bits, where xt_kv_append
    rotates in 32).
    Returns the rotated q (q_out if given, which may be q), or None without q."""
    here, D = _here(), cache.head_dim
    c = cache._on(here)
    t, S = _table(table, here)
    kp, ldk, _ = _head_rows(k, "k", D, here, None, cache.kv_heads)
    R = k.shape[0]
    vp, ldv, _ = _head_rows(v, "v", D, here, R, cache.kv_heads)
    sp = _vec(slots, _I32, "slots", (R,), here)
    if seq is not None:
        np_ = _vec(seq, _I32, "seq", (R,), here)
    elif R > S:
        raise _invalid(f"{R} rows for {S} sequences: seq is needed")
    else:
        np_ = None
    pp = _vec(positions, _I32, "positions", (R,), here) if positions is not None else None
    lp = _vec(lengths, _I32, "lengths", (R,), here) if lengths is not None else None
    rp = None
    if rope is not None:
        cos, sin = rope
        cp = _ptr(cos, _F32, "cos", here)
        if cos.dim() != 2 or not cos.is_contiguous():
            raise _invalid("cos must be contiguous [rows, dim / 2]")
        rp = ctypes.byref(_Rope(cp, _vec(sin, _F32, "sin", cos.shape, here), cos.shape[0], 2 * cos.shape[1]))
    hp = None
    if norm is not None:
        wq, wk, eps = norm
        hp = ctypes.byref(_HeadNorm(_vec(wq, _F32, "the query norm", (D,), here) if wq is not None else None,
                                    _vec(wk, _F32, "the key norm", (D,), here), eps))
    qp = op = None
    ldq = ldo = hq = 0
    if q is not None:
        qp, ldq, hq = _head_rows(q, "q", D, here, R)
        if q_out is None:
            q_out = _empty(stream, _F32, q.device, *q.shape)
        op, ldo, _ = _head_rows(q_out, "q_out", D, here, R, hq) if q_out is not q else (qp, ldq, hq)
    elif q_out is not None:
        raise _invalid("q_out without q")
    if stream is not None:
        _mark(stream, *cache._tensors(), table, slots, k, v, q, seq, positions, q_out, lengths, *(rope or ()),
              *(norm or ())[:2])
    if hp is not None or cache._sref is not None:
        _check(_lib.xt_kv_store(c, cache._sref, t, np_, sp, pp, rp, hp, qp, ldq, hq, op, ldo, kp, ldk, vp, ldv, R, lp,
                                _stream_ptr(stream)))
        return q_out
    _check(_lib.xt_kv_append_lengths(c, t, np_, sp, pp, rp, qp, ldq, hq, op, ldo, kp, ldk, vp, ldv, R, lp,
                                     _stream_ptr(stream)))
    return q_out


def kv_read(cache, table, slots, seq=None, dtype=None, stream=None):
    """xt_kv_read: keys and values of R positions as the cache holds them, row r
    of position slots[r] (int32 [R]) of sequence seq[r] (default r) of table
    (int32 [seqs, max_pages]), zeros where there is none.  Returns (k, v) [R,
    kv_heads, head_dim] of dtype (float32, the default, float16 or bfloat16)."""
    here, D = _here(), cache.head_dim
    c = cache._on(here)
    t, S = _table(table, here)
    if getattr(slots, "ndim", 1) != 1:
        raise _invalid(f"slots must be [rows], got {list(slots.shape)}")
    sp = _vec(slots, _I32, "slots", getattr(slots, "shape", None), here)
    R = slots.shape[0]
    if seq is not None:
        np_ = _vec(seq, _I32, "seq", (R,), here)
    elif R > S:
        raise _invalid(f"{R} rows for {S} sequences: seq is needed")
    else:
        np_ = None
    dtype = _F32 if dtype is None else dtype
    if dtype not in _DTYPES:
        raise _invalid(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    k, v = (_empty(stream, dtype, slots.device, R, cache.kv_heads, D) for _ in range(2))
    if stream is not None:
        _mark(stream, *cache._tensors(), table, slots, seq)
    ld = cache.kv_heads * D
    _check(_lib.xt_kv_read(c, cache._sref, t, np_, sp, R, _DTYPES[dtype], k.data_ptr(), ld, v.data_ptr(), ld,
                           _stream_ptr(stream)))
    return k, v


def _check_spans(R, tokens, window, sink):
    if window is not None and not 1 <= window <= 1 << 30:
        raise _invalid("window must be 1..2^30")
    if not 0 <= sink <= 1 << 30 or (sink and window is None):
        raise _invalid("sink must be 0..2^30, and 0 without a window")
    if not 1 <= tokens <= 65536 or R % tokens:
        raise _invalid("tokens must be 1..65536, a divisor of the rows")


def paged_attention(cache, table, lengths, q, seq=None, scale=None, lse=False, accumulate=False, out=None,
                    stream=None, window=None, sink=0, tokens=1):
    """xt_paged_attention: row r of q (float32 [R, q_heads, head_dim] or [R,
    q_heads * head_dim]) attends over the first lengths[r] (int32 [R])
    positions of sequence seq[r] (default r) of table (int32 [seqs,
    max_pages]).  scale defaults to head_dim ** -0.5.  Returns out (which may
    be q), shaped as q, or (out, lse [R, q_heads]) with lse=True; accumulate=True adds the
    weights to cache.score.
    xt_paged_attention_window: of those positions a row sees the newest `window`
    (1..2^30) and the first `sink`; groups of `tokens` rows belong to one
    sequence, the one that seq names for the group's first row (default: group
    g to sequence g), and share passes over an int8 cache."""
    here, D = _here(), cache.head_dim
    c = cache._on(here)
    t, S = _table(table, here)
    qp, ldq, hq = _head_rows(q, "q", D, here)
    R = q.shape[0]
    lp = _vec(lengths, _I32, "lengths", (R,), here)
    spans = window is not None or tokens != 1 or sink
    if spans:
        _check_spans(R, tokens, window, sink)
    if seq is not None:
        sp = _vec(seq, _I32, "seq", (R,), here)
    elif R > S * tokens:
        raise _invalid(f"{R // tokens} groups of rows for {S} sequences: seq is needed" if tokens > 1 else
                       f"{R} rows for {S} sequences: seq is needed")
    else:
        sp = None
    if out is None:
        out = _empty(stream, _F32, q.device, *q.shape)
    op, ldo, _ = _head_rows(out, "out", D, here, R, hq)
    l = _empty(stream, _F32, q.device, R, hq) if lse else None
    if stream is not None:
        _mark(stream, *cache._tensors(), table, lengths, q, seq, out)
    if scale is None:
        scale = D ** -0.5
    if spans or cache._sref is not None:
        _check(_lib.xt_paged_attention_window(c, cache._sref, t, sp, lp, tokens, window or 0, sink, qp, ldq, hq, scale,
                                              R, op, ldo, l.data_ptr() if lse else None, 1 if accumulate else 0,
                                              _stream_ptr(stream)))
    else:
        _check(_lib.xt_paged_attention(c, t, sp, lp, qp, ldq, hq, scale, R, op, ldo, l.data_ptr() if lse else None,
                                       1 if accumulate else 0, _stream_ptr(stream)))
    return (out, l) if lse else out


def kv_evict(cache, table, lengths, budget, sink=0, recent=0, stream=None):
    """xt_kv_evict: every sequence of table with lengths[b] (int32 [seqs]) >
    budget is cut down to budget positions per key-value head, the first
    `sink`, the last `recent` and those of the highest cache.score between
    them, moved in order to the front of its pages.  Positions without a page
    do not count and are not moved to.  Returns (new lengths [seqs], up to the
    last position in use; kept [seqs, kv_heads, budget]: the old position of
    each that stayed, then -1)."""
    here = _here()
    c = cache._on(here)
    t, S = _table(table, here)
    lp = _vec(lengths, _I32, "lengths", (S,), here)
    if not 1 <= budget < 1 << 31:
        raise _invalid("budget must be 1..2^31-1")
    new = _empty(stream, _I32, table.device, S)
    kept = _empty(stream, _I32, table.device, S, cache.kv_heads, budget)
    if stream is not None:
        _mark(stream, cache.k, cache.v, cache.score, table, lengths)
    _check(_lib.xt_kv_evict(c, t, lp, budget, sink, recent, new.data_ptr(), kept.data_ptr(), _stream_ptr(stream)))
    return new, kept


def token_logprobs(logits, tokens=None, top=0, stream=None):
    """xt_token_logprobs over the rows of logits [M, V] (float32, float16 or
    bfloat16, -inf for masked tokens; rows may be any distance apart).  tokens:
    int32 [M] or [M, T].  Returns (log probabilities shaped as tokens, or
    None; entropy [M]; ids int32 [M, top] of the most likely tokens and their
    log probabilities [M, top], or None, None)."""
    here = _here()
    dtype = getattr(logits, "dtype", None)
    xp = _ptr(logits, dtype, "logits", here)
    if dtype not in _DTYPES:
        raise _invalid(f"logits must be float32, float16 or bfloat16, got {dtype}")
    s = logits.shape
    if len(s) != 2 or (s[1] > 1 and logits.stride(1) != 1):
        raise _invalid("logits must be [rows, vocabulary], contiguous within a row")
    (M, V), T, tp, lp, ids, best = s, 0, None, None, None, None
    if not 0 <= top <= 64:
        raise _invalid("top must be 0..64, at most the vocabulary")
    dev = logits.device
    if tokens is not None:
        tp = _ptr(tokens, _I32, "tokens", here)
        n = tokens.shape
        if len(n) not in (1, 2) or n[0] != M or not tokens.is_contiguous():
            raise _invalid(f"tokens must be contiguous [{M}] or [{M}, T], got {list(n)}")
        T = 1 if len(n) == 1 else n[1]
        lp = _empty(stream, _F32, dev, *n)
    entropy = _empty(stream, _F32, dev, M)
    if top:
        ids, best = _empty(stream, _I32, dev, M, top), _empty(stream, _F32, dev, M, top)
    if stream is not None:
        _mark(stream, logits, tokens)
    _check(_lib.xt_token_logprobs(_DTYPES[dtype], xp, logits.stride(0), M, V, tp, T, lp.data_ptr() if T else None,
                                  entropy.data_ptr(), top, ids.data_ptr() if top else None,
                                  best.data_ptr() if top else None, _stream_ptr(stream)))
    return lp, entropy, ids, best


def _rows_of_logits(t, what, shape, dtype, here):
    """(address, sequence stride, row stride) of logits [S, rows, V] whose rows
    are contiguous."""
    p = _ptr(t, dtype, what, here)
    if t.shape != shape:
        raise _invalid(f"{what} must be {list(shape)}, got {list(t.shape)}")
    if shape[2] > 1 and t.stride(2) != 1 and shape[0] and shape[1]:
        raise _invalid(f"{what} must be contiguous within a row")
    return p, t.stride(0), t.stride(1)


def verify_drafts(target, drafted, uniforms, draft=None, counts=None, temperature=1.0, stream=None):
    """xt_verify_drafts: T (0..64) drafted tokens (int32 [S, T]) of each of S
    sequences against the target model's logits [S, T + 1, V] (float32, float16
    or bfloat16, -inf for masked tokens) and the logits that they were drawn
    from at the same temperature, draft [S, T, V] of target's type (None: each
    was certain).  uniforms: float32 [S, T +
    1] in [0, 1), the first T accept, the last one draws.  counts (int32 [S]):
    drafts of each sequence (default T; negative: no sequence).  temperature:
    a number >= 0 or float32 [S]; 0 takes the most likely token.  Returns
    (accepted int32 [S]: drafts that were; tokens int32 [S, T + 1]: these, the
    one drawn after them, then -1; logprobs float32 [S, T + 1]: the target's ln
    p of each)."""
    here = _here()
    dtype = getattr(target, "dtype", None)
    if dtype not in _DTYPES:
        raise _invalid(f"target must be a float32, float16 or bfloat16 tensor, got {dtype}")
    if len(target.shape) != 3 or target.shape[1] < 1:
        raise _invalid(f"target must be [seqs, drafts + 1, vocabulary], got {list(target.shape)}")
    S, T, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    xp, ls, lr = _rows_of_logits(target, "target", (S, T + 1, V), dtype, here)
    dp, us, cp, tp, ds, dr = (_vec(drafted, _I32, "drafted", (S, T), here), _vec(uniforms, _F32, "uniforms", (S, T + 1), here),
                              None, None, 0, 0)
    yp = None
    if draft is not None:
        yp, ds, dr = _rows_of_logits(draft, "draft", (S, T, V), dtype, here)
    if counts is not None:
        cp = _vec(counts, _I32, "counts", (S,), here)
    if isinstance(temperature, (int, float)):
        temp = float(temperature)
    else:
        temp, tp = 1.0, _vec(temperature, _F32, "temperature", (S,), here)
    dev = target.device
    accepted, tokens, logprobs = (_empty(stream, _I32, dev, S), _empty(stream, _I32, dev, S, T + 1),
                                  _empty(stream, _F32, dev, S, T + 1))
    if stream is not None:
        _mark(stream, target, drafted, uniforms, draft, counts, temperature if tp is not None else None)
    _check(_lib.xt_verify_drafts(_DTYPES[dtype], xp, ls, lr, yp, ds, dr, S, T, V, dp, cp, us, temp, tp,
                                 accepted.data_ptr(), tokens.data_ptr(), logprobs.data_ptr(), _stream_ptr(stream)))
    return accepted, tokens, logprobs
