"""The paged key-value cache and token probabilities over the C ABI: append,
attention, eviction (xt_kv_*, xt_paged_attention) and xt_token_logprobs.

Tensors are on the current device; a call runs on torch's current stream or
on `stream`.  With a `stream` of its own, results are allocated on that
stream and the inputs are marked as used there.
"""
import contextlib
import ctypes
import math

from . import (XT_ERR_INVALID, XternError, _check, _cur_device, _i64, _lib, _raw_stream, _stream_ptr,
               _torch, _vp)

XT_F32, XT_F16, XT_BF16 = 0, 1, 2


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


_cache_p, _table_p, _rope_p = (ctypes.POINTER(t) for t in (_KvCache, _KvTable, _Rope))
_lib.xt_kv_append.argtypes = [_cache_p, _table_p, _vp, _vp, _vp, _rope_p, _vp, _i64, ctypes.c_int, _vp, _i64,
                              _vp, _i64, _vp, _i64, _i64, _vp]
_lib.xt_paged_attention.argtypes = [_cache_p, _table_p, _vp, _vp, _vp, _i64, ctypes.c_int, ctypes.c_float, _i64,
                                    _vp, _i64, _vp, ctypes.c_int, _vp]
_lib.xt_kv_evict.argtypes = [_cache_p, _table_p, _vp, _i64, _i64, _i64, _vp, _vp, _vp]
_lib.xt_token_logprobs.argtypes = [ctypes.c_int, _vp, _i64, _i64, _i64, _vp, _i64, _vp, _vp, ctypes.c_int, _vp,
                                   _vp, _vp]


def _invalid(msg):
    return XternError(XT_ERR_INVALID, msg)


def _dtypes():
    torch = _torch()
    return {torch.float32: XT_F32, torch.float16: XT_F16, torch.bfloat16: XT_BF16}


def _ptr(t, dtype, what, shape=None):
    """Address of a tensor of this type (and shape) on the current device."""
    if not isinstance(t, _torch().Tensor) or not t.is_cuda:
        raise _invalid(f"{what} must be a CUDA (HIP) tensor")
    if t.dtype != dtype:
        raise _invalid(f"{what} must be {dtype}, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise _invalid(f"{what} must be {list(shape)}, got {list(t.shape)}")
    here = _torch().cuda.current_device() if _raw_stream is None else _cur_device()
    if t.device.index != here:
        raise _invalid(f"{what} is on {t.device}, the current device is cuda:{here}")
    return t.data_ptr()


def _vec(t, dtype, what, shape):
    p = _ptr(t, dtype, what, shape)
    if not t.is_contiguous():
        raise _invalid(f"{what} must be contiguous")
    return p


def _head_rows(t, what, heads, D, R=None):
    """(address, row stride) of f32 rows [R, heads * D] or [R, heads, D] whose
    elements lie side by side; rows may be any distance apart."""
    p = _ptr(t, _torch().float32, what)
    s, d = t.shape, t.stride()
    if tuple(s[1:]) not in ((heads * D,), (heads, D)):
        raise _invalid(f"{what} must be [rows, {heads * D}] or [rows, {heads}, {D}], got {list(s)}")
    if R is not None and s[0] != R:
        raise _invalid(f"{what} must have {R} rows, got {s[0]}")
    if (len(s) == 3 and heads > 1 and d[1] != D) or (d[-1] != 1 and s[-1] != 1):
        raise _invalid(f"{what} must be contiguous within a row")
    return p, d[0]


def _heads_of(t, what, D):
    """Heads of rows [R, heads * D] or [R, heads, D]."""
    if not isinstance(t, _torch().Tensor):
        raise _invalid(f"{what} must be a CUDA (HIP) tensor")
    n = t.shape[-1] if t.dim() == 2 else (t.shape[1] * t.shape[2] if t.dim() == 3 else 0)
    if t.dim() not in (2, 3) or n == 0 or n % D or (t.dim() == 3 and t.shape[2] != D):
        raise _invalid(f"{what} must be [rows, heads * {D}] or [rows, heads, {D}], got {list(t.shape)}")
    return n // D


def _on(stream, *inputs):
    """Allocations of the block belong to `stream`; inputs stay allocated
    until its work so far is done."""
    if stream is None:
        return contextlib.nullcontext()
    for t in inputs:
        if t is not None:
            t.record_stream(stream)
    return _torch().cuda.stream(stream)


class KvCache:
    """A pool of pages (xt_kv_cache): k and v [num_pages, page_size, kv_heads,
    head_dim] of one type (float32, float16, bfloat16) and of equal strides
    (any order; head_dim contiguous), score None or [num_pages, kv_heads,
    page_size] float32, the attention weight each position has received."""

    def __init__(self, k, v, score=None):
        torch = _torch()
        for t, what in ((k, "k"), (v, "v")):
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise _invalid(f"{what} must be a CUDA (HIP) tensor")
            if t.dim() != 4:
                raise _invalid(f"{what} must be [num_pages, page_size, kv_heads, head_dim], got {list(t.shape)}")
        if k.dtype not in _dtypes():
            raise _invalid(f"k must be float32, float16 or bfloat16, got {k.dtype}")
        if v.dtype != k.dtype or v.shape != k.shape or v.device != k.device:
            raise _invalid("k and v must have one type, shape and device")
        P, page, H, D = k.shape
        if D > 1 and (k.stride(3) != 1 or v.stride(3) != 1):
            raise _invalid("head_dim must be contiguous")
        if any(n > 1 and a != b for n, a, b in zip(k.shape, k.stride(), v.stride())):
            raise _invalid("k and v must have equal strides")
        if score is not None:
            if not isinstance(score, torch.Tensor) or score.device != k.device:
                raise _invalid("score must be on the device of k")
            if score.dtype != torch.float32 or tuple(score.shape) != (P, H, page) or not score.is_contiguous():
                raise _invalid(f"score must be contiguous float32 [{P}, {H}, {page}]")
        self.k, self.v, self.score = k, v, score
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = P, page, H, D
        self._c = _KvCache(k.data_ptr(), v.data_ptr(), score.data_ptr() if score is not None else None,
                           _dtypes()[k.dtype], H, D, page, P, k.stride(0), k.stride(1), k.stride(2))

    @classmethod
    def new(cls, num_pages, page_size, kv_heads, head_dim, dtype=None, score=False, device="cuda"):
        """A pool of zeros; the slots of a head lie side by side in a page."""
        torch = _torch()
        dtype = torch.bfloat16 if dtype is None else dtype
        k, v = (torch.zeros((num_pages, kv_heads, page_size, head_dim), dtype=dtype,
                            device=device).transpose(1, 2) for _ in range(2))
        return cls(k, v, torch.zeros((num_pages, kv_heads, page_size), dtype=torch.float32, device=device)
                   if score else None)

    def _here(self):
        _ptr(self.k, self.k.dtype, "the cache")
        return ctypes.byref(self._c)


def _table(table):
    """xt_kv_table of an int32 tensor [seqs, max_pages]."""
    p = _ptr(table, _torch().int32, "table")
    if table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise _invalid("table must be [seqs, max_pages], contiguous within a row")
    return ctypes.byref(_KvTable(p, table.stride(0), table.shape[0], table.shape[1]))


def kv_append(cache, table, slots, k, v, q=None, seq=None, positions=None, rope=None, q_out=None, stream=None):
    """xt_kv_append: R new tokens' k and v (float32 [R, kv_heads, head_dim])
    into position slots[r] (int32 [R]; -1 skips the row) of sequence seq[r]
    (default r) of table (int32 [seqs, max_pages]).  rope = (cos, sin), float32
    [rows, dim / 2] each, rotates k and q by row positions[r] (default
    slots[r]).  Returns the rotated q (q_out if given, which may be q), or
    None without q."""
    torch = _torch()
    i32, f32, D = torch.int32, torch.float32, cache.head_dim
    c, t = cache._here(), _table(table)
    kp, ldk = _head_rows(k, "k", cache.kv_heads, D)
    R = k.shape[0]
    vp, ldv = _head_rows(v, "v", cache.kv_heads, D, R)
    sp = _vec(slots, i32, "slots", (R,))
    np_ = _vec(seq, i32, "seq", (R,)) if seq is not None else None
    if seq is None and R > table.shape[0]:
        raise _invalid(f"{R} rows for {table.shape[0]} sequences: seq is needed")
    pp = _vec(positions, i32, "positions", (R,)) if positions is not None else None
    rp = None
    if rope is not None:
        cos, sin = rope
        cp = _ptr(cos, f32, "cos")
        if cos.dim() != 2 or not cos.is_contiguous():
            raise _invalid("cos must be contiguous [rows, dim / 2]")
        rp = ctypes.byref(_Rope(cp, _vec(sin, f32, "sin", cos.shape), cos.shape[0], 2 * cos.shape[1]))
    qp = op = None
    ldq = ldo = hq = 0
    with _on(stream, cache.k, cache.v, cache.score, table, slots, k, v, q, seq, positions, q_out, *(rope or ())):
        if q is not None:
            hq = _heads_of(q, "q", D)
            qp, ldq = _head_rows(q, "q", hq, D, R)
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=f32, device=q.device)
            op, ldo = _head_rows(q_out, "q_out", hq, D, R)
        elif q_out is not None:
            raise _invalid("q_out without q")
        _check(_lib.xt_kv_append(c, t, np_, sp, pp, rp, qp, ldq, hq, op, ldo, kp, ldk, vp, ldv, R,
                                 _stream_ptr(stream)))
    return q_out


def paged_attention(cache, table, lengths, q, seq=None, scale=None, lse=False, accumulate=False, out=None,
                    stream=None):
    """xt_paged_attention: row r of q (float32 [R, q_heads, head_dim] or [R,
    q_heads * head_dim]) attends over the first lengths[r] (int32 [R])
    positions of sequence seq[r] (default r) of table (int32 [seqs,
    max_pages]).  scale defaults to head_dim ** -0.5.  Returns out, shaped as
    q, or (out, lse [R, q_heads]) with lse=True; accumulate=True adds the
    weights to cache.score."""
    torch = _torch()
    i32, f32, D = torch.int32, torch.float32, cache.head_dim
    c, t = cache._here(), _table(table)
    hq = _heads_of(q, "q", D)
    qp, ldq = _head_rows(q, "q", hq, D)
    R = q.shape[0]
    lp = _vec(lengths, i32, "lengths", (R,))
    sp = _vec(seq, i32, "seq", (R,)) if seq is not None else None
    if seq is None and R > table.shape[0]:
        raise _invalid(f"{R} rows for {table.shape[0]} sequences: seq is needed")
    with _on(stream, cache.k, cache.v, cache.score, table, lengths, q, seq, out):
        if out is None:
            out = torch.empty(q.shape, dtype=f32, device=q.device)
        op, ldo = _head_rows(out, "out", hq, D, R)
        l = torch.empty((R, hq), dtype=f32, device=q.device) if lse else None
        _check(_lib.xt_paged_attention(c, t, sp, lp, qp, ldq, hq,
                                       1.0 / math.sqrt(D) if scale is None else float(scale), R, op, ldo,
                                       l.data_ptr() if lse else None, int(bool(accumulate)),
                                       _stream_ptr(stream)))
    return (out, l) if lse else out


def kv_evict(cache, table, lengths, budget, sink=0, recent=0, stream=None):
    """xt_kv_evict: every sequence of table with lengths[b] (int32 [seqs]) >
    budget is cut down to budget positions per key-value head, the first
    `sink`, the last `recent` and those of the highest cache.score between
    them, moved in order to the front of its pages.  Returns (new lengths
    [seqs], kept [seqs, kv_heads, budget]: each one's old position, -1 past
    the new length)."""
    torch = _torch()
    i32 = torch.int32
    c, t = cache._here(), _table(table)
    S = table.shape[0]
    lp = _vec(lengths, i32, "lengths", (S,))
    budget = int(budget)
    if budget < 1:
        raise _invalid("budget must be 1..2^31-1")
    with _on(stream, cache.k, cache.v, cache.score, table, lengths):
        new = torch.empty((S,), dtype=i32, device=table.device)
        kept = torch.empty((S, cache.kv_heads, budget), dtype=i32, device=table.device)
        _check(_lib.xt_kv_evict(c, t, lp, budget, int(sink), int(recent), new.data_ptr(), kept.data_ptr(),
                                _stream_ptr(stream)))
    return new, kept


def token_logprobs(logits, tokens=None, top=0, stream=None):
    """xt_token_logprobs over the rows of logits [M, V] (float32, float16 or
    bfloat16, -inf for masked tokens; rows may be any distance apart).  tokens:
    int32 [M] or [M, T].  Returns (log probabilities shaped as tokens, or
    None; entropy [M]; ids int32 [M, top] of the most likely tokens and their
    log probabilities [M, top], or None, None)."""
    torch = _torch()
    i32, f32 = torch.int32, torch.float32
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise _invalid("logits must be a CUDA (HIP) tensor")
    if logits.dtype not in _dtypes():
        raise _invalid(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise _invalid("logits must be [rows, vocabulary], contiguous within a row")
    xp = _ptr(logits, logits.dtype, "logits")
    (M, V), T, tp, top = logits.shape, 0, None, int(top)
    if tokens is not None:
        tp = _ptr(tokens, i32, "tokens")
        if tokens.dim() not in (1, 2) or tokens.shape[0] != M or not tokens.is_contiguous():
            raise _invalid(f"tokens must be contiguous [{M}] or [{M}, T], got {list(tokens.shape)}")
        T = 1 if tokens.dim() == 1 else tokens.shape[1]
    if not 0 <= top <= 64:
        raise _invalid("top must be 0..64, at most the vocabulary")
    dev = logits.device
    with _on(stream, logits, tokens):
        lp = torch.empty(tokens.shape, dtype=f32, device=dev) if tokens is not None else None
        entropy = torch.empty((M,), dtype=f32, device=dev)
        ids = torch.empty((M, top), dtype=i32, device=dev) if top else None
        best = torch.empty((M, top), dtype=f32, device=dev) if top else None
        _check(_lib.xt_token_logprobs(_dtypes()[logits.dtype], xp, logits.stride(0), M, V, tp, T,
                                      lp.data_ptr() if T else None, entropy.data_ptr(), top,
                                      ids.data_ptr() if top else None, best.data_ptr() if top else None,
                                      _stream_ptr(stream)))
    return lp, entropy, ids, best
