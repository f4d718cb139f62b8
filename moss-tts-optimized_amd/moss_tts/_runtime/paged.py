"""A batch of sequences over a paged key-value cache: new tokens in, and the attention that reads it.

The counterparts, for requests that are served together, of ``pointwise.qk_rope``,
``attention.decode_attention`` and ``attention.prefill_attention``, which serve one request from a cache of its
own.  Head counts come from the tensors: any number of query heads per KV head, heads of 64 or 128, bf16 or fp16.

``keys`` and ``values``: ``[pages, KV heads, page rows, head dim]``; the pages may lie any stride apart (a
view into a larger cache), a page is contiguous.  ``page rows`` is a power of two from 16 to 4096.
``table``: int32 ``[B, W]``; row ``r`` of sequence ``b`` is row ``r % rows`` of page ``table[b, r // rows]``.  An entry
outside ``[0, pages)`` names no page: its rows take no part and nothing is written to them.
``lengths``: int32 ``[B]``, the rows of each sequence with the new tokens' included.
``starts``: int32 ``[B + 1]``, rising from 0: the packed tokens ``starts[b] .. starts[b + 1] - 1`` are the newest ones of
sequence ``b`` and stand at its last positions.  Packed rows from ``starts[B]`` on are padding and left as they are.

Table, lengths and starts are device values, read when the kernels run and not checked by the host: a captured
graph follows them as sequences grow.  Whatever they hold, no access leaves the cache or the packed rows; what they have
to hold for results is the caller's to see to: lengths that the table's row can hold (all three operators take a
longer one as the rows that it holds, so new tokens go to the last of them), starts that rise, and no two new tokens on
one row of a page (sequences may share the pages that they only read).  A row that takes part with values that are not
finite makes what it touches not finite; rows that take no part may hold anything.
"""
from __future__ import annotations

import math

import torch

from . import native
from .w4g32 import _aligned, _apart, _cuda_contig, _require

_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_PAGE_ROWS = tuple(1 << s for s in range(4, 13))
_HEAD_DIMS = (64, 128)


# The checks below read a tensor's shape and strides once and compare plain integers: a call of these operators takes
# the host longer than most of their kernels take the device (28 us with a torch view or a generator per check, of
# which 8 are the launches).  What a check finds wrong is named by the slower functions that end in _refuse.
def _cache_refuse(keys, values, dtype, index):
    for name, t in (("keys", keys), ("values", values)):
        _require(isinstance(t, torch.Tensor) and t.dtype == dtype, f"{name} must be a {dtype} tensor")
        _require(t.is_cuda and t.get_device() == index, f"{name} must be on cuda:{index}")
        _require(t.dim() == 4 and t.shape == keys.shape and t.numel() > 0,
                 "matching [pages, KV heads, page rows, head dim] keys and values required")
        n, kh, rows, d = t.shape
        _require(rows in _PAGE_ROWS, "page rows must be a power of two from 16 to 4096")
        _require(d in _HEAD_DIMS, "head dim must be 64 or 128")
        _require(t.stride(3) == 1 and t.stride(2) == d and (kh == 1 or t.stride(1) == rows * d),
                 f"a page of {name} must be contiguous")
        _require(_aligned(t, 16) and (n == 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= kh * rows * d)),
                 f"{name}: pages must be 16-byte aligned and must not overlap")


class _Cache:
    """A checked cache as numbers: pages, KV heads, page rows, head dim, pointers and page strides, ends."""

    __slots__ = ("pages", "kh", "rows", "d", "k", "v", "ks", "vs", "kend", "vend")

    def __init__(self, keys, values, dtype, index):
        try:
            n, kh, rows, d = shape = keys.shape
            ks, k2, k1, k0 = keys.stride()
            vs, v2, v1, v0 = values.stride()
            k, v = keys.data_ptr(), values.data_ptr()
            page = kh * rows * d
            if n == 1:
                ks = vs = page
            if kh == 1:
                k2 = v2 = rows * d
            ok = (keys.dtype is dtype and values.dtype is dtype and values.shape == shape and page
                  and keys.get_device() == index and values.get_device() == index and rows in _PAGE_ROWS
                  and d in _HEAD_DIMS and k0 == 1 and v0 == 1 and k1 == d and v1 == d and k2 == v2 == rows * d
                  and not ((ks | vs) & 7 or (k | v) & 15) and ks >= page and vs >= page)
        except (AttributeError, ValueError, TypeError):
            ok = False
        if not ok:
            _cache_refuse(keys, values, dtype, index)
            raise ValueError("keys and values are not a paged cache")
        self.pages, self.kh, self.rows, self.d, self.k, self.v, self.ks, self.vs = n, kh, rows, d, k, v, ks, vs
        self.kend, self.vend = k + 2 * ((n - 1) * ks + page), v + 2 * ((n - 1) * vs + page)


def _batch_refuse(table, lengths, starts, rows, index):
    _require(isinstance(table, torch.Tensor) and table.dtype == torch.int32 and table.dim() == 2 and table.numel() > 0,
             "table must be an int32 [B, W] tensor")
    _require(table.is_cuda and table.get_device() == index, f"table must be on cuda:{index}")
    b, w = table.shape
    _require((w == 1 or table.stride(1) == 1) and (b == 1 or table.stride(0) >= w), "a row of table must be contiguous")
    _require(b <= 65535 and w * rows <= 1 << 30, "at most 65535 sequences of 2^30 rows")
    _cuda_contig("lengths", lengths, torch.int32, table.device)
    _require(lengths.numel() == b, "one length a sequence required")
    if starts is not None:
        _cuda_contig("starts", starts, torch.int32, table.device)
        _require(starts.numel() == b + 1, "starts must hold one value a sequence and the end")


def _batch(table, lengths, starts, rows, index):
    """(B, W, table stride, pointers of table, lengths and starts) of a checked batch."""
    try:
        b, w = table.shape
        ts, t1 = table.stride()
        if b == 1:
            ts = w
        ok = (table.dtype is torch.int32 and lengths.dtype is torch.int32 and table.get_device() == index
              and lengths.get_device() == index and (t1 == 1 or w == 1) and ts >= w > 0 and 0 < b <= 65535
              and w * rows <= 1 << 30 and lengths.numel() == b and lengths.is_contiguous()
              and (starts is None or (starts.dtype is torch.int32 and starts.get_device() == index
                                      and starts.numel() == b + 1 and starts.is_contiguous())))
    except (AttributeError, ValueError):
        ok = False
    if not ok:
        _batch_refuse(table, lengths, starts, rows, index)
        raise ValueError("table, lengths and starts do not describe a batch")
    return b, w, ts, table.data_ptr(), lengths.data_ptr(), None if starts is None else starts.data_ptr()


def _query(q):
    """(tokens, heads, head dim, row stride, device index) of checked queries."""
    _require(isinstance(q, torch.Tensor) and q.dtype in _TYPES, "q must be a bf16 or fp16 tensor")
    index = q.get_device()
    _require(index >= 0 and q.dim() == 3 and q.numel() > 0, "q must be a CUDA (HIP) tensor [tokens, heads, head dim]")
    n, h, d = q.shape
    stride, s1, s0 = q.stride()
    if n == 1:
        stride = h * d
    _require((s0 == 1 or d == 1) and (s1 == d or h == 1), "a row of q must be contiguous")
    _require(stride >= h * d and not (stride & 7 or q.data_ptr() & 15),
             "q: rows must be 16-byte aligned and must not overlap")
    return n, h, d, stride, index


def _norms_and_tables(q_weight, k_weight, cos, sin, d: int, dtype, index):
    """(q weight, k weight, cos, sin pointers, whether the tables are fp32, their rows), checked."""
    try:
        rows, width = shape = cos.shape
        kind = cos.dtype
        c, s = cos.data_ptr(), sin.data_ptr()
        qw = kw = None
        ok = ((kind is torch.float32 or kind is dtype) and sin.dtype is kind and sin.shape == shape and width == d
              and 0 < rows < 1 << 31 and cos.get_device() == index == sin.get_device() and cos.is_contiguous()
              and sin.is_contiguous() and not (c | s) & 15)
        if q_weight is None or k_weight is None:
            ok = ok and q_weight is k_weight
        else:
            qw, kw = q_weight.data_ptr(), k_weight.data_ptr()
            ok = (ok and q_weight.dtype is dtype and k_weight.dtype is dtype and q_weight.numel() == d == k_weight.numel()
                  and q_weight.get_device() == index == k_weight.get_device() and q_weight.is_contiguous()
                  and k_weight.is_contiguous() and not (qw | kw) & 15)
    except (AttributeError, ValueError):
        ok = False
    if ok:
        return qw, kw, c, s, int(kind is torch.float32), rows
    _require((q_weight is None) == (k_weight is None), "both head-norm weights or none")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None:
            _require(isinstance(t, torch.Tensor) and t.dtype == dtype and t.get_device() == index and t.numel() == d
                     and t.is_contiguous() and not t.data_ptr() & 15,
                     f"{name} must hold {d} {dtype} values on cuda:{index}, contiguous and 16-byte aligned")
    _require(isinstance(cos, torch.Tensor) and cos.dtype in (torch.float32, dtype), f"cos must be a float32 or {dtype} tensor")
    for name, t in (("cos", cos), ("sin", sin)):
        _require(isinstance(t, torch.Tensor) and t.dtype == cos.dtype and t.dim() == 2 and t.shape == cos.shape
                 and t.shape[1] == d and t.shape[0] > 0 and t.get_device() == index and t.is_contiguous()
                 and not t.data_ptr() & 15,
                 f"{name} must be a {cos.dtype} [positions, {d}] table on cuda:{index}, contiguous and 16-byte aligned, "
                 "as long as the other")
    raise ValueError("the head-norm weights and tables do not fit")


def _scale(scale, d: int) -> float:
    if scale is None:
        return d ** -0.5
    scale = float(scale)
    _require(scale == scale and abs(scale) != float("inf"), "scale must be finite")
    return scale


def _batch_spans(b, w, ts, table, lengths, starts):
    """What a batch's tensors cover, as (first, end): results written over them would change the work under the kernels."""
    spans = (table, table + 4 * ((b - 1) * ts + w)), (lengths, lengths + 4 * b)
    return spans if starts is None else spans + ((starts, starts + 4 * b + 4),)


def _workspace(ws, nbytes: int, like: torch.Tensor, out: torch.Tensor, spans):
    """A new workspace of ``nbytes`` (None for none), or the caller's, checked."""
    if ws is None:
        return like.new_empty(nbytes // 4, dtype=torch.float32) if nbytes else None
    _cuda_contig("ws", ws, torch.float32, like.device)
    _require(4 * ws.numel() >= nbytes and not ws.data_ptr() & 15, "workspace too small or not 16-byte aligned")
    at = out.data_ptr()
    _apart("ws", ws, (at, at + 2 * out.numel()), *spans)
    return ws


def _output(out, shape, like: torch.Tensor, index: int, spans) -> torch.Tensor:
    """A new output (which shares no memory with anything), or the caller's, checked."""
    if out is None:
        return like.new_empty(shape)
    if not (isinstance(out, torch.Tensor) and out.dtype is like.dtype and out.get_device() == index and out.is_contiguous()):
        _cuda_contig("out", out, like.dtype, like.device)
    if out.shape != shape:
        _require(out.numel() == math.prod(shape), f"out must hold {' x '.join(map(str, shape))} values")
        out = out.view(shape)
    _require(not out.data_ptr() & 15, "out must be 16-byte aligned")
    _apart("out", out, *spans)
    return out


def qk_rope(qkv: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, cos: torch.Tensor,
            sin: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
            eps: float, *, starts: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """q/k head RMSNorm + rotary embedding of ``T`` packed tokens, whose K and V rows are written to their pages.

    ``qkv`` ``[T, (query heads + 2 KV heads) * head dim]`` (q | k | v; rows may lie apart), head-norm weights ``[head
    dim]`` (both None: no norm), ``cos`` / ``sin`` ``[positions, head dim]`` tables in ``qkv``'s type or fp32.  Without
    ``starts`` every sequence has one token.  Returns ``q`` ``[T, query heads, head dim]``.  The arithmetic is fp32 up
    to one rounding, where ``pointwise.qk_rope`` rounds after every step.  A token at a negative position (more tokens
    than its length) or without a page is written to no row; a position behind the tables takes their last row."""
    _require(isinstance(qkv, torch.Tensor) and qkv.dtype in _TYPES, "qkv must be a bf16 or fp16 tensor")
    index, dtype = qkv.get_device(), qkv.dtype
    _require(index >= 0 and qkv.dim() == 2 and qkv.numel() > 0, "qkv must be a CUDA (HIP) tensor [tokens, width]")
    tokens, width = qkv.shape
    stride, s0 = qkv.stride()
    if tokens == 1:
        stride = width
    at = qkv.data_ptr()
    _require(s0 == 1 or width == 1, "a row of qkv must be contiguous")
    _require(stride >= width and not (stride & 7 or at & 15), "qkv: rows must be 16-byte aligned and must not overlap")
    c = _Cache(keys, values, dtype, index)
    kh, d = c.kh, c.d
    b, w, table_stride, table_at, lengths_at, starts_at = batch = _batch(table, lengths, starts, c.rows, index)
    qh = width // d - 2 * kh
    _require(width % d == 0 and 0 < qh <= 1024 and qh % kh == 0,
             "qkv must hold a multiple of the KV heads as query heads, then the keys and the values")
    _require(starts is not None or tokens == b, "without starts, one token a sequence required")
    norms = _norms_and_tables(q_weight, k_weight, cos, sin, d, dtype, index)
    _require(eps >= 0, "eps must not be negative")
    _require(tokens < 1 << 24, "fewer than 2^24 packed tokens required")
    span = (at, at + 2 * ((tokens - 1) * stride + width))
    _require((c.kend <= span[0] or span[1] <= c.k) and (c.vend <= span[0] or span[1] <= c.v),
             "qkv must not overlap the cache")
    if c.k < c.vend and c.v < c.kend:  # interleaved: the keys of a page lie between the values of two
        page, step = 2 * kh * c.rows * d, 2 * c.ks
        _require(c.ks == c.vs and page <= (c.v - c.k) % step <= step - page, "keys and values must not share memory")
    spans = ()
    if out is not None:
        qw, kw, cos_at, sin_at, f32, rows = norms
        size = rows * d * (4 if f32 else 2)
        spans = (span, (c.k, c.kend), (c.v, c.vend), (cos_at, cos_at + size), (sin_at, sin_at + size), *_batch_spans(*batch))
        if qw is not None:
            spans += (qw, qw + 2 * d), (kw, kw + 2 * d)
    q = _output(out, (tokens, qh, d), qkv, index, spans)
    native.call_on(qkv, "moss_paged_qk_rope", at, stride, *norms, q.data_ptr(), c.k, c.v, c.ks, c.vs, c.pages, c.rows,
                   table_at, table_stride, lengths_at, starts_at, b, w, tokens, qh, kh, d, eps, _TYPES[dtype])
    return q


def decode_workspace(q: torch.Tensor, keys: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """A workspace for :func:`decode_attention` calls of these shapes; calls that may overlap (other streams,
    graphs that replay side by side) need one each."""
    nbytes = native.lib().moss_paged_decode_workspace_bytes(table.shape[0], table.shape[1], keys.shape[2], q.shape[1],
                                                            keys.shape[1], keys.shape[3])
    return torch.empty(nbytes // 4, dtype=torch.float32, device=q.device)


def decode_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor,
                     lengths: torch.Tensor, *, scale: float | None = None, out: torch.Tensor | None = None,
                     ws: torch.Tensor | None = None) -> torch.Tensor:
    """One new token per sequence: ``q`` ``[B, query heads, head dim]`` (rows may lie apart) against the
    ``lengths[b]`` rows of each sequence, the new token's own among them; ``scale`` defaults to head dim ** -0.5.
    Returns ``[B, query heads * head dim]``; a sequence without rows gives zeros."""
    n, qh, hd, stride, index = _query(q)
    c = _Cache(keys, values, q.dtype, index)
    kh, d = c.kh, c.d
    b, w, table_stride, table_at, lengths_at, _ = batch = _batch(table, lengths, None, c.rows, index)
    _require(n == b and hd == d and qh % kh == 0 and qh <= 1024, "q must be [B, a multiple of the KV heads, head dim]")
    at = q.data_ptr()
    spans = ()
    if out is not None or ws is not None:
        spans = (at, at + 2 * ((n - 1) * stride + qh * d)), (c.k, c.kend), (c.v, c.vend), *_batch_spans(*batch)
    out = _output(out, (b, qh * d), q, index, spans)
    nbytes = native.lib().moss_paged_decode_workspace_bytes(b, w, c.rows, qh, kh, d)
    ws = _workspace(ws, nbytes, q, out, spans)
    native.call_on(q, "moss_paged_decode_attention", at, stride, c.k, c.v, c.ks, c.vs, c.pages, c.rows, table_at,
                   table_stride, lengths_at, b, w, qh, kh, d, _scale(scale, d), out.data_ptr(), ws.data_ptr(),
                   nbytes, _TYPES[q.dtype])
    return out


def prompt_workspace(q: torch.Tensor, keys: torch.Tensor, table: torch.Tensor) -> torch.Tensor | None:
    """A workspace for :func:`prompt_attention` calls of these shapes (None: none needed); calls that may overlap need
    one each."""
    nbytes = native.lib().moss_paged_prompt_workspace_bytes(table.shape[0], table.shape[1], keys.shape[2], q.shape[0],
                                                            q.shape[1], keys.shape[1], keys.shape[3])
    return torch.empty(nbytes // 4, dtype=torch.float32, device=q.device) if nbytes else None


def prompt_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor,
                     lengths: torch.Tensor, starts: torch.Tensor, *, scale: float | None = None,
                     out: torch.Tensor | None = None, ws: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed new tokens whose K and V rows are in the pages already: ``q`` ``[T, query heads,
    head dim]`` (rows may lie apart); each token attends its sequence's rows up to its own position, the cached
    ones before the new among them.  ``scale`` defaults to head dim ** -0.5.  Returns ``[T, query heads * head
    dim]``; a token without a visible row gives zeros."""
    n, qh, hd, stride, index = _query(q)
    c = _Cache(keys, values, q.dtype, index)
    kh, d = c.kh, c.d
    _require(starts is not None, "starts required")
    b, w, table_stride, table_at, lengths_at, starts_at = batch = _batch(table, lengths, starts, c.rows, index)
    _require(hd == d and qh % kh == 0 and qh <= 1024, "q must be [tokens, a multiple of the KV heads, head dim]")
    _require(n <= 1 << 20, "at most 2^20 packed tokens")
    at = q.data_ptr()
    spans = ()
    if out is not None or ws is not None:
        spans = (at, at + 2 * ((n - 1) * stride + qh * d)), (c.k, c.kend), (c.v, c.vend), *_batch_spans(*batch)
    out = _output(out, (n, qh * d), q, index, spans)
    nbytes = native.lib().moss_paged_prompt_workspace_bytes(b, w, c.rows, n, qh, kh, d)
    ws = _workspace(ws, nbytes, q, out, spans)
    native.call_on(q, "moss_paged_prompt_attention", at, stride, c.k, c.v, c.ks, c.vs, c.pages, c.rows, table_at,
                   table_stride, lengths_at, starts_at, b, w, n, qh, kh, d, _scale(scale, d),
                   out.data_ptr(), None if ws is None else ws.data_ptr(), nbytes, _TYPES[q.dtype])
    return out
