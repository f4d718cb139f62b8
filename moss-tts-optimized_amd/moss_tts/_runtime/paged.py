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
graph follows them as sequences grow.  Whatever they hold, no access leaves the cache or the packed rows.
"""
from __future__ import annotations

import torch

from . import native
from .w4g32 import _aligned, _cuda_contig, _require

_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_PAGE_ROWS = tuple(1 << s for s in range(4, 13))


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    def end(t):
        return t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()

    return a.data_ptr() < end(b) and b.data_ptr() < end(a)


def _pages(keys: torch.Tensor, values: torch.Tensor, dtype: torch.dtype, dev):
    """(KV heads, page rows, head dim) of a checked cache."""
    for name, t in (("keys", keys), ("values", values)):
        _require(isinstance(t, torch.Tensor) and t.dtype == dtype, f"{name} must be a {dtype} tensor")
        _require(t.is_cuda and t.device == dev, f"{name} must be on {dev}")
        _require(t.dim() == 4 and t.shape == keys.shape and t.numel() > 0,
                 "matching [pages, KV heads, page rows, head dim] keys and values required")
        n, kh, rows, d = t.shape
        _require(t.stride(3) == 1 and (rows == 1 or t.stride(2) == d) and (kh == 1 or t.stride(1) == rows * d),
                 f"a page of {name} must be contiguous")
        _require(_aligned(t, 16) and (n == 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= kh * rows * d)),
                 f"{name}: pages must be 16-byte aligned and must not overlap")
    _require(rows in _PAGE_ROWS, "page rows must be a power of two from 16 to 4096")
    _require(d in (64, 128), "head dim must be 64 or 128")
    return kh, rows, d


def _page_strides(keys: torch.Tensor, values: torch.Tensor):
    page = keys.shape[1] * keys.shape[2] * keys.shape[3]
    return tuple(t.stride(0) if t.shape[0] > 1 else page for t in (keys, values))


def _batch(table: torch.Tensor, lengths: torch.Tensor, starts, rows: int, dev):
    """(B, W, table stride) of a checked batch."""
    _require(isinstance(table, torch.Tensor) and table.dtype == torch.int32 and table.dim() == 2 and table.numel() > 0,
             "table must be an int32 [B, W] tensor")
    _require(table.is_cuda and table.device == dev, f"table must be on {dev}")
    b, w = table.shape
    stride = table.stride(0) if b > 1 else w
    _require((w == 1 or table.stride(1) == 1) and stride >= w, "a row of table must be contiguous")
    _require(b <= 65535 and w * rows <= 1 << 30, "at most 65535 sequences of 2^30 rows")
    _cuda_contig("lengths", lengths, torch.int32, dev)
    _require(lengths.numel() == b, "one length a sequence required")
    if starts is not None:
        _cuda_contig("starts", starts, torch.int32, dev)
        _require(starts.numel() == b + 1, "starts must hold one value a sequence and the end")
    return b, w, stride


def _heads(name: str, t: torch.Tensor):
    """Row stride of ``[rows, heads, d]`` (or ``[rows, width]``) whose rows are contiguous, 16-byte aligned and apart."""
    width = t[0].numel()
    _require(t[0].is_contiguous(), f"a row of {name} must be contiguous")
    stride = t.stride(0) if t.shape[0] > 1 else width
    _require(stride >= width and stride % 8 == 0 and _aligned(t, 16), f"{name}: rows must be 16-byte aligned and must not overlap")
    return stride


def _query(q: torch.Tensor):
    _require(isinstance(q, torch.Tensor) and q.dtype in _TYPES, "q must be a bf16 or fp16 tensor")
    _require(q.is_cuda and q.dim() == 3 and q.numel() > 0, "q must be a CUDA (HIP) tensor [tokens, heads, head dim]")
    return _heads("q", q)


def _scale(scale, d: int) -> float:
    scale = d ** -0.5 if scale is None else float(scale)
    _require(scale == scale and abs(scale) != float("inf"), "scale must be finite")
    return scale


def _output(out, shape, like: torch.Tensor, *others) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    _cuda_contig("out", out, like.dtype, like.device)
    _require(out.numel() == shape[0] * shape[1] and _aligned(out, 16), f"out must hold {shape[0]} x {shape[1]} values, 16-byte aligned")
    _require(not any(_overlap(out, t) for t in (like, *others)), "out must not overlap an input")
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
    _require(qkv.is_cuda and qkv.dim() == 2 and qkv.numel() > 0, "qkv must be a CUDA (HIP) tensor [tokens, width]")
    dev, dtype = qkv.device, qkv.dtype
    qkv_stride = _heads("qkv", qkv)
    kh, rows, d = _pages(keys, values, dtype, dev)
    b, w, table_stride = _batch(table, lengths, starts, rows, dev)
    tokens, width = qkv.shape
    qh = width // d - 2 * kh
    _require(width % d == 0 and qh > 0 and qh % kh == 0 and qh <= 1024,
             "qkv must hold a multiple of the KV heads as query heads, then the keys and the values")
    _require(starts is not None or tokens == b, "without starts, one token a sequence required")
    _require((q_weight is None) == (k_weight is None), "both head-norm weights or none")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None:
            _cuda_contig(name, t, dtype, dev)
            _require(t.numel() == d and _aligned(t, 16), f"{name} must hold {d} values, 16-byte aligned")
    _require(isinstance(cos, torch.Tensor) and cos.dtype in (dtype, torch.float32), f"cos must be {dtype} or float32")
    for name, t in (("cos", cos), ("sin", sin)):
        _cuda_contig(name, t, cos.dtype, dev)
        _require(t.dim() == 2 and t.shape == cos.shape and t.shape[0] > 0 and t.shape[1] == d and _aligned(t, 16),
                 f"{name} must be a [positions, {d}] table, 16-byte aligned")
    _require(eps >= 0, "eps must not be negative")
    _require(tokens < 1 << 31 and cos.shape[0] < 1 << 31, "too many tokens or positions")
    q = _output(out, (tokens, qh * d), qkv, keys, values).view(tokens, qh, d)
    for t in (keys, values):
        _require(not _overlap(t, qkv), "qkv must not overlap the cache")
    native.call_on(qkv, "moss_paged_qk_rope", qkv.data_ptr(), qkv_stride, None if q_weight is None else q_weight.data_ptr(),
                   None if k_weight is None else k_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                   int(cos.dtype == torch.float32), cos.shape[0], q.data_ptr(), keys.data_ptr(), values.data_ptr(),
                   *_page_strides(keys, values), keys.shape[0], rows, table.data_ptr(), table_stride, lengths.data_ptr(),
                   None if starts is None else starts.data_ptr(), b, w, tokens, qh, kh, d, float(eps), _TYPES[dtype])
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
    q_stride = _query(q)
    dev = q.device
    kh, rows, d = _pages(keys, values, q.dtype, dev)
    b, w, table_stride = _batch(table, lengths, None, rows, dev)
    qh = q.shape[1]
    _require(q.shape[0] == b and q.shape[2] == d and qh % kh == 0 and qh <= 1024,
             "q must be [B, a multiple of the KV heads, head dim]")
    scale = _scale(scale, d)
    if ws is None:
        ws = decode_workspace(q, keys, table)
    else:
        _cuda_contig("ws", ws, torch.float32, dev)
        _require(_aligned(ws, 16), "ws must be 16-byte aligned")
    out = _output(out, (b, qh * d), q, keys, values)
    _require(4 * ws.numel() >= native.lib().moss_paged_decode_workspace_bytes(b, w, rows, qh, kh, d), "workspace too small")
    _require(not any(_overlap(ws, t) for t in (q, out, keys, values)), "the workspace must not overlap the tensors")
    native.call_on(q, "moss_paged_decode_attention", q.data_ptr(), q_stride, keys.data_ptr(), values.data_ptr(),
                   *_page_strides(keys, values), keys.shape[0], rows, table.data_ptr(), table_stride, lengths.data_ptr(),
                   b, w, qh, kh, d, scale, out.data_ptr(), ws.data_ptr(), 4 * ws.numel(), _TYPES[q.dtype])
    return out


def prompt_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor,
                     lengths: torch.Tensor, starts: torch.Tensor, *, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed new tokens whose K and V rows are in the pages already: ``q`` ``[T, query heads,
    head dim]`` (rows may lie apart); each token attends its sequence's rows up to its own position, the cached
    ones before the new among them.  ``scale`` defaults to head dim ** -0.5.  Returns ``[T, query heads * head
    dim]``; a token without a visible row gives zeros."""
    q_stride = _query(q)
    dev = q.device
    kh, rows, d = _pages(keys, values, q.dtype, dev)
    _require(starts is not None, "starts required")
    b, w, table_stride = _batch(table, lengths, starts, rows, dev)
    tokens, qh = q.shape[:2]
    _require(q.shape[2] == d and qh % kh == 0 and qh <= 1024, "q must be [tokens, a multiple of the KV heads, head dim]")
    _require(tokens <= 1 << 20, "at most 2^20 packed tokens")
    scale = _scale(scale, d)
    out = _output(out, (tokens, qh * d), q, keys, values)
    native.call_on(q, "moss_paged_prompt_attention", q.data_ptr(), q_stride, keys.data_ptr(), values.data_ptr(),
                   *_page_strides(keys, values), keys.shape[0], rows, table.data_ptr(), table_stride, lengths.data_ptr(),
                   starts.data_ptr(), b, w, tokens, qh, kh, d, scale, out.data_ptr(), _TYPES[q.dtype])
    return out
