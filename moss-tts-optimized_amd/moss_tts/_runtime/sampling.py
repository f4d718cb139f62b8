"""Decode-step sampling on the gfx950 library.

``sample_topk(logits, temperature=1.7, top_k=25, top_p=0.8)`` keeps the reference's signature and
meaning (``src/moss_tts/_runtime/llm.py:10-19``); the random draw comes from a counter-based
Philox4x32-10 keyed by ``seed`` and indexed by the device-side ``position`` and the row, so a
captured decode graph samples fresh values at every position.  The key is read from a device
buffer when the kernel runs (``seed_buffer``), so each request can set its own seed without
recapturing.  ``compose_next_ids`` is the token logic of the reference's ``_decode``
(``llm.py:280-287``).  ``advance_step`` is the host loop's per-step update
(``src/moss_tts/_runtime/streaming.py:107-112``) on the device, so several decode steps can be
captured in one graph (``src/moss_tts/_runtime/first_audio_graph.py:14-29``).
"""
from __future__ import annotations

import torch

from . import native
from .w4g32 import _apart, _cuda_contig, _require

MAX_TOP_K = 64
MAX_VOCAB = 2048
_U64 = 0xFFFFFFFFFFFFFFFF


def seed_value(seed: int) -> int:
    """A 64-bit seed as the signed int64 whose bits the sampler reads as its Philox key."""
    _require(isinstance(seed, int), "seed must be an int")
    u = int(seed) & _U64
    return u - (1 << 64) if u >= 1 << 63 else u


def seed_buffer(seed: int, device) -> torch.Tensor:
    """A device int64 ``[1]`` holding ``seed``'s 64 bits: the sampler's key buffer."""
    return torch.full((1,), seed_value(seed), dtype=torch.int64, device=device)


def sample_topk(logits: torch.Tensor, temperature: float = 1.7, top_k: int = 25, top_p: float = 0.8, *,
                seed: int | torch.Tensor = 0, position: torch.Tensor | None = None, salt: int = 0,
                vocab: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 logits ``[rows, stride]`` (or ``[stride]``) -> int64 indices ``[rows]`` into the first
    ``vocab`` entries of each row.  ``seed``: an int, or a device int64 ``[1]`` buffer read when the
    kernel runs (what a captured graph uses)."""
    _cuda_contig("logits", logits, torch.bfloat16)
    rows = 1 if logits.dim() == 1 else logits.shape[0]
    stride = logits.shape[-1]
    vocab = stride if vocab is None else int(vocab)
    _require(0 < vocab <= min(stride, MAX_VOCAB), f"vocab must be in [1, min(stride, {MAX_VOCAB})]")
    if temperature > 0:
        _require(1 <= top_k <= min(MAX_TOP_K, vocab), f"top_k must be in [1, min({MAX_TOP_K}, vocab)]")
    if position is None:
        position = torch.zeros(1, dtype=torch.int64, device=logits.device)
    _cuda_contig("position", position, torch.int64, logits.device)
    _require(position.numel() == 1, "position holds one value")
    if not isinstance(seed, torch.Tensor):
        seed = seed_buffer(seed, logits.device)
    _cuda_contig("seed", seed, torch.int64, logits.device)
    _require(seed.numel() == 1, "seed holds one value")
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    else:
        _cuda_contig("out", out, torch.int64, logits.device)
        _require(out.numel() == rows, f"out must hold {rows} indices")
    native.call("moss_sample_topk", native.ptr(logits), rows, stride, vocab, float(temperature), int(top_k),
                float(top_p), native.ptr(seed), native.ptr(position), int(salt), native.ptr(out),
                native.stream_of(logits))
    return out


def _sample_set(logits, temperature, top_k, top_p, vocab, out):
    _cuda_contig("logits", logits, torch.bfloat16)
    rows = 1 if logits.dim() == 1 else logits.shape[0]
    stride = logits.shape[-1]
    vocab = stride if vocab is None else int(vocab)
    _require(0 < vocab <= min(stride, MAX_VOCAB), f"vocab must be in [1, min(stride, {MAX_VOCAB})]")
    if temperature > 0:
        _require(1 <= top_k <= min(MAX_TOP_K, vocab), f"top_k must be in [1, min({MAX_TOP_K}, vocab)]")
    _cuda_contig("out", out, torch.int64, logits.device)
    _require(out.numel() == rows, f"out must hold {rows} indices")
    return (native.ptr(logits), rows, stride, vocab, float(temperature), int(top_k), float(top_p))


def sample_topk_pair(a: dict, b: dict, *, seed: torch.Tensor, position: torch.Tensor) -> None:
    """Two :func:`sample_topk` calls sharing ``seed`` and ``position`` in one launch (the decode
    step's text row and audio rows, ``llm.py:280,284``); each of ``a`` and ``b`` holds ``logits``,
    ``temperature``, ``top_k``, ``top_p``, ``salt``, ``out`` and optionally ``vocab``.  The outputs
    equal the two separate calls'."""
    sets = []
    for d in (a, b):
        head = _sample_set(d["logits"], d["temperature"], d["top_k"], d["top_p"], d.get("vocab"), d["out"])
        _require(d["logits"].device == a["logits"].device, "both sets on one device")
        sets.append(head + (int(d["salt"]), native.ptr(d["out"])))
    dev = a["logits"].device
    for name, t in (("seed", seed), ("position", position)):
        _cuda_contig(name, t, torch.int64, dev)
        _require(t.numel() == 1, f"{name} holds one value")
    native.call("moss_sample_topk_pair", *sets[0], *sets[1], native.ptr(seed), native.ptr(position),
                native.stream_of(a["logits"]))


_SAMPLE_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_SAMPLE_VOCAB = 1 << 19
MAX_SAMPLE_ROWS = 1 << 21


def _setting(name: str, value, rows: int, dtype: torch.dtype, device):
    """(pointer, value) of one sampling setting: a device tensor with one value a row, or a number for all."""
    if isinstance(value, torch.Tensor):
        _cuda_contig(name, value, dtype, device)
        _require(value.numel() == rows, f"{name} must hold one value a row")
        return value.data_ptr(), 0
    _require(isinstance(value, (int, float)) and not isinstance(value, bool) and value == value,
             f"{name} must be a number or a tensor")
    return None, value


def sample_workspace(rows: int, vocab: int, device) -> torch.Tensor | None:
    """A workspace for :func:`sample` calls of up to these sizes (None: none needed); calls that may overlap need one
    each."""
    nbytes = native.lib().moss_sample_rows_workspace_bytes(rows, vocab)
    return torch.empty(nbytes // 4, dtype=torch.float32, device=device) if nbytes else None


def sample(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: float | torch.Tensor = 1.0,
           top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0, min_p: float | torch.Tensor = 0.0,
           vocab: int | None = None, out: torch.Tensor | None = None, ws: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 / fp16 / fp32 logits ``[rows, entries]`` (rows any stride apart) -> int64 indices ``[rows]`` into the
    first ``vocab`` entries, drawn by the given numbers ``uniform`` fp32 ``[rows]`` in [0, 1).

    Kept are the ``top_k`` largest (0: all; of equal logits the lower index first), of those the ones whose
    predecessors hold at most the share ``top_p`` of the kept probability (1: all), and those at least
    ``min_p`` times as probable as the largest.  The draw inverts the cumulative distribution of the kept entries
    in index order; entries less probable than 2^-45 of the largest weigh nothing.  ``temperature`` <= 0 takes the first
    of the largest logits.  NaN counts as ``-inf``; a row with nothing above ``-inf`` gives -1.  Each setting is a number, or a device tensor with one value a row
    (fp32; ``top_k`` int32) that is read when the kernel runs, so a captured graph serves rows with settings of
    their own.  Where :func:`sample_topk` draws its own numbers over at most 2048 entries, this takes the
    caller's, over up to 2^19.  ``ws``: a :func:`sample_workspace`, for callers that keep one; neither it nor ``out``
    may share memory with another argument."""
    _require(isinstance(logits, torch.Tensor) and logits.dtype in _SAMPLE_TYPES, "logits must be a bf16, fp16 or fp32 tensor")
    _require(logits.is_cuda, "logits must be a CUDA (HIP) tensor")
    _require(logits.dim() == 2 and logits.shape[0] > 0 and logits.shape[1] > 0, "logits must be [rows, entries]")
    rows, entries = logits.shape
    _require(rows <= MAX_SAMPLE_ROWS, f"at most {MAX_SAMPLE_ROWS} rows")
    _require(entries == 1 or logits.stride(1) == 1, "a row's logits must be contiguous")
    stride = logits.stride(0) if rows > 1 else entries
    _require(stride >= entries, "rows must not overlap")
    vocab = entries if vocab is None else int(vocab)
    _require(0 < vocab <= min(entries, MAX_SAMPLE_VOCAB), f"vocab must be in [1, min(entries, {MAX_SAMPLE_VOCAB})]")
    dev = logits.device
    _cuda_contig("uniform", uniform, torch.float32, dev)
    _require(uniform.numel() == rows, "uniform must hold one number a row")
    t_ptr, t = _setting("temperature", temperature, rows, torch.float32, dev)
    k_ptr, k = _setting("top_k", top_k, rows, torch.int32, dev)
    p_ptr, p = _setting("top_p", top_p, rows, torch.float32, dev)
    m_ptr, m = _setting("min_p", min_p, rows, torch.float32, dev)
    _require(int(k) == k and 0 <= k < 1 << 31, "top_k must be a non-negative integer")
    _require(0 <= p and 0 <= m <= 1, "top_p must not be negative, min_p must lie in [0, 1]")
    if out is not None or ws is not None:  # memory of the caller's, which must be nobody else's: (first, end) of the rest
        at = logits.data_ptr()
        spans = [(first, first + 4 * rows) for first in (uniform.data_ptr(), t_ptr, k_ptr, p_ptr, m_ptr) if first is not None]
        spans.append((at, at + ((rows - 1) * stride + entries) * logits.element_size()))
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=dev)
    else:
        _cuda_contig("out", out, torch.int64, dev)
        _require(out.numel() == rows, f"out must hold {rows} indices")
        _apart("out", out, *spans)
    if ws is None:
        ws = sample_workspace(rows, vocab, dev)
    else:
        _cuda_contig("ws", ws, torch.float32, dev)
        _require(4 * ws.numel() >= native.lib().moss_sample_rows_workspace_bytes(rows, vocab) and ws.data_ptr() % 16 == 0,
                 "workspace too small or not 16-byte aligned")
        _apart("ws", ws, (out.data_ptr(), out.data_ptr() + 8 * rows), *spans)
    native.call_on(logits, "moss_sample_rows", logits.data_ptr(), _SAMPLE_TYPES[logits.dtype], rows, stride, vocab,
                   uniform.data_ptr(), t_ptr, float(t), k_ptr, int(k), p_ptr, float(p), m_ptr, float(m), out.data_ptr(),
                   None if ws is None else ws.data_ptr(), 0 if ws is None else 4 * ws.numel())
    return out


def compose_next_ids(text_index: torch.Tensor, audio_index: torch.Tensor, text_ids: torch.Tensor,
                     audio_length: torch.Tensor, delay_length: torch.Tensor, *, delay_slot_id: int,
                     audio_end_id: int, pad_code: int = 1024, out: torch.Tensor | None = None) -> torch.Tensor:
    """int64 ``[1 + channels]``: the next text token and audio codes (``llm.py:280-287``)."""
    dev = audio_index.device
    for name, t in (("text_index", text_index), ("audio_index", audio_index), ("text_ids", text_ids),
                    ("audio_length", audio_length), ("delay_length", delay_length)):
        _cuda_contig(name, t, torch.int64, dev)
    _require(text_ids.numel() == 2, "text_ids holds the gen-slot and delay-slot ids")
    channels = audio_index.numel()
    _require(0 < channels <= 64, "at most 64 channels")
    if out is None:
        out = torch.empty(1 + channels, dtype=torch.int64, device=dev)
    native.call("moss_compose_next_ids", native.ptr(text_index), native.ptr(audio_index), native.ptr(text_ids),
                native.ptr(audio_length), native.ptr(delay_length), int(delay_slot_id), int(audio_end_id),
                channels, int(pad_code), native.ptr(out), native.stream_of(audio_index))
    return out


def advance_step(next_ids: torch.Tensor, ids: torch.Tensor, position: torch.Tensor, audio_length: torch.Tensor,
                 delay_length: torch.Tensor, *, step: int = 0, history: torch.Tensor | None = None,
                 status: torch.Tensor | None = None, audio_start_id: int, gen_slot_id: int,
                 delay_slot_id: int) -> None:
    """In place: ``ids <- next_ids`` (and ``history[step]``), position + 1, the audio length and delay
    counter advanced by the text token ``next_ids[0]``; ``status = (text, length, delay, position)``."""
    dev = next_ids.device
    for name, t in (("next_ids", next_ids), ("ids", ids), ("position", position), ("audio_length", audio_length),
                    ("delay_length", delay_length)):
        _cuda_contig(name, t, torch.int64, dev)
    width = next_ids.numel()
    _require(0 < width <= 64 and ids.numel() == width, "ids and next_ids must hold the same 1..64 ids")
    _require(next_ids.data_ptr() != ids.data_ptr(), "next_ids and ids must be distinct buffers")
    for name, t in (("position", position), ("audio_length", audio_length), ("delay_length", delay_length)):
        _require(t.numel() == 1, f"{name} holds one value")
    if history is not None:
        _cuda_contig("history", history, torch.int64, dev)
        _require(history.dim() == 2 and history.shape[1] == width and 0 <= step < history.shape[0],
                 "history must be [steps, width] with 0 <= step < steps")
    else:
        _require(step >= 0, "step must be non-negative")
    if status is not None:
        _cuda_contig("status", status, torch.int64, dev)
        _require(status.numel() == 4, "status holds 4 values")
    native.call("moss_advance_step", native.ptr(next_ids), native.ptr(ids), native.ptr(position),
                native.ptr(audio_length), native.ptr(delay_length), native.ptr(history) if history is not None else None,
                native.ptr(status) if status is not None else None, int(step), width, int(audio_start_id),
                int(gen_slot_id), int(delay_slot_id), native.stream_of(next_ids))
