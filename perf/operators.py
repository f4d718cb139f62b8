"""Serving a batch of requests from a paged key-value cache: its operators as cases that can be timed and compared.

Four operators: the q/k head norm, rotary embedding and page write of new tokens (``paged.qk_rope``), the
attention of one new token per sequence (``paged.decode_attention``), the causal attention of packed prompts
(``paged.prompt_attention``), and the draw of the next tokens (``sampling.sample``).  Where ``own`` is false
``run`` computes the same from elementary torch operations in 32 bits (the draw in 64).

A cache holds ``[pages, KV heads, page rows, head dim]``; row ``j`` of sequence ``b`` lies in page
``table[b, j // rows]``.  Pages are handed out in a random order, as after a while of serving; rows that no
sequence owns hold large values, as memory that other requests have used.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS = 1e-6
VOCAB_TEXT, VOCAB_AUDIO = 151936, 1024
#: (query heads, KV heads, head dim): the backbone's, and other groupings
LAYOUTS = ((32, 8, 128), (28, 4, 128), (12, 12, 64), (16, 2, 64), (16, 1, 128))
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------ the cases
def _text(values):
    return ",".join(str(int(v)) for v in values)


def _numbers(text):
    return [int(v) for v in text.split(",")]


def _spread(seed, count, low, high):
    """``count`` lengths whose logarithms are spread over [low, high], the same ones every time."""
    rng = random.Random(seed)
    return [_log_int(rng, low, high) for _ in range(count)]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _heads(layout):
    return dict(qh=layout[0], kh=layout[1], d=layout[2])


def listed():
    base = _heads(LAYOUTS[0])
    return [
        # one request's next token: q/k norm, rotary and its cache row; launch latency
        dict(name="rope_decode_1", kind="rope", **base, dtype="bf16", page=16, new="1", old="812", pad=0),
        # a step that takes in seven prompts of different lengths, two of them continued, in a padded batch
        dict(name="rope_prompts_7", kind="rope", **base, dtype="bf16", page=64, new="733,5,391,128,64,1017,211",
             old="0,1200,0,640,0,0,7", pad=23),
        # one request's next token over a short cache: latency
        dict(name="decode_1_of_509", kind="decode", **base, dtype="bf16", page=16, lengths="509"),
        # a handful of requests of very different lengths, one slot of the batch empty
        dict(name="decode_16_ragged", kind="decode", **base, dtype="bf16", page=16,
             lengths=_text(_spread(1, 15, 17, 8000) + [0])),
        # a full server: 64 requests of 4 to 8 thousand tokens
        dict(name="decode_64_long", kind="decode", **base, dtype="bf16", page=64, lengths=_text(_spread(2, 64, 4096, 8192))),
        # heads that share nothing, 64 wide, in half precision
        dict(name="decode_48_single_heads", kind="decode", **_heads(LAYOUTS[2]), dtype="fp16", page=32,
             lengths=_text(_spread(3, 48, 60, 2000))),
        # one short prompt: the smallest prompt pass
        dict(name="prompt_1_of_45", kind="prompt", **base, dtype="bf16", page=16, new="45", old="0", pad=0),
        # a mixed step: long and short prompts, two that continue a cached prefix, a single token, padding
        dict(name="prompts_9_packed", kind="prompt", **base, dtype="bf16", page=16,
             new="611,37,1,902,256,75,450,130,333", old="0,0,1777,0,1024,0,0,600,0", pad=13),
        # one long document
        dict(name="prompt_1_of_8000", kind="prompt", **base, dtype="bf16", page=64, new="8000", old="0", pad=0),
        # the audio heads of one frame of 16 requests
        dict(name="sample_audio_512", kind="sample", rows=512, vocab=VOCAB_AUDIO, dtype="bf16", style="audio"),
        # one request's next text token
        dict(name="sample_text_1", kind="sample", rows=1, vocab=VOCAB_TEXT, dtype="bf16", style="mixed"),
        # a full server's text tokens, every request with its own settings
        dict(name="sample_text_128", kind="sample", rows=128, vocab=VOCAB_TEXT, dtype="bf16", style="mixed"),
    ]


def draw(rng):
    kind = rng.choice(("rope", "decode", "decode", "prompt", "prompt", "sample"))
    if kind == "sample":
        rows, vocab = _log_int(rng, 1, 512), _log_int(rng, 900, VOCAB_TEXT)
        return dict(kind=kind, rows=max(1, min(rows, 128 * VOCAB_TEXT // (2 * vocab))), vocab=vocab,
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), style=rng.choice(("audio", "mixed", "plain")))
    layout = rng.choice((LAYOUTS[0], LAYOUTS[0]) + LAYOUTS[1:])
    case = dict(kind=kind, **_heads(layout), dtype=rng.choice(("bf16", "bf16", "fp16")), page=rng.choice((16, 32, 64, 128)))
    if kind == "decode":
        count = _log_int(rng, 1, 64)
        top = _log_int(rng, 64, 5000)
        lengths = [0 if rng.random() < 0.03 else _log_int(rng, max(1, top // rng.choice((1, 2, 20))), top) for _ in range(count)]
        return dict(case, lengths=_text(lengths if any(lengths) else [top]))
    count = _log_int(rng, 1, 12)
    top = _log_int(rng, 2, 2048 if kind == "rope" else 1500)
    new = [_log_int(rng, max(1, top // 20), top) for _ in range(count)]
    old = [0 if rng.random() < 0.6 else _log_int(rng, 1, 1500) for _ in range(count)]
    return dict(case, new=_text(new), old=_text(old), pad=rng.choice((0, 0, rng.randint(1, 40))))


# ------------------------------------------------------------------------------------ their inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _cache(case, lengths, g, filled):
    """Keys, values and the page table of sequences of ``lengths`` rows; ``filled``: rows that are written already."""
    page, dtype = case["page"], TYPES[case["dtype"]]
    counts = [-(-n // page) for n in lengths]
    pages, width = sum(counts) + 3, max(counts) + 2  # a table has room for what is still to come
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros((len(lengths), width), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (pages, case["kh"], page, case["d"])
    keys, values = _normal(shape, dtype, g), _normal(shape, dtype, g)
    for b, n in enumerate(filled):  # behind a sequence's last row: what an earlier request left
        if n % page:
            keys[table[b, n // page].long(), :, n % page:] = 200.0
            values[table[b, n // page].long(), :, n % page:] = 200.0
    return dict(keys=keys, values=values, table=table, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))


def _prepare_rope(case, seed):
    g, dtype = _generator(seed), TYPES[case["dtype"]]
    new, old = _numbers(case["new"]), _numbers(case["old"])
    lengths = [a + b for a, b in zip(new, old)]
    state = _cache(case, lengths, g, old)
    qh, kh, d = case["qh"], case["kh"], case["d"]
    total = sum(new)
    rows = (max(lengths) + 63) // 64 * 64
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (
        -torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    angle = torch.cat((angle, angle), 1)
    return dict(state, qkv=_normal((total + case["pad"], (qh + 2 * kh) * d), dtype, g, 2.0),
                q_weight=_normal((d,), dtype, g, 0.1) + 1, k_weight=_normal((d,), dtype, g, 0.1) + 1,
                cos=angle.cos().float(), sin=angle.sin().float(),
                starts=torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32),
                q=torch.zeros((total + case["pad"], qh, d), dtype=dtype, device="cuda"))


def _prepare_decode(case, seed):
    g = _generator(seed)
    lengths = _numbers(case["lengths"])
    return dict(_cache(case, lengths, g, lengths),
                q=_normal((len(lengths), case["qh"], case["d"]), TYPES[case["dtype"]], g, 2.0))


def _prepare_prompt(case, seed):
    g, dtype = _generator(seed), TYPES[case["dtype"]]
    new, old = _numbers(case["new"]), _numbers(case["old"])
    lengths = [a + b for a, b in zip(new, old)]
    total = sum(new) + case["pad"]
    return dict(_cache(case, lengths, g, lengths), q=_normal((total, case["qh"], case["d"]), dtype, g, 2.0),
                starts=torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32), longest=max(new),
                out=torch.zeros((total, case["qh"] * case["d"]), dtype=dtype, device="cuda"))


def _prepare_sample(case, seed):
    g = _generator(seed)
    rows, vocab = case["rows"], case["vocab"]
    # a language model's logits: a broad bell and a few entries that stand out
    logits = torch.randn((rows, vocab), device="cuda", generator=g) * 2.0
    few = torch.randint(0, vocab, (rows, 24), device="cuda", generator=g)
    logits.scatter_add_(1, few, torch.rand((rows, 24), device="cuda", generator=g) * 12.0)

    def pick(values, dtype):
        return torch.tensor(values, dtype=dtype, device="cuda")[
            torch.randint(0, len(values), (rows,), device="cuda", generator=g)]

    if case["style"] == "audio":  # the audio heads' settings
        settings = (pick([1.7], torch.float32), pick([25], torch.int32), pick([0.8], torch.float32),
                    pick([0.0], torch.float32))
    elif case["style"] == "plain":  # temperature alone
        settings = (pick([0.7, 1.0], torch.float32), pick([0], torch.int32), pick([1.0], torch.float32),
                    pick([0.0], torch.float32))
    else:  # each request its own; some greedy
        settings = (pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.5], torch.float32), pick([0, 0, 20, 50, 1000], torch.int32),
                    pick([0.8, 0.9, 0.95, 1.0], torch.float32), pick([0.0, 0.0, 0.05, 0.1], torch.float32))
    return dict(logits=logits.to(TYPES[case["dtype"]]), uniform=torch.rand(rows, device="cuda", generator=g),
                temperature=settings[0], top_k=settings[1], top_p=settings[2], min_p=settings[3])


def prepare(case, seed):
    made = {"rope": _prepare_rope, "decode": _prepare_decode, "prompt": _prepare_prompt, "sample": _prepare_sample}
    return dict(made[case["kind"]](case, seed), kind=case["kind"])


# ------------------------------------------------------------------------------------ the operators
def _plain_rope(s):
    keys, values, table, starts = s["keys"], s["values"], s["table"].long(), s["starts"].long()
    kh, page, d = keys.shape[1:]
    tokens = s["qkv"].shape[0]
    x = s["qkv"].float().view(tokens, -1, d)
    qh = x.shape[1] - 2 * kh
    t = torch.arange(tokens, device=x.device)
    held = t < starts[-1]  # tokens behind the last sequence are padding
    b = (torch.searchsorted(starts, t, right=True) - 1).clamp(0, table.shape[0] - 1)
    position = (s["lengths"].long()[b] - starts[b + 1] + t).clamp(0, s["cos"].shape[0] - 1)
    cos, sin = s["cos"].float()[position][:, None], s["sin"].float()[position][:, None]

    def turned(v, weight):
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * weight.float()
        return v * cos + torch.cat((-v[..., d // 2:], v[..., :d // 2]), -1) * sin

    q = turned(x[:, :qh], s["q_weight"]).to(s["q"].dtype)
    s["q"].copy_(torch.where(held[:, None, None], q, s["q"]))
    # padding writes again what the last token of the last sequence writes
    t = torch.minimum(t, starts[-1] - 1)
    place, row = table[b[t], position[t] // page], position[t] % page
    keys[place, :, row] = turned(x[:, qh:qh + kh], s["k_weight"]).to(keys.dtype)[t]
    values[place, :, row] = s["qkv"].view(tokens, -1, d)[:, qh + kh:][t]
    return s["q"], keys, values


def _gathered(pages, table):
    """``[B, KV heads, rows, d]`` in 32 bits from the pages of each sequence."""
    b, w = table.shape
    kh, page, d = pages.shape[1:]
    return pages[table.long()].float().permute(0, 2, 1, 3, 4).reshape(b, kh, w * page, d)


def _plain_attention(q, keys, values, seen, written):
    """q ``[B, KH, rows, d]``, keys and values ``[B, KH, L, d]``, seen ``[B, 1, rows, L]``, written ``[B, 1, L, 1]``."""
    score = torch.matmul(q, keys.transpose(2, 3).contiguous()) * (q.shape[-1] ** -0.5)
    score = score.masked_fill_(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = weight.sum(-1, keepdim=True)
    return torch.matmul(weight, torch.where(written, values, torch.zeros_like(values))) / torch.where(
        total == 0, torch.ones_like(total), total)


def _plain_decode(s):
    q, keys = s["q"], _gathered(s["keys"], s["table"])
    values = _gathered(s["values"], s["table"])
    b, qh, d = q.shape
    kh, rows = keys.shape[1:3]
    seen = torch.arange(rows, device=q.device)[None] < s["lengths"][:, None]
    o = _plain_attention(q.float().view(b, kh, qh // kh, d), keys, values, seen[:, None, None], seen[:, None, :, None])
    return o.reshape(b, qh * d).to(q.dtype)


def _plain_prompt(s):
    q, starts = s["q"], s["starts"].long()
    keys, values = _gathered(s["keys"], s["table"]), _gathered(s["values"], s["table"])
    tokens, qh, d = q.shape
    b, kh, rows = keys.shape[:3]
    n = s["longest"]
    i = torch.arange(n, device=q.device)
    token = (starts[:-1, None] + i).clamp(max=tokens - 1)  # [B, n], a row of padding behind each shorter prompt
    position = s["lengths"].long()[:, None] - (starts[1:] - starts[:-1])[:, None] + i
    j = torch.arange(rows, device=q.device)
    written = j[None] < s["lengths"][:, None]
    seen = (j <= position[..., None]) & written[:, None]
    group = qh // kh
    x = q.float()[token].view(b, n, kh, group, d).permute(0, 2, 3, 1, 4).reshape(b, kh, group * n, d)
    o = _plain_attention(x, keys, values, seen.repeat(1, group, 1)[:, None], written[:, None, :, None])
    o = o.view(b, kh, group, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, qh * d).to(q.dtype)
    t = torch.arange(tokens, device=q.device)
    of = (torch.searchsorted(starts, t, right=True) - 1).clamp(0, b - 1)
    s["out"].copy_(torch.where((t < starts[-1])[:, None], o[of, (t - starts[of]).clamp(0, n - 1)], s["out"]))
    return s["out"]


def _plain_sample(s):
    x = s["logits"].double()
    temperature = s["temperature"].double()[:, None]
    ordered, order = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = temperature <= 0
    weight = torch.exp((ordered - ordered[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature))
    top_k = s["top_k"].long()[:, None]
    rank = torch.arange(x.shape[1], device=x.device)[None]
    weight = torch.where((rank < top_k) | (top_k <= 0), weight, torch.zeros_like(weight))
    through = torch.cumsum(weight, 1)
    top_p = s["top_p"].double()[:, None]
    keep = (through - weight <= top_p * through[:, -1:]) | (top_p >= 1)
    weight = torch.where(keep & (weight >= s["min_p"].double()[:, None]), weight, torch.zeros_like(weight))
    through = torch.cumsum(torch.zeros_like(x).scatter_(1, order, weight), 1)
    drawn = (through <= s["uniform"].double()[:, None] * through[:, -1:]).sum(1)
    return torch.where(greedy[:, 0], order[:, 0], drawn.clamp(max=x.shape[1] - 1))


def _own(s):
    from moss_tts._runtime import paged, sampling

    if s["kind"] == "rope":
        q = paged.qk_rope(s["qkv"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["keys"], s["values"], s["table"],
                          s["lengths"], EPS, starts=s["starts"], out=s["q"])
        return q, s["keys"], s["values"]
    if s["kind"] == "decode":
        return paged.decode_attention(s["q"], s["keys"], s["values"], s["table"], s["lengths"])
    if s["kind"] == "prompt":
        return paged.prompt_attention(s["q"], s["keys"], s["values"], s["table"], s["lengths"], s["starts"], out=s["out"])
    return sampling.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                           min_p=s["min_p"])


if os.path.join(ROOT, "moss-tts-optimized_amd") not in sys.path:
    sys.path.insert(0, os.path.join(ROOT, "moss-tts-optimized_amd"))


def run(state):
    if own:
        return _own(state)
    plain = {"rope": _plain_rope, "decode": _plain_decode, "prompt": _plain_prompt, "sample": _plain_sample}
    return plain[state["kind"]](state)


# ------------------------------------------------------------------------------------ what they cannot do without
def work(case):
    kind = case["kind"]
    if kind == "sample":
        wide = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * wide + 28), "flops": 8 * case["rows"] * case["vocab"]}
    qh, kh, d, wide = case["qh"], case["kh"], case["d"], 2
    if kind == "decode":
        lengths = _numbers(case["lengths"])
        return {"bytes": wide * d * (2 * kh * sum(lengths) + 2 * qh * len(lengths)), "flops": 4 * d * qh * sum(lengths)}
    new, old = _numbers(case["new"]), _numbers(case["old"])
    tokens, lengths = sum(new), [a + b for a, b in zip(new, old)]
    if kind == "rope":
        return {"bytes": 2 * tokens * (qh + 2 * kh) * d * wide + 8 * d * max(new), "flops": 10 * tokens * (qh + kh) * d}
    seen = sum(n * o + n * (n + 1) // 2 for n, o in zip(new, old))
    return {"bytes": wide * d * (2 * kh * sum(lengths) + 2 * qh * tokens), "flops": 4 * d * qh * seen}


# ------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_rope(case, s):
    new, old = _numbers(case["new"]), _numbers(case["old"])
    kh, d, page = case["kh"], case["d"], case["page"]
    q, keys, values = s["q"].double(), s["keys"].double(), s["values"].double()
    at = 0
    for b, (n, first) in enumerate(zip(new, old)):
        x = s["qkv"][at:at + n].double().view(n, -1, d)
        cos, sin = (s[name][first:first + n].double().view(n, 1, d) for name in ("cos", "sin"))
        for part, weight in ((slice(0, case["qh"]), "q_weight"), (slice(case["qh"], case["qh"] + kh), "k_weight")):
            y = x[:, part]
            y = y / (y.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * s[weight].double()
            low, high = y.chunk(2, -1)
            x[:, part] = torch.cat((low * cos[..., :d // 2] - high * sin[..., :d // 2],
                                    high * cos[..., d // 2:] + low * sin[..., d // 2:]), -1)
        q[at:at + n] = x[:, :case["qh"]]
        for p in range(first // page, (first + n - 1) // page + 1):
            low, high = max(first, p * page), min(first + n, (p + 1) * page)
            place, rows, mine = int(s["table"][b, p]), slice(low - p * page, high - p * page), slice(low - first, high - first)
            keys[place, :, rows] = x[mine, case["qh"]:case["qh"] + kh].transpose(0, 1)
            values[place, :, rows] = x[mine, case["qh"] + kh:].transpose(0, 1)
        at += n
    return q, keys, values


def _exact_rows(q, s, b, length, first):
    """Queries ``[n, heads, d]`` at positions ``first ..`` over the ``length`` rows of sequence ``b``."""
    kh, page, d = s["keys"].shape[1:]
    group = q.shape[1] // kh
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    own_pages = s["table"][b, :-(-length // page)].long()
    for h in range(kh if length else 0):
        k, v = (s[name][own_pages, h].reshape(-1, d)[:length].double() for name in ("keys", "values"))
        for low in range(0, q.shape[0], 1024):
            x = q[low:low + 1024, h * group:(h + 1) * group].double()
            a = (x.reshape(-1, d) @ k.T / math.sqrt(d)).view(x.shape[0], group, length)
            last = first + low + torch.arange(x.shape[0], device=q.device)
            a[(torch.arange(length, device=q.device) > last[:, None])[:, None].expand_as(a)] = -math.inf
            out[low:low + 1024, h * group:(h + 1) * group] = (torch.softmax(a, -1).view(-1, length) @ v).view(x.shape)
    return out.flatten(1)


def exact(case, seed):
    if case["kind"] == "sample":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, s)
    if case["kind"] == "decode":
        lengths = _numbers(case["lengths"])
        return torch.cat([_exact_rows(s["q"][b:b + 1], s, b, n, n) for b, n in enumerate(lengths)])
    out, at = s["out"].double(), 0
    for b, (n, first) in enumerate(zip(_numbers(case["new"]), _numbers(case["old"]))):
        out[at:at + n] = _exact_rows(s["q"][at:at + n], s, b, n + first, first)
        at += n
    return out
