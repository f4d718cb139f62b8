"""What a server of a batch needs around its paged cache: operators as cases that can be timed and compared.

Three sets.  A cache in 8 bits: new tokens' rows written as e4m3 codes with a power of two a row (``paged.qk_rope`` and,
to have the rows back, ``paged.gather``), and the attentions that read it (``paged.decode_attention``,
``paged.prompt_attention``).  Decode attention of sequences that share a long prefix, which is read once for all of them
(``paged.shared_decode_attention``).  Penalties for repeated tokens, biases and grammar masks on logits
(``sampling.adjust``).  Where ``own`` is false ``run`` computes the same from elementary torch operations in 32 bits.

A cache holds ``[pages, KV heads, page rows, head dim]``; row ``j`` of sequence ``b`` lies in page
``table[b, j // rows]``.  In 8 bits a value is its code times 2^(byte - 127), with one byte for each row of each KV head.
Pages are handed out in a random order, as after a while of serving; what no sequence owns holds large values.
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
#: exponents that a row's scale may take: its values stay exact in the 16-bit type
EXPONENTS = {torch.bfloat16: (-100, 120), torch.float16: (-15, 8)}


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
    base = dict(_heads(LAYOUTS[0]), dtype="bf16")
    return [
        # one request's next token into an 8-bit cache: launch latency
        dict(name="write8_1", kind="write", **base, page=16, new="1", old="812", pad=0),
        # a step that takes in seven prompts of different lengths, two of them continued, in a padded batch
        dict(name="write8_prompts_7", kind="write", **base, page=64, new="733,5,391,128,64,1017,211",
             old="0,1200,0,640,0,0,7", pad=23),
        # one request's next token over a short 8-bit cache: latency
        dict(name="decode8_1_of_509", kind="decode", **base, page=16, lengths="509"),
        # a handful of requests of very different lengths, one slot of the batch empty
        dict(name="decode8_16_ragged", kind="decode", **base, page=16, lengths=_text(_spread(1, 15, 17, 8000) + [0])),
        # a full server: 64 requests of 4 to 8 thousand tokens
        dict(name="decode8_64_long", kind="decode", **base, page=64, lengths=_text(_spread(2, 64, 4096, 8192))),
        # a mixed step over an 8-bit cache: long and short prompts, continued prefixes, a single token, padding
        dict(name="prompt8_9_packed", kind="prompt", **base, page=16, new="611,37,1,902,256,75,450,130,333",
             old="0,0,1777,0,1024,0,0,600,0", pad=13),
        # one long document
        dict(name="prompt8_1_of_8000", kind="prompt", **base, page=64, new="8000", old="0", pad=0),
        # four takes of one sentence after a short voice prompt
        dict(name="shared_4_of_640", kind="shared", **base, bits=16, page=16, sizes="4", prefix="640", lengths="61,85,3,120"),
        # a full server whose 64 requests all speak with one voice and its long instruction
        dict(name="shared_64_of_4096", kind="shared", **base, bits=16, page=64, sizes="64", prefix="4096",
             lengths=_text(_spread(4, 64, 30, 1500))),
        # several voices of different popularity, two requests without one, an 8-bit cache
        dict(name="shared8_40_in_groups", kind="shared", **base, bits=8, page=32, sizes="17,1,9,5,1,7",
             prefix="1504,0,2912,480,0,6016", lengths=_text(_spread(5, 40, 10, 900))),
        # the audio heads of one frame of 16 requests: codes said before are damped
        dict(name="adjust_audio_512", kind="adjust", rows=512, vocab=VOCAB_AUDIO, dtype="bf16", width=400, style="repetition"),
        # a full server's text tokens, every request with its own penalties, biases and grammar
        dict(name="adjust_text_128", kind="adjust", rows=128, vocab=VOCAB_TEXT, dtype="bf16", width=4096, style="all"),
    ]


def draw(rng):
    kind = rng.choice(("write", "decode", "decode", "prompt", "shared", "shared", "adjust", "adjust"))
    if kind == "adjust":
        rows, vocab = _log_int(rng, 1, 512), _log_int(rng, 900, VOCAB_TEXT)
        return dict(kind=kind, rows=max(1, min(rows, 128 * VOCAB_TEXT // (2 * vocab))), vocab=vocab,
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), width=_log_int(rng, 1, 4000),
                    style=rng.choice(("repetition", "all", "mask", "penalties")))
    layout = rng.choice((LAYOUTS[0], LAYOUTS[0]) + LAYOUTS[1:])
    case = dict(kind=kind, **_heads(layout), dtype=rng.choice(("bf16", "bf16", "fp16")), page=rng.choice((16, 32, 64, 128)))
    if kind == "decode":
        count = _log_int(rng, 1, 64)
        top = _log_int(rng, 64, 5000)
        lengths = [0 if rng.random() < 0.03 else _log_int(rng, max(1, top // rng.choice((1, 2, 20))), top) for _ in range(count)]
        return dict(case, lengths=_text(lengths if any(lengths) else [top]))
    if kind == "shared":
        sizes = [1 if rng.random() < 0.15 else _log_int(rng, 2, 40) for _ in range(rng.choice((1, 1, 2, 3, 5)))]
        prefix = [0 if n == 1 else max(1, _log_int(rng, 100, 4000) // case["page"]) * case["page"] for n in sizes]
        top = _log_int(rng, 10, 1000)
        return dict(case, bits=rng.choice((16, 16, 8)), sizes=_text(sizes), prefix=_text(prefix),
                    lengths=_text(_log_int(rng, 1, top) for _ in range(sum(sizes))))
    count = _log_int(rng, 1, 12)
    top = _log_int(rng, 2, 2048 if kind == "write" else 1500)
    new = [_log_int(rng, max(1, top // 20), top) for _ in range(count)]
    old = [0 if rng.random() < 0.6 else _log_int(rng, 1, 1500) for _ in range(count)]
    return dict(case, new=_text(new), old=_text(old), pad=rng.choice((0, 0, rng.randint(1, 40))))


# ------------------------------------------------------------------------------------ their inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _codes(x, dtype):
    """e4m3 codes and scale bytes of rows ``[..., d]`` in 32 bits: the least power of two that brings a row under 448."""
    low, high = EXPONENTS[dtype]
    part, exponent = torch.frexp(x.abs().amax(-1))
    exponent = torch.where(part == 0, torch.full_like(exponent, low), exponent - 9 + (part > 0.875).int()).clamp(low, high)
    return (x * _power(127 - exponent)[..., None]).to(torch.float8_e4m3fn), (exponent + 127).to(torch.uint8)


def _power(byte):
    """2^(byte - 127), from its bits."""
    return (byte.int() << 23).view(torch.float32)


def _fill(shape, case, g, bits):
    """Keys or values, rows of different sizes, and the scale bytes of an 8-bit cache."""
    dtype = TYPES[case["dtype"]]
    x = torch.randn(shape, device="cuda", generator=g)
    if bits == 16:
        return x.to(dtype), None
    x *= torch.exp2(torch.rand(shape[:3], device="cuda", generator=g) * 3 - 1.5)[..., None]
    return _codes(x, dtype)


def _cache(case, table, lengths, filled, pages, g, bits):
    """Keys, values, their scale bytes, table and lengths; ``filled``: rows that are written already."""
    page = case["page"]
    shape = (pages, case["kh"], page, case["d"])
    (keys, key_scales), (values, value_scales) = _fill(shape, case, g, bits), _fill(shape, case, g, bits)
    for b, n in enumerate(filled):  # behind a sequence's last row: what an earlier request left
        if n % page:
            for t in (keys, values):
                if bits == 16:
                    t[table[b, n // page].long(), :, n % page:] = 200.0
                else:  # the code of 192
                    t.view(torch.uint8)[table[b, n // page].long(), :, n % page:] = 0x74
    return dict(keys=keys, values=values, scales=None if bits == 16 else (key_scales, value_scales), table=table,
                lengths=_ints(lengths))


def _pages(case, lengths, g):
    """A table with a page for every row, in a random order, and the number of pages."""
    counts = [-(-n // case["page"]) for n in lengths]
    pages = sum(counts) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros((len(lengths), max(counts) + 2), dtype=torch.int32, device="cuda")  # room for what is still to come
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def _prepare_write(case, seed):
    g, dtype = _generator(seed), TYPES[case["dtype"]]
    new, old = _numbers(case["new"]), _numbers(case["old"])
    lengths = [a + b for a, b in zip(new, old)]
    table, pages = _pages(case, lengths, g)
    state = _cache(case, table, lengths, old, pages, g, 8)
    qh, kh, d = case["qh"], case["kh"], case["d"]
    total = sum(new) + case["pad"]
    rows = (max(lengths) + 63) // 64 * 64
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (
        -torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    angle = torch.cat((angle, angle), 1)
    return dict(state, qkv=_normal((total, (qh + 2 * kh) * d), dtype, g, 2.0), q_weight=_normal((d,), dtype, g, 0.1) + 1,
                k_weight=_normal((d,), dtype, g, 0.1) + 1, cos=angle.cos().float(), sin=angle.sin().float(),
                starts=_ints([0] + new).cumsum(0).to(torch.int32), q=torch.zeros((total, qh, d), dtype=dtype, device="cuda"),
                rows=tuple(torch.zeros((total, kh, d), dtype=dtype, device="cuda") for _ in range(2)))


def _prepare_decode(case, seed):
    g = _generator(seed)
    lengths = _numbers(case["lengths"])
    table, pages = _pages(case, lengths, g)
    return dict(_cache(case, table, lengths, lengths, pages, g, 8),
                q=_normal((len(lengths), case["qh"], case["d"]), TYPES[case["dtype"]], g, 2.0))


def _prepare_prompt(case, seed):
    g, dtype = _generator(seed), TYPES[case["dtype"]]
    new, old = _numbers(case["new"]), _numbers(case["old"])
    lengths = [a + b for a, b in zip(new, old)]
    total = sum(new) + case["pad"]
    table, pages = _pages(case, lengths, g)
    return dict(_cache(case, table, lengths, lengths, pages, g, 8), q=_normal((total, case["qh"], case["d"]), dtype, g, 2.0),
                starts=_ints([0] + new).cumsum(0).to(torch.int32), longest=max(new),
                out=torch.zeros((total, case["qh"] * case["d"]), dtype=dtype, device="cuda"))


def _prepare_shared(case, seed):
    g = _generator(seed)
    sizes, prefix, mine = _numbers(case["sizes"]), _numbers(case["prefix"]), _numbers(case["lengths"])
    page = case["page"]
    before = [p for n, p in zip(sizes, prefix) for _ in range(n)]
    lengths = [p + n for p, n in zip(before, mine)]
    front, shared_pages = _pages(case, prefix, g)   # each prefix once
    rest, own_pages = _pages(case, mine, g)
    table = torch.zeros((len(mine), front.shape[1] + rest.shape[1]), dtype=torch.int32, device="cuda")
    for b, p in enumerate(before):
        run = sum(b >= sum(sizes[:i + 1]) for i in range(len(sizes)))
        table[b, :p // page] = front[run, :p // page]
        table[b, p // page:p // page + rest.shape[1]] = rest[b] + shared_pages
    run = [i if n > 1 else -1 for i, n in enumerate(sizes) for _ in range(n)]
    return dict(_cache(case, table, lengths, lengths, shared_pages + own_pages, g, case["bits"]), groups=_ints(run),
                shared=_ints(before), q=_normal((len(mine), case["qh"], case["d"]), TYPES[case["dtype"]], g, 2.0))


def _prepare_adjust(case, seed):
    g = _generator(seed)
    rows, vocab, width, style = case["rows"], case["vocab"], case["width"], case["style"]

    def uniform(*shape):
        return torch.rand(shape, device="cuda", generator=g)

    # a language model's logits: a broad bell and a few entries that stand out
    logits = torch.randn((rows, vocab), device="cuda", generator=g) * 2.0
    few = torch.randint(0, vocab, (rows, 24), device="cuda", generator=g)
    logits.scatter_add_(1, few, uniform(rows, 24) * 12.0)
    state = dict(logits=logits.to(TYPES[case["dtype"]]))
    if style != "mask":
        # what was said so far: some tokens often, others once; the first part of it is the prompt
        tokens = (vocab * uniform(rows, width) ** 3).long().clamp(max=vocab - 1)
        lengths = (uniform(rows) * (width + 1)).int()
        state |= dict(tokens=tokens, lengths=lengths, repetition=1.0 + 0.4 * uniform(rows))
    if style in ("all", "penalties"):
        state |= dict(prompt=(lengths * uniform(rows)).int(), presence=uniform(rows), frequency=0.3 * uniform(rows))
    if style == "all":
        # requests bias a few tokens each; places without one hold -1
        ids = torch.randint(0, vocab, (rows, 16), device="cuda", generator=g).int()
        state |= dict(bias_ids=torch.where(uniform(rows, 16) < 0.3, torch.full_like(ids, -1), ids),
                      bias=4.0 * torch.randn((rows, 16), device="cuda", generator=g))
    if style in ("all", "mask"):
        # a grammar allows a few tokens, most of them, or all
        share = torch.tensor([0.002, 0.5, 0.98, 1.0], device="cuda")[torch.randint(0, 4, (rows, 1), device="cuda", generator=g)]
        words = torch.zeros((rows, (vocab + 31) // 32), dtype=torch.int32, device="cuda")
        for bit in range(32):
            words |= (uniform(*words.shape) < share).int() << bit
        state |= dict(mask=words)
    return state


def prepare(case, seed):
    made = {"write": _prepare_write, "decode": _prepare_decode, "prompt": _prepare_prompt, "shared": _prepare_shared,
            "adjust": _prepare_adjust}
    return dict(made[case["kind"]](case, seed), kind=case["kind"])


# ------------------------------------------------------------------------------------ the operators
def _plain_write(s):
    keys, values, table, starts = s["keys"], s["values"], s["table"].long(), s["starts"].long()
    kh, page, d = keys.shape[1:]
    dtype, tokens = s["qkv"].dtype, s["qkv"].shape[0]
    x = s["qkv"].float().view(tokens, -1, d)
    qh = x.shape[1] - 2 * kh
    t = torch.arange(tokens, device=x.device)
    held = (t < starts[-1])[:, None, None]  # tokens behind the last sequence are padding
    b = (torch.searchsorted(starts, t, right=True) - 1).clamp(0, table.shape[0] - 1)
    position = (s["lengths"].long()[b] - starts[b + 1] + t).clamp(0, s["cos"].shape[0] - 1)
    cos, sin = s["cos"][position][:, None], s["sin"][position][:, None]

    def turned(v, weight):
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * weight.float()
        return v * cos + torch.cat((-v[..., d // 2:], v[..., :d // 2]), -1) * sin

    s["q"].copy_(torch.where(held, turned(x[:, :qh], s["q_weight"]).to(dtype), s["q"]))
    # padding writes again what the last token of the last sequence writes
    t = torch.minimum(t, starts[-1] - 1)
    place, row = table[b[t], position[t] // page], position[t] % page
    for pages, scales, rows, back in zip((keys, values), s["scales"], (turned(x[:, qh:qh + kh], s["k_weight"]), x[:, qh + kh:]),
                                         s["rows"]):
        codes, scale = _codes(rows[t], dtype)
        pages.view(torch.uint8)[place, :, row] = codes.view(torch.uint8)
        scales[place, :, row] = scale
        read = pages.view(torch.uint8)[place, :, row].view(torch.float8_e4m3fn).float() * _power(scales[place, :, row])[..., None]
        back.copy_(torch.where(held, read.to(dtype), back))
    return s["q"], *s["rows"]


def _gathered(pages, scales, table):
    """``[B, KV heads, rows, d]`` in 32 bits from the pages of each sequence."""
    b, w = table.shape
    kh, page, d = pages.shape[1:]
    table = table.long()
    if scales is None:
        x = pages[table].float()
    else:
        x = pages.view(torch.uint8)[table].view(torch.float8_e4m3fn).float().mul_(_power(scales[table])[..., None])
    return x.permute(0, 2, 1, 3, 4).reshape(b, kh, w * page, d)


def _plain_attention(q, keys, values, seen, written):
    """q ``[B, KH, rows, d]``, keys and values ``[B, KH, L, d]``, seen ``[B, 1, rows, L]``, written ``[B, 1, L, 1]``."""
    score = torch.matmul(q, keys.transpose(2, 3).contiguous()) * (q.shape[-1] ** -0.5)
    score = score.masked_fill_(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = weight.sum(-1, keepdim=True)
    return torch.matmul(weight, torch.where(written, values, torch.zeros_like(values))) / torch.where(
        total == 0, torch.ones_like(total), total)


def _both(s):
    key_scales, value_scales = s["scales"] or (None, None)
    return _gathered(s["keys"], key_scales, s["table"]), _gathered(s["values"], value_scales, s["table"])


def _plain_decode(s):
    q = s["q"]
    keys, values = _both(s)
    b, qh, d = q.shape
    kh, rows = keys.shape[1:3]
    seen = torch.arange(rows, device=q.device)[None] < s["lengths"][:, None]
    o = _plain_attention(q.float().view(b, kh, qh // kh, d), keys, values, seen[:, None, None], seen[:, None, :, None])
    return o.reshape(b, qh * d).to(q.dtype)


def _plain_prompt(s):
    q, starts = s["q"], s["starts"].long()
    keys, values = _both(s)
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


def _plain_adjust(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    if "tokens" in s:
        i = torch.arange(s["tokens"].shape[1], device=x.device)
        held = (i < s["lengths"][:, None]).float()
        said = torch.zeros_like(x).scatter_add_(1, s["tokens"], held)
        rate = s["repetition"][:, None]
        x = torch.where(said > 0, torch.where(x > 0, x / rate, x * rate), x)
        if "prompt" in s:
            count = torch.zeros_like(x).scatter_add_(1, s["tokens"], held * (i >= s["prompt"][:, None]))
            x = x - (count * s["frequency"][:, None] + (count > 0) * s["presence"][:, None])
    if "bias" in s:
        # of equal ids the last one's bias holds
        ids = s["bias_ids"].long()
        later = (ids[:, :, None] == ids[:, None, :]).triu(1).any(2)
        bias = torch.where((ids < 0) | later, torch.zeros_like(s["bias"]), s["bias"])
        x = x + torch.zeros_like(x).scatter_add_(1, ids.clamp(min=0), bias)
    if "mask" in s:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = x.masked_fill(bits.view(rows, -1)[:, :vocab] == 0, float("-inf"))
    return x.to(s["logits"].dtype)


def _own(s):
    from moss_tts._runtime import paged, sampling

    if s["kind"] == "adjust":
        return sampling.adjust(s["logits"], tokens=s.get("tokens"), lengths=s.get("lengths"), prompt=s.get("prompt"),
                               repetition=s.get("repetition", 1.0), presence=s.get("presence", 0.0),
                               frequency=s.get("frequency", 0.0), bias_ids=s.get("bias_ids"), bias=s.get("bias"),
                               mask=s.get("mask"))
    cache = s["keys"], s["values"], s["table"], s["lengths"]
    if s["kind"] == "write":
        q = paged.qk_rope(s["qkv"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], *cache, EPS, starts=s["starts"],
                          out=s["q"], scales=s["scales"])
        return q, *paged.gather(*cache, s["starts"], q.shape[0], scales=s["scales"], out=s["rows"])
    if s["kind"] == "decode":
        return paged.decode_attention(s["q"], *cache, scales=s["scales"])
    if s["kind"] == "prompt":
        return paged.prompt_attention(s["q"], *cache, s["starts"], out=s["out"], scales=s["scales"])
    return paged.shared_decode_attention(s["q"], *cache, s["groups"], s["shared"], scales=s["scales"])


if os.path.join(ROOT, "moss-tts-optimized_amd") not in sys.path:
    sys.path.insert(0, os.path.join(ROOT, "moss-tts-optimized_amd"))


def run(state):
    if own:
        return _own(state)
    plain = {"write": _plain_write, "decode": _plain_decode, "prompt": _plain_prompt, "shared": _plain_decode,
             "adjust": _plain_adjust}
    return plain[state["kind"]](state)


# ------------------------------------------------------------------------------------ what they cannot do without
def work(case):
    kind = case["kind"]
    if kind == "adjust":
        rows, vocab, style = case["rows"], case["vocab"], case["style"]
        moved = rows * vocab * 2 * (4 if case["dtype"] == "fp32" else 2)
        if style != "mask":
            moved += rows * (case["width"] // 2 * 8 + 16)
        if style in ("all", "mask"):
            moved += rows * (vocab + 31) // 32 * 4
        if style == "all":
            moved += rows * 16 * 8
        return {"bytes": moved, "flops": 6 * rows * vocab}
    qh, kh, d = case["qh"], case["kh"], case["d"]
    row = 2 * kh * (2 * d if case.get("bits") == 16 else d + 1)  # a token's keys and values in the cache
    if kind == "decode":
        lengths = _numbers(case["lengths"])
        return {"bytes": row * sum(lengths) + 4 * qh * d * len(lengths), "flops": 4 * d * qh * sum(lengths)}
    if kind == "shared":
        sizes, prefix, mine = _numbers(case["sizes"]), _numbers(case["prefix"]), _numbers(case["lengths"])
        seen = sum(n * p for n, p in zip(sizes, prefix)) + sum(mine)
        return {"bytes": row * (sum(prefix) + sum(mine)) + 4 * qh * d * len(mine), "flops": 4 * d * qh * seen}
    new, old = _numbers(case["new"]), _numbers(case["old"])
    tokens, lengths = sum(new), [a + b for a, b in zip(new, old)]
    if kind == "write":  # the rows go into the cache and come back
        return {"bytes": tokens * (4 * (qh + 2 * kh) * d + 2 * row) + 8 * d * max(new), "flops": 14 * tokens * (qh + 2 * kh) * d}
    seen = sum(n * o + n * (n + 1) // 2 for n, o in zip(new, old))
    return {"bytes": row * sum(lengths) + 4 * qh * d * tokens, "flops": 4 * d * qh * seen}


# ------------------------------------------------------------------------------------ the definitions in 64 bits
def _held(x, dtype):
    """What an 8-bit cache holds of rows in 64 bits: four significant bits above 2^(e - 6), steps of 2^(e - 9) below."""
    low, high = EXPONENTS[dtype]
    e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 448.0)).clamp(low, high)
    step = torch.exp2(torch.floor(torch.log2(x.abs())).maximum(e - 6) - 3)
    return torch.round(x / step) * step


def _exact_write(case, s):
    dtype = s["qkv"].dtype
    new, old = _numbers(case["new"]), _numbers(case["old"])
    qh, kh, d = case["qh"], case["kh"], case["d"]
    q, k, v = s["q"].double(), s["rows"][0].double(), s["rows"][1].double()
    at = 0
    for n, first in zip(new, old):
        x = s["qkv"][at:at + n].double().view(n, -1, d)
        cos, sin = (s[name][first:first + n].double().view(n, 1, d) for name in ("cos", "sin"))
        for to, part, weight in ((q, slice(0, qh), "q_weight"), (k, slice(qh, qh + kh), "k_weight")):
            y = x[:, part]
            y = y / (y.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * s[weight].double()
            low, high = y.chunk(2, -1)
            to[at:at + n] = torch.cat((low * cos[..., :d // 2] - high * sin[..., :d // 2],
                                       high * cos[..., d // 2:] + low * sin[..., d // 2:]), -1)
        k[at:at + n] = _held(k[at:at + n], dtype)
        v[at:at + n] = _held(x[:, qh + kh:], dtype)
        at += n
    return q, k, v


def _exact_rows(q, s, b, length, first):
    """Queries ``[n, heads, d]`` at positions ``first ..`` over the ``length`` rows of sequence ``b``."""
    kh, page, d = s["keys"].shape[1:]
    group = q.shape[1] // kh
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    own_pages = s["table"][b, :-(-length // page)].long()

    def rows_of(pages, scales, h):
        if scales is None:
            return pages[own_pages, h].reshape(-1, d)[:length].double()
        exponent = scales[own_pages, h].reshape(-1)[:length].double() - 127
        return pages[:, h].view(torch.uint8)[own_pages].view(pages.dtype).double().reshape(-1, d)[:length] * 2.0 ** exponent[:, None]

    scales = s["scales"] or (None, None)
    for h in range(kh if length else 0):
        k, v = rows_of(s["keys"], scales[0], h), rows_of(s["values"], scales[1], h)
        for low in range(0, q.shape[0], 1024):
            x = q[low:low + 1024, h * group:(h + 1) * group].double()
            a = (x.reshape(-1, d) @ k.T / math.sqrt(d)).view(x.shape[0], group, length)
            last = first + low + torch.arange(x.shape[0], device=q.device)
            a[(torch.arange(length, device=q.device) > last[:, None])[:, None].expand_as(a)] = -math.inf
            out[low:low + 1024, h * group:(h + 1) * group] = (torch.softmax(a, -1).view(-1, length) @ v).view(x.shape)
    return out.flatten(1)


def _exact_adjust(s):
    out = s["logits"].double()
    vocab = out.shape[1]
    for r in range(out.shape[0]):
        x = out[r]
        if "tokens" in s:
            said = s["tokens"][r, :int(s["lengths"][r])]
            known = torch.bincount(said, minlength=vocab) > 0
            rate = s["repetition"][r].double()
            x = torch.where(known, torch.where(x < 0, x * rate, x / rate), x)
            if "prompt" in s:
                count = torch.bincount(said[int(s["prompt"][r]):], minlength=vocab)
                x = x - s["frequency"][r].double() * count - s["presence"][r].double() * count.clamp(max=1)
        if "bias" in s:
            last = {i: v for i, v in zip(s["bias_ids"][r].tolist(), s["bias"][r].tolist()) if i >= 0}
            x = x.index_add(0, torch.tensor(list(last), device=x.device, dtype=torch.long),
                            torch.tensor(list(last.values()), device=x.device, dtype=torch.float64))
        if "mask" in s:
            i = torch.arange(vocab, device=x.device)
            allowed = (s["mask"][r].long()[i // 32] // 2 ** (i % 32)) % 2 == 1
            x = torch.where(allowed, x, torch.full_like(x, -math.inf))
        out[r] = x
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "adjust":
        return _exact_adjust(s)
    if case["kind"] == "write":
        return _exact_write(case, s)
    if case["kind"] in ("decode", "shared"):
        lengths = s["lengths"].tolist()
        return torch.cat([_exact_rows(s["q"][b:b + 1], s, b, n, n) for b, n in enumerate(lengths)])
    out, at = s["out"].double(), 0
    for b, (n, first) in enumerate(zip(_numbers(case["new"]), _numbers(case["old"]))):
        out[at:at + n] = _exact_rows(s["q"][at:at + n], s, b, n + first, first)
        at += n
    return out
