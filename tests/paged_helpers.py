"""Inputs and bounds for the tests of the operators over a paged cache."""
import numpy as np
import torch


def values(t):
    """A tensor's values as float64."""
    return t.detach().cpu().to(torch.float64).numpy()


def cache(dev, g, lengths, *, kh, d, page, dtype, spare=3, width=None, poison=float("nan"), interleaved=False):
    """(keys, values, table, lengths): random rows where a sequence has them, ``poison`` everywhere else."""
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    width = max(max(counts), 1) + 1 if width is None else width
    order = torch.randperm(pages, generator=g)[:sum(counts)].tolist()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    if interleaved:  # keys and values of a page side by side
        both = torch.full((pages, 2, kh, page, d), poison, dtype=dtype)
        keys, vals = both[:, 0], both[:, 1]
    else:
        keys, vals = (torch.full((pages, kh, page, d), poison, dtype=dtype) for _ in range(2))
    at = 0
    for b, (n, c) in enumerate(zip(lengths, counts)):
        table[b, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
        for j in range(c):
            m = min(page, n - j * page)
            keys[order[at + j], :, :m] = torch.randn((kh, m, d), generator=g).to(dtype)
            vals[order[at + j], :, :m] = torch.randn((kh, m, d), generator=g).to(dtype)
        at += c
    if interleaved:
        both = both.to(dev)
        keys, vals = both[:, 0], both[:, 1]
    else:
        keys, vals = keys.to(dev), vals.to(dev)
    return keys, vals, table.to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev)


def attention_bound(q, keys, vals, ref, ref_abs, scale, dtype, rounded_p):
    """How far an attention output may be from the 64-bit one.

    Scores: an fp32 dot product of D exact products is off by at most D 2^-24 sum |q k|, the exponent's scaling,
    subtraction and exp2 by a few 2^-24 of a score and 2^-23 of the result.  A relative error r in every weight moves
    the output by at most 2 r sum p |v| (numerator and denominator).  Weights that are split into two 16-bit values are
    off by 2^-17, rounded ones by half a step; fp16 weights below 2^-14 by 2^-25 (of a largest weight of at least 2^-0,
    at most 2^13 of them here).  Then one rounding of the output."""
    half = torch.finfo(dtype).eps / 2
    d = q.shape[-1]
    kmax = np.nan_to_num(np.abs(keys), nan=0.0).max() if keys.size else 0.0
    vmax = np.nan_to_num(np.abs(vals), nan=0.0).max() if vals.size else 0.0
    s = np.abs(q).sum(-1).max() * kmax * abs(scale)
    r = (d + 8) * 2.0 ** -24 * s + 2.0 ** -17 + (half if rounded_p else 0.0)
    tiny = 2.0 ** -12 * vmax * 2.0 ** -1 if rounded_p and dtype == torch.float16 else 0.0
    # an output below the type's normal range is off by half its smallest step
    floor = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    return half * np.abs(ref) * (1 + 2 * r) + 2 * r * ref_abs + tiny + floor


def attend_all(q, keys, vals, table, lengths, starts, before, scale):
    """``oracle.paged.prompt_attention`` of whole tensors, in float64 on the device that holds them: for shapes with too
    many tokens and heads to take one at a time."""
    tokens, qh, d = q.shape
    pages, kh, page, _ = keys.shape
    group, width, dev = qh // kh, table.shape[1], q.device
    out = before.double().reshape(tokens, qh, d).clone()
    for b, (length, row) in enumerate(zip(lengths.tolist(), table.long())):
        first, n = starts[b], starts[b + 1] - starts[b]
        length = min(max(length, 0), width * page)
        if not n:
            continue
        if not length:
            out[first:first + n] = 0
            continue
        own = row[:-(-length // page)]
        has_page = (own >= 0) & (own < pages)
        there = has_page.repeat_interleave(page)[:length]
        at = torch.where(has_page, own, torch.zeros_like(own))
        position = length - n + torch.arange(n, device=dev)
        seen = (there & (torch.arange(length, device=dev) <= position[:, None])).repeat_interleave(group, 0)
        for h in range(kh):
            k, v = (t[at, h].reshape(-1, d)[:length].double() for t in (keys, vals))
            k, v = (torch.where(there[:, None], t, torch.zeros_like(t)) for t in (k, v))
            x = q[first:first + n, h * group:(h + 1) * group].double().reshape(n * group, d)
            s = torch.matmul(x, k.T.contiguous()).mul_(scale).masked_fill_(~seen, float("-inf"))
            top = s.amax(1, keepdim=True)
            e = s.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
            total = e.sum(1, keepdim=True)
            y = torch.matmul(e, v) / torch.where(total == 0, torch.ones_like(total), total)
            out[first:first + n, h * group:(h + 1) * group] = y.view(n, group, d)
    return out.view(before.shape)
