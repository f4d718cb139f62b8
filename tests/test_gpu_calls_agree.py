"""GPU: the compiled calls accept what Python's checks accept, argument by argument: every argument of every operator in forms that
are right, nearly right and wrong, through the compiled calls and without them, with the same outcome."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_calls import NAMES, _batch, _same

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def filled():
    """New tensors hold NaN: rows that a call leaves are the same in two of them."""
    torch.use_deterministic_algorithms(True, warn_only=True)
    yield
    torch.use_deterministic_algorithms(False)


def _forms(t):
    """(name, form) of a tensor argument: other types, devices, shapes, strides and alignments, over memory of their own."""
    yield "none", None
    yield "number", 3
    yield "host", t.cpu()
    for dtype in (torch.float32, torch.float16, torch.bfloat16, torch.int32, torch.int64, torch.uint8, torch.float8_e4m3fn):
        if dtype != t.dtype:
            yield str(dtype), torch.zeros(t.shape, dtype=dtype, device=t.device)

    def like(*shape):
        return torch.zeros(shape, dtype=torch.uint8, device=t.device).view(torch.uint8).to(torch.float32).to(t.dtype)

    def wide(shape, stride, offset=0):
        n = offset + 1 + sum((s - 1) * k for s, k in zip(shape, stride))
        v = like(n).as_strided(shape, stride, offset)
        v.copy_(t) if v.shape == t.shape and all(k for k in stride) else None
        return v

    shape, stride = tuple(t.shape), tuple(t.stride())
    yield "same", wide(shape, stride)
    yield "contiguous", t.clone(memory_format=torch.contiguous_format)
    yield "one element on", wide(shape, stride, 1)
    yield "16 bytes on", wide(shape, stride, max(1, 16 // t.element_size()))
    yield "more dims", t[None]
    yield "fewer dims", t[0] if t.dim() else t
    for i, s in enumerate(shape):
        yield f"dim {i} + 1", like(*shape[:i], s + 1, *shape[i + 1:])
        yield f"dim {i} - 1", like(*shape[:i], s - 1, *shape[i + 1:])
        if s != 1:
            yield f"dim {i} of 1", like(*shape[:i], 1, *shape[i + 1:])
        yield f"dim {i} of 0", like(*shape[:i], 0, *shape[i + 1:])
        if s > 1:
            yield f"dim {i} repeated", t.select(i, 0).unsqueeze(i).expand(shape)
    if t.dim():
        dense = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
        yield "every second", wide(shape, [2 * k for k in dense])
        for more in (1, 4, 8, 16):
            yield f"rows {more} apart", wide(shape, [dense[0] + more, *dense[1:]])
        if t.dim() > 1:
            yield "turned", t.transpose(0, 1).contiguous().transpose(0, 1)
            yield "turned at the end", t.transpose(-1, -2).contiguous().transpose(-1, -2)


NUMBERS = [None, True, 0, 1, -1, 2.5, -0.25, 1e-50, 1e39, float("nan"), float("inf"), "x", 1 << 70, 1 << 24, (1 << 24) - 1, np.float64(0.5),
           torch.tensor(1.0)]


def _operator(name):
    from moss_tts._runtime import paged, sampling

    return sampling.adjust if name == "adjust" else getattr(paged, name)


def _outcome(run):
    try:
        out = run()
    except (ValueError, TypeError, RuntimeError, OverflowError, AttributeError, ctypes.ArgumentError) as e:
        return type(e).__name__, str(e)
    torch.cuda.synchronize()
    return tuple(t.clone() for t in out) if isinstance(out, tuple) else out.clone()


def _agree(monkeypatch, name, args, what, taken):
    from moss_tts._runtime import native

    real = native.calls()

    class Watch:
        def __getattr__(self, function):
            def call(*a):
                got = getattr(real, function)(*a)
                taken.append(got is not None)
                return got
            return call

    positional, named = args
    operator = _operator(name)
    monkeypatch.setattr(native, "calls", lambda watch=Watch(): watch)
    one = _outcome(lambda: operator(*positional, **named))
    monkeypatch.setattr(native, "calls", lambda: native._NoCalls)
    two = _outcome(lambda: operator(*positional, **named))
    monkeypatch.undo()
    refused = [isinstance(x, tuple) and isinstance(x[0], str) for x in (one, two)]
    assert refused[0] == refused[1], (name, what, one if refused[0] else two)
    assert one == two if refused[0] else _same(one, two), (name, what)
    return refused[0]


def _arguments(s, name):
    """(positional, named) of a call that is right, and the shape of its output."""
    given = [s.keys, s.vals, s.table, s.lens]
    more = {"scales": s.scales}
    if name == "decode_attention":
        return [s.q, *given], more | dict(scale=0.125, out=None, ws=None)
    if name == "shared_decode_attention":
        return [s.q, *given, s.groups, s.shared], more | dict(scale=0.125, out=None, ws=None)
    if name == "prompt_attention":
        return [s.packed, *given, s.starts], more | dict(scale=0.125, out=None, ws=None)
    if name == "gather":
        return [*given, s.starts, 79], more | dict(out=None)
    return [s.qkv, s.weights[0], s.weights[1], s.cos, s.sin, *given, 1e-6], more | dict(starts=s.starts, out=None)


OUT = {"decode_attention": (4, 1024), "shared_decode_attention": (4, 1024), "prompt_attention": (79, 1024), "qk_rope": (79, 8, 128)}


def _cases(positional, named, out):
    """(what, positional, named) with one argument at a time in another form."""
    for at, value in [*enumerate(positional), *named.items()]:
        if isinstance(value, torch.Tensor):
            forms = _forms(value)
        elif at == "out" and out is not None:
            forms = _forms(out)
        elif at == "ws":
            forms = _forms(torch.zeros(1 << 23, device=out.device))
        elif at == "scales" and value is not None:
            forms = [("none", None), ("one", value[0]), ("a list", list(value)), ("three", (*value, value[0])), ("turned", value[::-1])]
            forms += [(f"{i}: {n}", tuple(f if j == i else t for j, t in enumerate(value))) for i in range(2) for n, f in _forms(value[i])]
        elif at == "scales":
            forms = [("a pair", (positional[0], positional[0])), ("a number", 3)]
        else:
            forms = [(str(n), n) for n in NUMBERS]
        for what, form in forms:
            if isinstance(at, int):
                yield f"{at} {what}", [*positional[:at], form, *positional[at + 1:]], named
            else:
                yield f"{at} {what}", positional, {**named, at: form}


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_paged(dev, monkeypatch, name, eight):
    s = _batch(dev, torch.bfloat16, eight)
    positional, named = _arguments(s, name)
    out = torch.zeros(OUT[name], dtype=torch.bfloat16, device=dev) if name in OUT else None
    taken, refused, count = [], 0, 0
    assert not _agree(monkeypatch, name, (positional, named), "as it is", taken) and taken == [True]
    for what, *args in _cases(positional, named, out):
        print(name, eight, what, flush=True)
        refused += _agree(monkeypatch, name, args, what, taken)
        count += 1
    assert count > 100 and sum(taken) > 10 and refused > 50


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_adjust(dev, monkeypatch, dtype):
    g = torch.Generator().manual_seed(1)
    logits = torch.randn((5, 1024), generator=g).to(dtype).to(dev)

    def ints(low, high, *shape):
        return torch.randint(low, high, shape, generator=g).to(torch.int32).to(dev)

    named = dict(tokens=ints(0, 1024, 5, 60).long(), lengths=ints(0, 61, 5), prompt=ints(0, 30, 5), repetition=torch.full((5,), 1.25, device=dev),
                 presence=0.5, frequency=torch.full((5,), 0.25, device=dev), bias_ids=ints(0, 1024, 5, 9), bias=torch.randn((5, 9), generator=g).to(dev),
                 mask=ints(-2 ** 31, 2 ** 31 - 1, 1, 32), out=None)
    taken, refused, count = [], 0, 0
    assert not _agree(monkeypatch, "adjust", ([logits], named), "as it is", taken) and taken == [True]
    for what, *args in _cases([logits], named, torch.zeros_like(logits)):
        print("adjust", dtype, what, flush=True)
        refused += _agree(monkeypatch, "adjust", args, what, taken)
        count += 1
    for missing in named:
        args = [logits], {k: v for k, v in named.items() if k != missing}
        refused += _agree(monkeypatch, "adjust", args, f"without {missing}", taken)
    for name in ("repetition", "presence", "frequency"):
        for value in NUMBERS:
            refused += _agree(monkeypatch, "adjust", ([logits], {**named, name: value}), f"{name} {value}", taken)
    assert count > 100 and sum(taken) > 10 and refused > 50


def test_bounds(dev, monkeypatch):
    """The largest of what is counted, and one more."""
    taken = []

    def zeros(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device=dev)

    keys = zeros(2, 1, 16, 64)

    def batch(n, w=1, packed=None):
        starts = torch.full((n + 1,), 0 if packed is None else packed, dtype=torch.int32, device=dev)
        starts[0] = 0
        return zeros(n, w, dtype=torch.int32), torch.full((n,), 3, dtype=torch.int32, device=dev), starts

    checks = []
    for n, fine in ((65535, True), (65536, False)):
        table, lens, _ = batch(n)
        checks.append(("decode_attention", [zeros(n, 1, 64), keys, keys.clone(), table, lens], {}, fine))
        checks.append(("shared_decode_attention", [zeros(n, 1, 64), keys, keys.clone(), table, lens, lens.clone(), lens.clone()], {}, fine))
    for w, fine in ((1 << 26, True), ((1 << 26) + 1, False)):
        table, lens, _ = batch(1, w)
        checks.append(("decode_attention", [zeros(1, 1, 64), keys, keys.clone(), table, lens], {}, fine))
    for qh, fine in ((1024, True), (1025, False)):
        table, lens, _ = batch(2)
        checks.append(("decode_attention", [zeros(2, qh, 64), keys, keys.clone(), table, lens], {}, fine))
    for n, fine in ((1 << 20, True), ((1 << 20) + 1, False)):
        table, lens, starts = batch(1, packed=3)
        checks.append(("prompt_attention", [zeros(n, 1, 64), keys, keys.clone(), table, lens, starts], {}, fine))
    for rows, fine in ((1 << 21, True), ((1 << 21) + 1, False)):
        checks.append(("adjust", [zeros(rows, 4)], {}, fine))
    for entries, fine in ((1 << 19, True), ((1 << 19) + 1, False)):
        checks.append(("adjust", [zeros(2, entries)], {}, fine))
    for n, fine in ((65535, True), (65536, False)):
        checks.append(("adjust", [zeros(2, 70)], dict(bias_ids=zeros(1, n, dtype=torch.int32), bias=zeros(2, n, dtype=torch.float32)), fine))
    for words, fine in ((3, True), (2, False)):
        checks.append(("adjust", [zeros(2, 70)], dict(mask=zeros(2, words, dtype=torch.int32)), fine))
    cos = zeros(4, 64, dtype=torch.float32)
    for page, fine in ((4096, True), (8192, False), (8, False), (48, False)):
        table, lens, starts = batch(2, packed=5)
        pool = zeros(2, 1, page, 64)
        checks.append(("qk_rope", [zeros(5, 3 * 64), None, None, cos, cos.clone(), pool, pool.clone(), table, lens, 1e-6], dict(starts=starts), fine))
        checks.append(("gather", [pool, pool.clone(), table, lens, starts, 5], {}, fine))
    for name, positional, named, fine in checks:
        shapes = [tuple(t.shape) for t in positional if isinstance(t, torch.Tensor)]
        print(name, shapes, flush=True)
        before = len(taken)
        assert _agree(monkeypatch, name, (positional, named), shapes, taken) == (not fine)
        assert taken[before] == fine, (name, shapes)
