"""GPU: the compiled calls take what is in order, and give bit for bit what Python's own calls give."""
import threading
import types

import pytest
import torch

from paged_helpers import cache, cache8

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
NAMES = ["decode_attention", "shared_decode_attention", "prompt_attention", "qk_rope", "gather"]


def _batch(dev, dtype, eight, seed=0):
    g = torch.Generator().manual_seed(seed)
    lengths, new, qh, kh, d = [40, 3, 300, 65], [5, 3, 70, 1], 8, 2, 128
    if eight:
        keys, vals, scales, table, lens = cache8(dev, g, lengths, kh=kh, d=d, page=32)
    else:
        keys, vals, table, lens = cache(dev, g, lengths, kh=kh, d=d, page=32, dtype=dtype)
        scales = None
    starts = torch.tensor([0, 5, 8, 78, 79], dtype=torch.int32, device=dev)
    groups = torch.tensor([0, 1, 1, -1], dtype=torch.int32, device=dev)
    shared = torch.tensor([16, 0, 0, 16], dtype=torch.int32, device=dev)

    def rows(n, m):
        return torch.randn((n, m), generator=g).to(dtype).to(dev)

    q, packed, qkv = rows(4, qh * d).unflatten(1, (qh, d)), rows(79, qh * d + 8)[:, :qh * d].unflatten(1, (qh, d)), rows(79, (qh + 2 * kh) * d)
    cos, sin = torch.randn((2, 400, d), generator=g).to(dev)
    weights = rows(2, d)
    return types.SimpleNamespace(**{k: v for k, v in locals().items() if k not in ("rows", "g")})


def _call(s, name, **more):
    from moss_tts._runtime import paged

    given = (s.keys, s.vals, s.table, s.lens)
    more["scales"] = s.scales
    if name == "decode_attention":
        return paged.decode_attention(s.q, *given, **more)
    if name == "shared_decode_attention":
        return paged.shared_decode_attention(s.q, *given, s.groups, s.shared, **more)
    if name == "prompt_attention":
        return paged.prompt_attention(s.packed, *given, s.starts, **more)
    if name == "gather":
        return paged.gather(*given, s.starts, 79, **more)
    return paged.qk_rope(s.qkv, s.weights[0], s.weights[1], s.cos, s.sin, *given, 1e-6, starts=s.starts, **more)


class _Watch:
    """The compiled calls with a count of those that they took; or none of them, so that Python makes each call."""

    def __init__(self, taken=None):
        from moss_tts._runtime import native

        self.real, self.taken = native.calls(), taken

    def __call__(self):
        return self

    def __getattr__(self, name):
        def function(*args):
            if self.taken is None:
                return None
            out = getattr(self.real, name)(*args)
            if out is not None:
                self.taken.append(name)
            return out
        return function


def _both(monkeypatch, run):
    from moss_tts._runtime import native

    taken = []
    watch, plain = _Watch(taken), _Watch()
    monkeypatch.setattr(native, "calls", watch)
    one = run()
    monkeypatch.setattr(native, "calls", plain)
    two = run()
    monkeypatch.undo()
    torch.cuda.synchronize()
    assert len(taken) == 1, "Python made the call"
    return one, two


def _same(a, b):
    if isinstance(a, tuple):
        return len(a) == len(b) and all(_same(x, y) for x, y in zip(a, b))
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", NAMES)
def test_paged(dev, monkeypatch, name, dtype, eight):
    if eight and name == "gather":
        dtype = torch.bfloat16  # what gather gives unasked
    s = _batch(dev, dtype, eight)
    print(name, dtype, eight, flush=True)
    rows = {"decode_attention": (4, 1024), "shared_decode_attention": (4, 1024), "prompt_attention": (79, 1024),
            "qk_rope": (79, 8, 128), "gather": (79, 2, 128)}[name]
    one, two = _both(monkeypatch, lambda: _call(s, name))
    assert _same(one, two)
    if name == "gather":
        outs = tuple(torch.zeros(rows, dtype=dtype, device=dev) for _ in range(2))
        given, _ = _both(monkeypatch, lambda: _call(s, name, out=outs))
        assert given[0] is outs[0] and given[1] is outs[1]
    else:
        out = torch.zeros(rows, dtype=dtype, device=dev)
        more = {"out": out}
        if name != "qk_rope":
            more.update(scale=0.125, ws=torch.empty(1 << 24, device=dev))
        given, _ = _both(monkeypatch, lambda: _call(s, name, **more).clone())
        assert _call(s, name, **more) is out
        del more["out"]
        assert _same(given, _call(s, name, **more))


@pytest.mark.parametrize("eight", [False, True])
def test_written_rows(dev, monkeypatch, eight):
    """The cache that a call writes, too."""
    a, b = (_batch(dev, torch.bfloat16, eight) for _ in range(2))
    taken = iter((a, b))
    _both(monkeypatch, lambda: _call(next(taken), "qk_rope"))
    for x, y in [(a.keys, b.keys), (a.vals, b.vals)] + (list(zip(a.scales, b.scales)) if eight else []):
        assert _same(x, y)


@pytest.mark.parametrize("dtype", [*DTYPES, torch.float32])
@pytest.mark.parametrize("tensors", [False, True])
def test_adjust(dev, monkeypatch, dtype, tensors):
    from moss_tts._runtime import sampling

    g = torch.Generator().manual_seed(1)
    logits = torch.randn((5, 1030), generator=g).to(dtype).to(dev)[:, :1025]
    history = torch.randint(0, 1025, (60, 5), generator=g).to(dev).T
    lengths, prompt = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([60, 0, 7, 61, -1], [0, 3, 7, 20, 0]))
    settings = dict(repetition=1.3, presence=0.25, frequency=0.5)
    if tensors:
        settings = {k: torch.full((5,), v, device=dev) for k, v in settings.items()}
    ids = torch.randint(0, 1025, (1, 9), generator=g).to(torch.int32).to(dev)
    bias, mask = torch.randn((5, 9), generator=g).to(dev), torch.randint(-2 ** 31, 2 ** 31, (1, 33), generator=g).to(torch.int32).to(dev)
    more = dict(tokens=history, lengths=lengths, prompt=prompt, bias_ids=ids, bias=bias, mask=mask, **settings)
    for given in ({}, dict(mask=mask), dict(bias_ids=ids, bias=bias), more):
        print(dtype, tensors, sorted(given), flush=True)
        one, two = _both(monkeypatch, lambda: sampling.adjust(logits, **given))
        assert _same(one.contiguous(), two.contiguous())
    inplace = [logits.clone(), logits.clone()]
    taken = iter(inplace)

    def run():
        t = next(taken)
        return sampling.adjust(t, **more, out=t)

    one, two = _both(monkeypatch, run)
    assert one is inplace[0] and _same(one, two)


def test_stream_graph_and_threads(dev, monkeypatch):
    s = _batch(dev, torch.bfloat16, True)
    _call(s, "qk_rope")  # the rows that every later call writes again
    want = {name: _call(s, name) for name in NAMES}
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        q = s.q.clone().mul_(1)  # ready on this stream alone
        got = _call(types.SimpleNamespace(**{**vars(s), "q": q}), "decode_attention")
    side.synchronize()
    assert _same(got, want["decode_attention"])

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = {name: _call(s, name) for name in NAMES}
    for _ in range(3):
        for t in captured.values():
            for x in t if isinstance(t, tuple) else (t,):
                x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for name in NAMES:
            assert _same(captured[name], want[name]), name

    batches, failed = [_batch(dev, torch.bfloat16, bool(i % 2), seed=i) for i in range(3)], []
    for b in batches:
        _call(b, "qk_rope")
    expected = [{name: _call(b, name) for name in NAMES} for b in batches]
    torch.cuda.synchronize()

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = {name: _call(batches[i], name) for name in NAMES}
                    stream.synchronize()
                    failed.extend((i, name) for name in NAMES if not _same(got[name], expected[i][name]))
        except Exception as e:  # noqa: BLE001
            failed.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("eight", [False, True])
def test_one_output_of_two(dev, eight):
    s = _batch(dev, torch.bfloat16, eight)
    out = torch.zeros((79, 2, 128), dtype=torch.bfloat16, device=dev)
    for outs in ((out, None), (None, out), (None, None), (out, out), (out,), (out, out.clone(), out.clone())):
        with pytest.raises(ValueError):
            _call(s, "gather", out=outs)


def test_lists_are_left_to_python(dev):
    s = _batch(dev, torch.bfloat16, True)
    want = _call(s, "gather")
    outs = [torch.zeros_like(t) for t in want]
    got = _call(s, "gather", out=outs)
    torch.cuda.synchronize()
    assert got[0] is outs[0] and _same(tuple(got), want)


def test_no_reference_is_lost(dev):
    """Arguments and outputs are held as often after many calls as before."""
    import sys

    s = _batch(dev, torch.bfloat16, True)
    out = torch.zeros((4, 1024), dtype=torch.bfloat16, device=dev)
    outs = tuple(torch.zeros((79, 2, 128), dtype=torch.bfloat16, device=dev) for _ in range(2))
    things = [s.q, s.keys, s.table, s.scales, s.scales[0], s.lens, out, outs, outs[0]]

    def run():
        for _ in range(50):
            _call(s, "decode_attention", out=out)
            _call(s, "gather", out=outs)
            _call(s, "gather")

    run()
    torch.cuda.synchronize()
    before, held = [sys.getrefcount(t) for t in things], torch.cuda.memory_allocated()
    run()
    torch.cuda.synchronize()
    assert [sys.getrefcount(t) for t in things] == before and torch.cuda.memory_allocated() == held
