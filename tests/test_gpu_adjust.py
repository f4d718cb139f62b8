"""GPU: penalties, biases and masks on logits (``sampling.adjust``) against the definition in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import paged as o
from paged_helpers import values

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(dev, rows, vocab, dtype, *, seed=0, width=50, biases=5, token_type=torch.int64, what="hpbm", lengths=None):
    """``what``: h a history, p a prompt and the counted penalties, b biases, m a mask."""
    g = torch.Generator().manual_seed(seed)
    s = dict(logits=(torch.randn((rows, vocab), generator=g) * 4).to(dtype))
    if "h" in what:
        tokens = (vocab * 1.1 * torch.rand((rows, width), generator=g) ** 3).long() - 1  # some outside the row, many equal
        s |= dict(tokens=tokens.to(token_type), repetition=torch.rand(rows, generator=g) + 0.7,
                  lengths=torch.randint(0, width + 1, (rows,), generator=g).int() if lengths is None else
                  torch.tensor(lengths, dtype=torch.int32))
    if "p" in what:
        s |= dict(prompt=(s["lengths"] * torch.rand(rows, generator=g)).int(), presence=torch.randn(rows, generator=g),
                  frequency=torch.randn(rows, generator=g))
    if "b" in what:
        s |= dict(bias_ids=torch.randint(-2, min(vocab, 12) + 2, (rows, biases), generator=g).int(),
                  bias=torch.randn((rows, biases), generator=g) * 5)
    if "m" in what:
        words = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=g)
        words[0] = -1
        if rows > 2:
            words[2] = 0
        s |= dict(mask=words.int())
    return {k: v.to(dev) for k, v in s.items()}


def _reference(s):
    rows = s["logits"].shape[0]
    x = values(s["logits"])
    at = {k: v.cpu().numpy() for k, v in s.items() if k != "logits" and isinstance(v, torch.Tensor)}

    def of(name, i, none):
        v = s.get(name, none)
        return float(at[name][i]) if isinstance(v, torch.Tensor) else v

    out, size = [], []
    for i in range(rows):
        n = int(np.clip(at["lengths"][i], 0, at["tokens"].shape[1])) if "lengths" in at else at["tokens"].shape[1] if "tokens" in at else 0
        said = at["tokens"][i, :n] if "tokens" in at else []
        pairs = list(zip(at["bias_ids"][i % len(at["bias_ids"])], at["bias"][i % len(at["bias"])].astype(np.float64))) if "bias" in at else []
        words = at["mask"][i % len(at["mask"])] if "mask" in at else None
        prompt = int(at["prompt"][i]) if "prompt" in at else 0
        settings = of("repetition", i, 1.0), of("presence", i, 0.0), of("frequency", i, 0.0)
        out.append(o.adjust(x[i], said, prompt, *settings, pairs, words))
        # the terms that the result is the sum of
        magnitude = np.abs(o.adjust(x[i], said, prompt, settings[0], 0.0, 0.0, [], None))
        counts = np.zeros(x.shape[1])
        for t in said[max(prompt, 0):]:
            if 0 <= t < len(counts):
                counts[t] += 1
        magnitude += counts * abs(settings[2]) + (counts > 0) * abs(settings[1])
        for t, b in pairs:
            if 0 <= t < len(counts):
                magnitude[t] += abs(b)
        size.append(magnitude)
    return np.stack(out), np.stack(size)


def _check(s, out):
    dtype = s["logits"].dtype
    ref, size = _reference(s)
    got = values(out)
    assert np.array_equal(np.isneginf(ref), np.isneginf(got))
    assert np.array_equal(np.isnan(ref), np.isnan(got))
    fine = np.isfinite(ref)
    # at most five fp32 roundings of the terms, then one of the result
    bound = torch.finfo(dtype).eps / 2 * np.abs(ref) * (1 + 2.0 ** -8) + 6 * 2.0 ** -24 * size + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    err = np.abs(got[fine] - ref[fine])
    assert (err <= bound[fine]).all(), float((err / bound[fine]).max())
    # what nothing names keeps its bits
    bits = {2: torch.int16, 4: torch.int32}[s["logits"].element_size()]
    same = torch.from_numpy((ref == values(s["logits"]))).to(out.device)
    assert torch.equal(out.contiguous().view(bits)[same], s["logits"].contiguous().view(bits)[same])


def _run(s, **more):
    from moss_tts._runtime import sampling

    out = sampling.adjust(s["logits"], **{k: v for k, v in s.items() if k != "logits"}, **more)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["h", "hp", "b", "m", "hb", "bm", "hpbm", ""])
def test_parts(dev, dtype, what):
    s = _inputs(dev, 5, 1024, dtype, what=what)
    print(f"adjust {dtype} {what}", flush=True)
    _check(s, _run(s))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 7), (4, 8), (2, 31), (3, 33), (5, 1025), (3, 8185), (2, 8192), (3, 8193), (2, 20001)])
def test_sizes(dev, dtype, rows, vocab):
    """Rows that begin anywhere among 16 bytes, chunks that end inside a group of eight."""
    s = _inputs(dev, rows, vocab, dtype, seed=vocab)
    print(f"adjust {dtype} {rows} x {vocab}", flush=True)
    _check(s, _run(s))


def test_histories(dev):
    """Lengths of none, one, all and past the width; one token alone; long ones; int32 tokens; a history kept by time."""
    for token_type in (torch.int64, torch.int32):
        s = _inputs(dev, 5, 700, torch.bfloat16, token_type=token_type, lengths=[0, 1, 50, 2 ** 31 - 1, -3])
        _check(s, _run(s))
    s = _inputs(dev, 2, 700, torch.float32, width=1, lengths=[1, 0])
    _check(s, _run(s))
    s = _inputs(dev, 3, 9000, torch.float32, width=5000)
    _check(s, _run(s))
    s["tokens"] = s["tokens"].T.contiguous().T
    assert s["tokens"].stride() == (1, 3)
    _check(s, _run(s))
    del s["lengths"]
    _check(s, _run(s))
    del s["prompt"]
    _check(s, _run(s))
    s["prompt"] = torch.tensor([-5, 2 ** 31 - 1, 4999], dtype=torch.int32, device=dev)
    _check(s, _run(s))


def test_one_token_many_times(dev):
    s = dict(logits=torch.zeros((1, 64), device=dev), tokens=torch.full((1, 30000), 9, device=dev), frequency=0.5, presence=2.0)
    out = _run(s)
    assert float(out[0, 9]) == -15002.0 and float(out.sum()) == -15002.0


def test_numbers_for_all_rows(dev):
    s = _inputs(dev, 4, 300, torch.float16, what="h")
    s |= dict(repetition=1.3, presence=0.5, frequency=0.25)
    _check(s, _run(s))
    s |= dict(presence=torch.rand(4).to(dev))
    _check(s, _run(s))


def test_one_row_for_all(dev):
    """Biases and a mask that all rows share."""
    s = _inputs(dev, 4, 300, torch.bfloat16)
    s["mask"], s["bias"], s["bias_ids"] = s["mask"][1:2], s["bias"][:1], s["bias_ids"][:1]
    _check(s, _run(s))
    s["mask"] = s["mask"].expand(4, -1)
    _check(s, _run(s))


def test_biases_that_name_one_entry(dev):
    """Of equal ids the last holds, whatever the order of the threads; the largest number of biases."""
    n = 65535
    ids = torch.zeros((2, n), dtype=torch.int32, device=dev)
    ids[:, n // 2:] = 1
    ids[:, -1] = 0
    bias = torch.arange(n, dtype=torch.float32, device=dev).repeat(2, 1)
    out = _run(dict(logits=torch.zeros((2, 40), device=dev), bias_ids=ids, bias=bias))
    assert out[0, :3].tolist() == [n - 1.0, n - 2.0, 0.0] and torch.equal(out[0], out[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_places(dev, dtype):
    """Rows apart, a view that begins inside a group, results in place, beside the logits, and where rows begin elsewhere."""
    s = _inputs(dev, 4, 700, dtype)
    wide = torch.full((4, 900), 3.0, dtype=dtype, device=dev)
    for first in (0, 1, 8, 13):
        part = wide[:, first:first + 700]
        part.copy_(s["logits"])
        t = dict(s, logits=part)
        plain = _run(t)
        _check(t, plain)
        beside = torch.full((4, 901), 5.0, dtype=dtype, device=dev)
        for at in (first, first + 3):
            out = beside[:, at:at + 700]
            assert _run(t, out=out).data_ptr() == out.data_ptr()
            assert torch.equal(out, plain)
            assert float(beside[:, :at].sub(5).abs().sum()) == 0 and float(beside[:, at + 700:].sub(5).abs().sum()) == 0
            beside.fill_(5.0)
        kept = wide.clone()
        kept[:, first:first + 700] = plain
        assert _run(t, out=part).data_ptr() == part.data_ptr()
        assert torch.equal(wide, kept)


def test_logits_that_are_not_finite(dev):
    s = _inputs(dev, 3, 100, torch.float32, what="hpb")
    s["logits"][:, ::7] = float("-inf")
    s["logits"][:, 1::9] = float("inf")
    s["logits"][:, 2::11] = float("nan")
    _check(s, _run(s))
    mask = torch.zeros((1, 4), dtype=torch.int32, device=dev)
    assert (_run(dict(s, mask=mask)) == float("-inf")).all()


def test_then_sample(dev):
    """With the row sampler: a masked entry is never drawn, a row without any gives -1, a graph of both follows its inputs
    over replays with other work between."""
    from moss_tts._runtime import sampling

    s = _inputs(dev, 6, 5000, torch.bfloat16, width=64)
    s["mask"][5] = 0
    u = torch.rand(6, device=dev)

    def both():
        x = sampling.adjust(s["logits"], **{k: v for k, v in s.items() if k != "logits"})
        return x, sampling.sample(x, u, temperature=0.8, top_k=50)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x, drawn = both()
    g = torch.Generator().manual_seed(1)
    for i in range(6):
        s["logits"].copy_(torch.randn((6, 5000), generator=g) * 4)
        s["tokens"].copy_(torch.randint(0, 5000, (6, 64), generator=g))
        u.copy_(torch.rand(6, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        _check(s, x)
        again, index = both()
        assert torch.equal(again, x) and torch.equal(index, drawn)
        assert int(drawn[2]) == -1 and int(drawn[5]) == -1
        for r in (0, 1, 3, 4):
            v = int(drawn[r])
            assert int(s["mask"][r, v // 32]) >> (v % 32) & 1


def test_on_another_stream(dev):
    s = _inputs(dev, 8, 3001, torch.float16, width=500)
    want = _run(s)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append(_run(s))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in outs)


def test_refusals(dev):
    from moss_tts._runtime import sampling

    s = _inputs(dev, 4, 300, torch.bfloat16)
    _run(s)
    logits = s["logits"]
    f = torch.ones(4, device=dev)
    for bad in (dict(tokens=s["tokens"][:3]), dict(tokens=s["tokens"].float()), dict(tokens=s["tokens"].cpu()), dict(tokens=s["tokens"][0]),
                dict(tokens=s["tokens"][:, :0]), dict(lengths=s["lengths"].long()), dict(lengths=s["lengths"][:3]), dict(prompt=s["prompt"].cpu()),
                dict(repetition=f[:3]), dict(repetition=f.double()), dict(repetition=0.0), dict(repetition=-1.0), dict(presence=float("nan")),
                dict(frequency=float("inf")), dict(repetition=True), dict(bias=None), dict(bias_ids=None), dict(bias=s["bias"][:, :4]),
                dict(bias=s["bias"].half()), dict(bias_ids=s["bias_ids"].long()), dict(bias=s["bias"][:2], bias_ids=s["bias_ids"][:2]),
                dict(mask=s["mask"][:, :9]), dict(mask=s["mask"].long()), dict(mask=s["mask"][:3]), dict(mask=s["mask"][0]),
                dict(out=logits[:, :299]), dict(out=logits.float()), dict(out=torch.zeros((300, 4), dtype=logits.dtype, device=dev).T),
                dict(out=logits.cpu())):
        with pytest.raises(ValueError):
            sampling.adjust(logits, **{k: v for k, v in {**s, **bad}.items() if k != "logits"})
    for bad in (dict(repetition=1.2), dict(lengths=s["lengths"]), dict(prompt=s["prompt"]), dict(presence=f), dict(frequency=0.1)):
        with pytest.raises(ValueError, match="without tokens"):
            sampling.adjust(logits, **bad)
    for bad in (logits.cpu(), logits.double(), logits[0], logits[:0], logits[:, ::2], logits[:1].expand(4, -1)):
        with pytest.raises(ValueError):
            sampling.adjust(bad)
    wide = torch.zeros((4, 304), dtype=logits.dtype, device=dev)
    with pytest.raises(ValueError, match="overlap"):  # one entry further
        sampling.adjust(wide[:, :300], out=wide[:, 1:301])
    history = torch.zeros((4, 600), dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="overlap"):
        sampling.adjust(logits, tokens=history, out=history.view(torch.bfloat16)[:, :300])


def test_calls_beside_each_other(dev):
    """Many rows: more workgroups than the device holds at once; the result does not depend on what came before."""
    s = _inputs(dev, 700, 1024, torch.bfloat16, width=90)
    first = _run(s)
    _check(s, first)
    for _ in range(3):
        assert torch.equal(_run(s), first)


@pytest.mark.parametrize("rows, vocab, width", [(19, 2041, 300), (17, 2042, 300), (9, 16377, 33000), (16, 16384, 32768), (3, 33000, 32767), (11, 40001, 70)])
def test_every_way_of_counting(dev, rows, vocab, width):
    """Rows of one small workgroup and of several; histories that 15 bits count, and longer ones; more than eight rows, and rows behind
    the last eight."""
    s = _inputs(dev, rows, vocab, torch.bfloat16, width=width, seed=rows, token_type=torch.int32 if rows % 2 else torch.int64)
    s["tokens"][0] = 5
    s["lengths"][0] = width
    s["prompt"][0] = 0
    print(f"adjust {rows} x {vocab}, {width} tokens", flush=True)
    _check(s, _run(s))


def test_a_width_past_everything(dev):
    """Tokens that lie at one place can be any number; the rows of a history are 2^30 at most."""
    from moss_tts._runtime import sampling

    logits = torch.zeros((1, 100), device=dev)
    one = torch.full((1, 1), 7, device=dev)
    with pytest.raises(ValueError, match="2\\^30"):
        sampling.adjust(logits, tokens=one.expand(1, (1 << 30) + 1), frequency=1.0)
    out = sampling.adjust(logits, tokens=one.expand(1, 1 << 30), lengths=torch.tensor([100000], dtype=torch.int32, device=dev), frequency=1.0)
    assert float(out[0, 7]) == -100000.0 and float(out.sum()) == -100000.0
