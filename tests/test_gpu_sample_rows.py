"""GPU: ``sampling.sample`` against the 64-bit definition (``oracle.paged.sample``): whole numbers, so equal, unless a
border of the distribution lies within the kernel's sums' error (2^-45 of the largest weight an entry) of a decision."""
import math

import numpy as np
import pytest
import torch

from oracle import paged as o

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _logits(rows, vocab, g, dtype, kind):
    if kind == "ties":  # few distinct values
        return torch.randint(-3, 4, (rows, vocab), generator=g).to(dtype)
    if kind == "equal":
        return torch.full((rows, vocab), 1.5).to(dtype)
    if kind == "near_zero":  # many distinct keys in a narrow range
        return (torch.randn((rows, vocab), generator=g) * 1e-3).to(dtype)
    x = torch.randn((rows, vocab), generator=g) * 2
    if kind == "negative":
        return (x - 20).to(dtype)
    if kind == "between":  # a few entries above, most around 0
        x = x * 4e-3
        x[:, ::37] += 0.05
        return x.to(dtype)
    if kind == "far":
        return (x * 300).to(dtype)
    if kind == "masked":  # all but a few entries masked, by -inf or the type's lowest value
        keep = torch.rand((rows, vocab), generator=g) < 4 / vocab
        keep[:, 0] = True
        low = torch.full((rows, vocab), -math.inf)
        low[::2] = torch.finfo(dtype).min
        return torch.where(keep, x, low).to(dtype)
    if kind == "special":
        x[0, 1::3] = math.nan
        x[1, vocab // 2] = math.inf
        x[2, 1:] = -math.inf
        x[3] = -math.inf
        x[4] = math.nan
        x[5, ::2] = math.inf
        return x.to(dtype)
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 5), generator=g), torch.rand((rows, 5), generator=g) * 10)
    return x.to(dtype)


def _check(logits, u, settings, dev, vocab=None, padded=0):
    from moss_tts._runtime import sampling

    rows, entries = logits.shape
    wide = torch.full((rows, entries + padded), 99.0, dtype=logits.dtype)
    wide[:, :entries] = logits
    view = wide.to(dev)[:, :entries]
    print(f"sample {tuple(logits.shape)} {logits.dtype} vocab={vocab} padded={padded}", flush=True)
    got = sampling.sample(view, u.to(dev), vocab=vocab,
                          **{k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in settings.items()}).cpu()
    x = logits.double().numpy()[:, :vocab]
    error = x.shape[1] * 2.0 ** -44
    full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **settings)
    for i in range(rows):
        at = {k: v[i].item() if isinstance(v, torch.Tensor) else v for k, v in full.items()}
        # the settings are fp32 numbers
        at = {k: float(np.float32(v)) if k != "top_k" else v for k, v in at.items()}
        want, near = o.sample(x[i], float(u[i]), at["temperature"], at["top_k"], at["top_p"], at["min_p"])
        if near == 0 or near > error:
            assert got[i].item() == want, f"row {i}: {got[i].item()} for {want} ({at}, u={float(u[i])}, border {near:.3g} away)"


def _mixed(rows, g):
    def pick(v, dtype):
        return torch.tensor(v, dtype=dtype)[torch.randint(0, len(v), (rows,), generator=g)]

    return dict(temperature=pick([0.0, 0.3, 1.0, 1.7, 4.0], torch.float32), top_k=pick([0, 1, 2, 25, 300, 10 ** 9], torch.int32),
                top_p=pick([0.0, 0.1, 0.8, 0.95, 1.0], torch.float32), min_p=pick([0.0, 0.0, 0.02, 0.5, 1.0], torch.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 63, 512, 513, 1024, 2041, 2048, 2049, 4096, 8191, 9000])
def test_sizes(dev, dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    _check(_logits(24, vocab, g, dtype, "plain"), torch.rand(24, generator=g), _mixed(24, g), dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["ties", "equal", "near_zero", "masked", "negative", "between", "far"])
@pytest.mark.parametrize("vocab", [300, 1000, 2000, 4100, 30000])
def test_hard_rows(dev, dtype, kind, vocab):
    g = torch.Generator().manual_seed(1)
    _check(_logits(40, vocab, g, dtype, kind), torch.rand(40, generator=g), _mixed(40, g), dev)


@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "near_zero", "masked", "negative", "between", "far", "special"])
@pytest.mark.parametrize("vocab, padded", [(2049, 0), (4100, 3), (30000, 0)])
def test_many_long_rows(dev, kind, vocab, padded):
    """More long rows than are drawn by several workgroups each; rows whose border lies between their key bins, rows without
    key bins, rows without anything to cut."""
    g = torch.Generator().manual_seed(10)
    _check(_logits(40, vocab, g, torch.bfloat16, kind), torch.rand(40, generator=g), _mixed(40, g), dev, padded=padded)


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values(dev, dtype):
    g = torch.Generator().manual_seed(2)
    x = _logits(6, 700, g, dtype, "special")
    for settings in (dict(), dict(temperature=0.0), dict(top_k=5), dict(top_p=0.5), dict(min_p=0.3), dict(top_k=300, top_p=0.3)):
        _check(x, torch.rand(6, generator=g), settings, dev)


def test_signed_zero_and_lowest(dev):
    """-0 and 0 are equal logits; the type's lowest value everywhere is an ordinary row."""
    x = torch.tensor([[-0.0, 0.0, -0.0, -5.0], [0.0, -0.0, 0.0, -5.0]]).bfloat16()
    for k in (1, 2, 3):
        _check(x, torch.tensor([0.99, 0.4]), dict(top_k=k), dev)
    low = torch.full((2, 40), torch.finfo(torch.bfloat16).min).bfloat16()
    _check(low, torch.tensor([0.99, 0.4]), dict(top_k=7), dev)
    _check(low, torch.tensor([0.99, 0.4]), dict(temperature=1e30), dev)


@pytest.mark.parametrize("dtype", DTYPES)
def test_text_vocabulary(dev, dtype):
    g = torch.Generator().manual_seed(3)
    _check(_logits(16, 151936, g, dtype, "plain"), torch.rand(16, generator=g), _mixed(16, g), dev)
    _check(_logits(2, 151936, g, dtype, "equal"), torch.rand(2, generator=g), dict(top_k=1000, top_p=0.5), dev)
    _check(_logits(4, 151936, g, dtype, "between"), torch.rand(4, generator=g), dict(top_p=0.5), dev)


def test_strides_and_vocab(dev):
    g = torch.Generator().manual_seed(4)
    x = _logits(9, 1025, g, torch.bfloat16, "plain")
    for padded in (0, 1, 7, 8):
        _check(x, torch.rand(9, generator=g), dict(top_k=25, top_p=0.8, temperature=1.7), dev, vocab=1024, padded=padded)


def test_uniform_at_its_ends(dev):
    """u = 0 draws the first kept entry, u = 1 and above the last, a negative one or NaN the first."""
    from moss_tts._runtime import sampling

    x = torch.tensor([[-math.inf, 1.0, 3.0, 2.0, -math.inf]] * 5, device=dev).bfloat16()
    u = torch.tensor([0.0, 1.0, 7.0, -1.0, math.nan], device=dev)
    assert sampling.sample(x, u).tolist() == [1, 3, 3, 1, 1]
    assert sampling.sample(x, u, top_k=2).tolist() == [2, 3, 3, 2, 2]


def test_distribution(dev):
    """Evenly spaced u count each kept entry in proportion to its weight."""
    from moss_tts._runtime import sampling

    n = 4096
    w = torch.tensor([1.0, 2.0, 5.0, 8.0], device=dev)
    u = (torch.arange(n, device=dev, dtype=torch.float32) + 0.5) / n
    got = torch.bincount(sampling.sample(w.log().expand(n, 4).contiguous(), u), minlength=4)
    assert (got - n * w / 16).abs().max() <= 1


def test_graph_reads_settings_at_replay(dev):
    from moss_tts._runtime import sampling

    g = torch.Generator().manual_seed(5)
    x = _logits(8, 2000, g, torch.bfloat16, "plain").to(dev)
    u = torch.rand(8, generator=g).to(dev)
    s = {k: v.to(dev) for k, v in _mixed(8, g).items()}
    sampling.sample(x, u, **s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sampling.sample(x, u, **s)
    for _ in range(4):
        u.copy_(torch.rand(8, generator=g))
        for k, v in _mixed(8, g).items():
            s[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, sampling.sample(x, u, **s))
        torch.cuda.synchronize()


@pytest.mark.parametrize("rows, vocab", [(2, 40000), (70, 9000), (1100, 2500)])
def test_long_rows_graph_and_kept_workspace(dev, rows, vocab):
    """Several launches in one graph, with a workspace of a larger call's, new logits and settings between the replays; eager
    work and synchronizations between them too."""
    from moss_tts._runtime import sampling

    g = torch.Generator().manual_seed(6)
    x = _logits(rows, vocab, g, torch.bfloat16, "plain").to(dev)
    u = torch.rand(rows, generator=g).to(dev)
    s = {k: v.to(dev) for k, v in _mixed(rows, g).items()}
    ws = sampling.sample_workspace(rows + 3, vocab + 7000, dev).fill_(math.nan)
    sampling.sample(x, u, **s, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sampling.sample(x, u, **s, ws=ws)
    for _ in range(4):
        x.copy_(_logits(rows, vocab, g, torch.bfloat16, "plain"))
        u.copy_(torch.rand(rows, generator=g))
        for k, v in _mixed(rows, g).items():
            s[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, sampling.sample(x, u, **s))
        torch.cuda.synchronize()


def test_kept_workspace_of_more_rows(dev):
    """65 rows are read by fewer workgroups than 64."""
    from moss_tts._runtime import sampling

    g = torch.Generator().manual_seed(7)
    ws = sampling.sample_workspace(65, 151936, dev)
    x = _logits(64, 151936, g, torch.bfloat16, "plain").to(dev)
    u = torch.rand(64, generator=g).to(dev)
    assert torch.equal(sampling.sample(x, u, top_k=50, top_p=0.9, ws=ws), sampling.sample(x, u, top_k=50, top_p=0.9))


def test_calls_on_two_streams(dev):
    from moss_tts._runtime import sampling

    g = torch.Generator().manual_seed(8)
    sets = [(_logits(n, 30000, g, torch.bfloat16, "plain").to(dev), torch.rand(n, generator=g).to(dev)) for n in (3, 40)]
    alone = [sampling.sample(*s, top_k=100, top_p=0.95) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(sampling.sample(*sets[i], top_k=100, top_p=0.95))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, alone[i]) for y in outs[i])


@pytest.mark.parametrize("dtype", DTYPES)
def test_largest_vocabulary(dev, dtype):
    g = torch.Generator().manual_seed(9)
    _check(_logits(6, 1 << 19, g, dtype, "plain"), torch.rand(6, generator=g), _mixed(6, g), dev)


def test_refusals(dev):
    from moss_tts._runtime import sampling

    x = torch.zeros((3, 10), dtype=torch.bfloat16, device=dev)
    u = torch.zeros(3, device=dev)
    assert sampling.sample(x, u).tolist() == [0, 0, 0]
    for match, a, k in (("logits must be a bf16", (x.double(), u), {}), ("logits must be a CUDA", (x.cpu(), u), {}),
                        ("rows, entries", (x[0], u), {}), ("contiguous", (x.t().contiguous().t(), u), {}),
                        ("overlap", (x[:1].expand(3, 10), u), {}), ("uniform must be", (x, u.double()), {}),
                        ("one number a row", (x, u[:2]), {}), ("temperature must be", (x, u), dict(temperature=u.double())),
                        ("one value a row", (x, u), dict(top_p=u[:2])), ("top_k must be", (x, u), dict(top_k=u)),
                        ("non-negative", (x, u), dict(top_k=-1)), ("non-negative", (x, u), dict(top_k=1.5)),
                        ("min_p", (x, u), dict(min_p=1.5)), ("top_p", (x, u), dict(top_p=-0.1)),
                        ("temperature", (x, u), dict(temperature=math.nan)), ("vocab", (x, u), dict(vocab=11)),
                        ("vocab", (x, u), dict(vocab=0)), ("out must hold", (x, u), dict(out=torch.zeros(2, dtype=torch.int64, device=dev)))):
        with pytest.raises(ValueError, match=match):
            sampling.sample(*a, **k)
    x = torch.zeros((3, 3000), dtype=torch.float32, device=dev)
    ws = sampling.sample_workspace(3, 3000, dev)
    for match, bad in (("workspace too small", ws[:-4]), ("16-byte", torch.zeros(ws.numel() + 4, device=dev)[1:]),
                       ("must not overlap", torch.zeros(ws.numel() + 9000, device=dev))):
        with pytest.raises(ValueError, match=match):
            if match == "must not overlap":
                sampling.sample(bad[-9000:].view(3, 3000), u, ws=bad)
            else:
                sampling.sample(x, u, ws=bad)
