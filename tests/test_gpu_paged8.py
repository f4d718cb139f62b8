"""GPU: a paged cache in 8 bits: rows written and read back, decode attention over it, against the 64-bit definitions.
Rows that no sequence owns hold e4m3's NaN and scale bytes that are no scale."""
import numpy as np
import pytest
import torch

from oracle import paged as o
from paged_helpers import attention_bound, cache8, cache8_values, values

pytestmark = pytest.mark.gpu

LAYOUTS = [(32, 8, 128), (4, 4, 64), (28, 4, 128), (16, 2, 64), (16, 1, 128), (40, 2, 128), (3, 3, 128)]
DTYPES = [torch.bfloat16, torch.float16]
KIND = {torch.bfloat16: "bf16", torch.float16: "fp16"}


def _close(got, ref, bound, what):
    err = np.abs(values(got).reshape(ref.shape) - ref)
    assert np.isfinite(values(got)).all(), f"{what}: not finite"
    assert (err <= bound).all(), f"{what}: {int((err > bound).sum())} off, worst {float((err / bound).max()):.3g} of the bound"


def _decode(dev, lengths, layout, dtype, page, *, seed=0, scale=None, edit=None, stride=0, interleaved=False):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(seed)
    qh, kh, d = layout
    keys, vals, scales, table, lens = cache8(dev, g, lengths, kh=kh, d=d, page=page, interleaved=interleaved)
    if edit is not None:
        table, lens = edit(table.cpu(), lens.cpu())
        table, lens = table.to(dev), lens.to(dev)
    wide = (torch.randn((len(lengths), qh * d + stride), generator=g) * 1.5).to(dtype).to(dev)
    q = wide[:, :qh * d].unflatten(1, (qh, d))
    print(f"decode8 lengths={lengths} layout={layout} {dtype} page={page}", flush=True)
    ws = paged.decode_workspace(q, keys, table).fill_(float("nan"))
    out = paged.decode_attention(q, keys, vals, table, lens, scale=scale, scales=scales, ws=ws)
    torch.cuda.synchronize()
    args = values(q), cache8_values(keys, scales[0]), cache8_values(vals, scales[1])
    t, n = table.cpu().numpy(), lens.cpu().numpy()
    ref = o.decode_attention(*args, t, n, scale)
    ref_abs = o.decode_attention(args[0], args[1], np.abs(args[2]), t, n, scale)
    bound = attention_bound(args[0], *(np.where(np.abs(a) < 1e6, a, 0.0) for a in args[1:]), ref, ref_abs,
                            d ** -0.5 if scale is None else scale, dtype, False)
    _close(out, ref, bound, "decode8")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_decode_layouts(dev, layout, dtype):
    _decode(dev, [1, 77, 0, 128, 300], layout, dtype, 16)


@pytest.mark.parametrize("page", [16, 32, 64, 256, 4096])
@pytest.mark.parametrize("lengths", [[1], [15, 16, 17, 31, 32, 33], [0], [127, 129, 640, 1000, 255, 2], [0, 0, 500, 0]])
def test_decode_lengths(dev, lengths, page):
    _decode(dev, lengths, (8, 2, 128), torch.bfloat16, page)


def test_decode_many_sequences(dev):
    rng = np.random.default_rng(3)
    lengths = [int(n) for n in rng.integers(0, 60, 150)]
    lengths[0] = lengths[63] = lengths[64] = lengths[149] = 0
    _decode(dev, lengths, (4, 2, 64), torch.bfloat16, 16)


def test_decode_strides_and_scale(dev):
    for stride in (8, 1024):
        _decode(dev, [40, 3, 200], (8, 4, 128), torch.bfloat16, 32, stride=stride, interleaved=True)
    for scale in (0.0, 1.0, -0.3):
        _decode(dev, [40, 3, 200], (8, 4, 64), torch.float16, 32, scale=scale)


def test_decode_pages_that_are_none(dev):
    def edit(table, lens):
        table[0, 1] = -5
        table[1, 0] = 2 ** 31 - 1
        table[2, :] = -(2 ** 31)
        lens[3] = 2 ** 31 - 1
        lens[4] = -7
        return table, lens

    _decode(dev, [100, 130, 90, 64, 30], (8, 2, 128), torch.bfloat16, 16, edit=edit)


def _tables(g, positions, d, dev):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 1e4 ** (-(torch.arange(d, dtype=torch.float64) % (d // 2)) / (d // 2))
    return angle.cos().float().to(dev), angle.sin().float().to(dev)


@pytest.mark.parametrize("layout, dtype", [((32, 8, 128), torch.bfloat16), ((4, 4, 64), torch.float16),
                                           ((28, 4, 128), torch.float16), ((5, 1, 64), torch.bfloat16)])
@pytest.mark.parametrize("normed", [True, False])
def test_write(dev, layout, dtype, normed):
    """Prompts that begin and continue, an empty slot, padding, a token without a position, pages that are none; what is not
    written keeps its bits."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(2)
    qh, kh, d = layout
    new, old = [20, 1, 0, 35, 6, 3], [0, 47, 9, 14, 0, 0]
    lengths = [a + b for a, b in zip(new, old)]
    keys, vals, scales, table, lens = cache8(dev, g, lengths, kh=kh, d=d, page=16, interleaved=normed)
    table[3, 2] = -1
    table[5, 0] = 2 ** 30
    lens[4] = 2
    starts = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device=dev)
    total, width = sum(new) + 4, (qh + 2 * kh) * d
    qkv = (torch.randn((total, width + 64), generator=g) * 2).to(dtype)
    qkv[1, -64 - d:] *= 2.0 ** -9     # rows of other sizes
    qkv[2, -64 - d:] = 0
    qkv[3, -64 - d:] *= 2.0 ** 10
    qkv = qkv.to(dev)[:, :width]
    qw, kw = ((torch.randn(d, generator=g) * 0.3 + 1).to(dtype).to(dev) if normed else None for _ in range(2))
    cos, sin = _tables(g, 40, d, dev)
    q = torch.full((total, qh, d), 5.0, dtype=dtype, device=dev)
    w = [None if t is None else values(t) for t in (qw, kw)]
    before = [t.clone() for t in (keys.view(torch.uint8), vals.view(torch.uint8), *scales)]
    zeros = np.zeros(tuple(keys.shape))
    rest = table.cpu().numpy(), lens.cpu().numpy(), starts.cpu().numpy(), 1e-6, values(q)
    ref = o.qk_rope(values(qkv), *w, values(cos), values(sin), zeros, zeros, *rest)
    # which rows are written: those that ones leave a one in
    ones = o.qk_rope(np.ones(tuple(qkv.shape)), None, None, np.ones((40, d)), np.zeros((40, d)), zeros, zeros, *rest)
    assert paged.qk_rope(qkv, qw, kw, cos, sin, keys, vals, table, lens, 1e-6, starts=starts, out=q, scales=scales) is not None
    torch.cuda.synchronize()
    half = torch.finfo(dtype).eps / 2
    top = np.abs(ref[0]).max(-1, keepdims=True)
    fp32 = (d / 2 + 16) * 2.0 ** -24 * 1.5
    _close(q, ref[0], half * np.abs(ref[0]) + fp32 * top, "q")
    for name, t, scale, x, mark, was, was_scale in (("keys", keys, scales[0], ref[1], ones[1], before[0], before[2]),
                                                    ("values", vals, scales[1], ref[2], ones[2], before[1], before[3])):
        written = mark[..., 0] == 1
        codes, byte = t.view(torch.uint8).cpu().numpy(), scale.cpu().numpy()
        assert np.array_equal(codes[~written], was.cpu().numpy()[~written]), name
        assert np.array_equal(byte[~written], was_scale.cpu().numpy()[~written]), name
        got = o.cache_values(codes[written], byte[written])
        for have, have_byte, row in zip(got, byte[written], x[written]):
            want, want_byte = o.quantize_row(row, KIND[dtype])
            if name == "values":  # nothing is computed before the rounding
                assert have_byte == want_byte and np.array_equal(have, want)
                continue
            # fp32 steps may put the row's largest value on the other side of a power of two's border: then the scale is twice or
            # half; a value is off by half a step of e4m3, at least of its smallest one, and what fp32 leaves
            assert abs(int(have_byte) - want_byte) <= int(abs(np.abs(row).max() / 448 / 2.0 ** np.round(np.log2(np.abs(row).max() / 448)) - 1) < 2 * fp32 if row.any() else 0)
            bound = np.maximum(2.0 ** -4 * np.abs(row), 2.0 ** (float(have_byte) - 127 - 10)) * (1 + 2.0 ** -10) + fp32 * np.abs(row).max() * (1 + 2.0 ** -4)
            assert (np.abs(have - row) <= bound).all(), name


@pytest.mark.parametrize("dtype", DTYPES)
def test_written_keys_are_the_definitions(dev, dtype):
    """Keys of a million values, code for code: the kernel's 64-bit steps are off by 2^-44 of |x cos| + |y sin|, and a border
    lies within that of one value in 10^10."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(12)
    n, d, page = 8192, 128, 64
    qkv = (torch.randn((n, 3 * d), generator=g) * torch.exp2(torch.randint(-6, 7, (n, 1), generator=g).float())).to(dtype).to(dev)
    weight = (torch.randn(d, generator=g) * 0.3 + 1).to(dtype).to(dev)
    cos, sin = _tables(g, n, d, dev)
    keys, vals = (torch.zeros((n // page, 1, page, d), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2))
    scales = tuple(torch.zeros((n // page, 1, page), dtype=torch.uint8, device=dev) for _ in range(2))
    table = torch.arange(n // page, dtype=torch.int32, device=dev)[None]
    eps = float(np.float32(1e-6))
    paged.qk_rope(qkv, weight, weight, cos, sin, keys, vals, table, torch.tensor([n], dtype=torch.int32, device=dev), eps,
                  starts=torch.tensor([0, n], dtype=torch.int32, device=dev), scales=scales)
    torch.cuda.synchronize()
    x = values(qkv)[:, d:2 * d]
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * values(weight)
    x = x * values(cos) + np.concatenate((-x[:, d // 2:], x[:, :d // 2]), -1) * values(sin)
    codes, byte = keys.view(torch.uint8).cpu().numpy().reshape(n, d), scales[0].cpu().numpy().reshape(n)
    got = o.cache_values(codes, byte)
    for i in range(n):
        want, want_byte = o.quantize_row(x[i], KIND[dtype])
        assert byte[i] == want_byte and np.array_equal(got[i], want), i


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_values_that_are_not_finite(dev, dtype):
    """NaN and infinities become NaN and leave the rest of the row alone; the largest numbers of the type are held; rows of
    zeros and of the smallest numbers."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(8)
    d, n = 128, 6
    keys, vals, scales, table, lens = cache8(dev, g, [n], kh=1, d=d, page=16)
    qkv = torch.randn((n, 3 * d), generator=g).to(dtype)
    big = torch.finfo(dtype).max
    qkv[0, 2 * d:2 * d + 3] = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=dtype)
    qkv[1, 2 * d:] = float("inf")
    qkv[2, 2 * d] = big
    qkv[3, 2 * d:] = -big
    qkv[4, 2 * d:] = 0
    qkv[5, 2 * d:] = torch.finfo(dtype).tiny * 0.25  # below the normal range
    x = values(qkv[:, 2 * d:])
    cos, sin = _tables(g, 16, d, dev)
    starts = torch.tensor([0, n], dtype=torch.int32, device=dev)
    paged.qk_rope(qkv.to(dev), None, None, cos, sin, keys, vals, table, lens, 1e-6, starts=starts, scales=scales)
    got = cache8_values(vals, scales[1])[int(table[0, 0]), 0, :n]
    for i in range(n):
        want, byte = o.quantize_row(x[i], KIND[dtype])
        assert int(scales[1][int(table[0, 0]), 0, i]) == byte
        assert np.array_equal(got[i], want, equal_nan=True), i
    k, v = paged.gather(keys, vals, table, lens, starts, n, scales=scales, dtype=dtype)
    assert np.array_equal(values(v)[:, 0], got, equal_nan=True) and np.isfinite(values(v)[2:]).all()


@pytest.mark.parametrize("layout, dtype", [((8, 128), torch.bfloat16), ((2, 64), torch.float16), ((5, 128), torch.float16), ((13, 64), torch.bfloat16)])
@pytest.mark.parametrize("bits", [16, 8])
def test_gather(dev, layout, dtype, bits):
    from moss_tts._runtime import paged
    from paged_helpers import cache

    g = torch.Generator().manual_seed(3)
    kh, d = layout
    new, old = [20, 1, 0, 35, 6, 3, 70], [0, 47, 9, 14, 0, 0, 0]
    lengths = [a + b for a, b in zip(new, old)]
    if bits == 8:
        keys, vals, scales, table, lens = cache8(dev, g, lengths, kh=kh, d=d, page=16, interleaved=kh == 5)
    else:
        keys, vals, table, lens = cache(dev, g, lengths, kh=kh, d=d, page=16, dtype=dtype, interleaved=kh == 5)
        scales = None
    table[3, 2] = -1
    table[5, 0] = 2 ** 30
    lens[4] = 2
    starts = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device=dev)
    total = sum(new) + 9
    out = tuple(torch.full((total, kh, d), 7.0, dtype=dtype, device=dev) for _ in range(2))
    rest = table.cpu().numpy(), lens.cpu().numpy(), starts.cpu().numpy(), values(out[0])
    got = paged.gather(keys, vals, table, lens, starts, total, scales=scales, out=out)
    assert got[0].data_ptr() == out[0].data_ptr() and got[1].data_ptr() == out[1].data_ptr()
    for t, pages in zip(got, (keys, vals) if bits == 16 else ((keys, scales[0]), (vals, scales[1]))):
        assert np.array_equal(values(t), o.gather(values(pages) if bits == 16 else cache8_values(*pages), *rest))
    fresh = paged.gather(keys, vals, table, lens, starts, total, scales=scales, dtype=dtype)
    assert torch.equal(fresh[0][:sum(new)], got[0][:sum(new)]) and torch.equal(fresh[1][:sum(new)], got[1][:sum(new)])


def test_gather_many_sequences(dev):
    """More sequences than a wave counts at once."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(4)
    lengths = [int(n) for n in np.random.default_rng(3).integers(0, 40, 150)]
    keys, vals, scales, table, lens = cache8(dev, g, lengths, kh=2, d=64, page=16)
    starts = torch.tensor([0, *np.cumsum(lengths)], dtype=torch.int32, device=dev)
    k, v = paged.gather(keys, vals, table, lens, starts, sum(lengths), scales=scales)
    before = np.zeros((sum(lengths), 2, 64))
    for t, pages in ((k, (keys, scales[0])), (v, (vals, scales[1]))):
        assert np.array_equal(values(t), o.gather(cache8_values(*pages), table.cpu().numpy(), lens.cpu().numpy(), starts.cpu().numpy(), before))


def test_values_are_exact_in_either_type(dev):
    """Every code at every exponent that a row is written with, as the attentions and gather read it."""
    from moss_tts._runtime import paged

    for dtype in DTYPES:
        low, high = o.EXPONENTS[KIND[dtype]]
        exponents = list(range(low, high + 1))
        codes = torch.arange(256, dtype=torch.uint8).view(2, 128)
        rows = 2 * len(exponents)
        pages = -(-rows // 16)
        data = torch.zeros((pages * 16, 128), dtype=torch.uint8)
        byte = torch.full((pages * 16,), 127, dtype=torch.uint8)
        for i, e in enumerate(exponents):
            data[2 * i:2 * i + 2] = codes
            byte[2 * i:2 * i + 2] = e + 127
        most = 240 if high == 8 else 240
        top = o.cache_values(data.numpy(), byte.numpy())
        keys = data.view(pages, 1, 16, 128).to(dev)
        scale = byte.view(pages, 1, 16).to(dev)
        table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
        lens = torch.tensor([rows], dtype=torch.int32, device=dev)
        starts = torch.tensor([0, rows], dtype=torch.int32, device=dev)
        k, v = paged.gather(keys.view(torch.float8_e4m3fn), keys.clone().view(torch.float8_e4m3fn), table, lens, starts, rows,
                            scales=(scale, scale.clone()), dtype=dtype)
        want = top[:rows]
        written = np.abs(want) <= most * 2.0 ** high  # the codes that a row is written with
        written |= np.isnan(want)
        for t in (k, v):
            got = values(t)[:, 0]
            assert np.array_equal(got[written], want[written], equal_nan=True)


def test_refusals(dev):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(0)
    keys, vals, scales, table, lens = cache8(dev, g, [20, 30], kh=2, d=64, page=16)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=dev)
    ok = dict(scales=scales)
    paged.decode_attention(q, keys, vals, table, lens, **ok)
    starts = torch.tensor([0, 20, 50], dtype=torch.int32, device=dev)
    for bad in (None, scales[0], (scales[0],), (scales[0], scales[1].short()), (scales[0], scales[1][:, :1]), (scales[0], scales[1].cpu()),
                (scales[0], scales[1][..., ::2]), (scales[0][:-1], scales[1][:-1])):
        with pytest.raises(ValueError):
            paged.decode_attention(q, keys, vals, table, lens, scales=bad)
        with pytest.raises(ValueError):
            paged.gather(keys, vals, table, lens, starts, 50, scales=bad)
    with pytest.raises(ValueError, match="float8"):
        paged.decode_attention(q, keys.view(torch.uint8), vals, table, lens, **ok)
    with pytest.raises(ValueError):
        paged.decode_attention(q, keys, vals, table, lens, scales=scales, out=vals.view(torch.bfloat16).flatten()[:512].view(2, 256))
    qkv = torch.zeros((2, 8 * 64), dtype=torch.bfloat16, device=dev)
    cos = torch.ones((64, 64), device=dev)
    rope = [qkv, None, None, cos, cos.clone(), keys, vals, table, lens, 1e-6]
    paged.qk_rope(*rope, scales=scales)
    with pytest.raises(ValueError, match="share memory"):
        paged.qk_rope(*rope, scales=(scales[0], scales[0]))
    inside = keys.view(torch.uint8).flatten()[:scales[0].numel()].view(scales[0].shape)
    with pytest.raises(ValueError, match="share memory"):
        paged.qk_rope(*rope, scales=(scales[0], inside))
    with pytest.raises(ValueError, match="share memory"):
        paged.qk_rope(*rope[:5], keys, keys, *rope[7:], scales=scales)
    for tokens in (0, 1 << 24, 2.0):
        with pytest.raises(ValueError):
            paged.gather(keys, vals, table, lens, starts, tokens, scales=scales)
    out = tuple(torch.zeros((50, 2, 64), dtype=torch.bfloat16, device=dev) for _ in range(2))
    for bad in (out[0], (out[0], out[0]), (out[0], out[1][:49]), (out[0].half(), out[1]), (out[0], out[1].float())):
        with pytest.raises(ValueError):
            paged.gather(keys, vals, table, lens, starts, 50, scales=scales, out=bad)
    with pytest.raises(ValueError):
        paged.gather(keys, vals, table, lens, starts, 50, scales=scales, dtype=torch.float32)
    with pytest.raises(ValueError):
        paged.gather(keys, vals, table, lens, None, 50, scales=scales)


def test_captured(dev):
    """A step's write and attention in a graph that follows the batch, on another stream, replayed with other work between."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(6)
    qh, kh, d, n = 8, 2, 128, 3
    keys, vals, scales, table, lens = cache8(dev, g, [33, 5, 100], kh=kh, d=d, page=16, spare=12, width=12)
    free = [p for p in range(keys.shape[0]) if p not in set(table.cpu().flatten().tolist())]
    qkv = torch.zeros((n, (qh + 2 * kh) * d), dtype=torch.bfloat16, device=dev)
    cos, sin = _tables(g, 256, d, dev)

    def step(k, v, s):
        q = paged.qk_rope(qkv, None, None, cos, sin, k, v, table, lens, 1e-6, scales=s)
        return paged.decode_attention(q, k, v, table, lens, scales=s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(keys.clone(), vals.clone(), tuple(t.clone() for t in scales))
    torch.cuda.current_stream().wait_stream(side)
    mirror = keys.clone(), vals.clone(), tuple(t.clone() for t in scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(keys, vals, scales)
    for i in range(20):
        for b in range(n):
            length = int(lens[b])
            if length % 16 == 0:
                table[b, length // 16] = free.pop()
            lens[b] = length + 1
        qkv.copy_((torch.randn(qkv.shape, generator=g) * 2).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(step(*mirror), out), i
        assert torch.equal(mirror[0].view(torch.uint8), keys.view(torch.uint8)) and torch.equal(mirror[2][1], scales[1])


def _prompt(dev, new, old, layout, dtype, page, *, seed=0, pad=0, edit=None, stride=0, scale=None, interleaved=False):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(seed)
    qh, kh, d = layout
    lengths = [a + b for a, b in zip(new, old)]
    keys, vals, scales, table, lens = cache8(dev, g, lengths, kh=kh, d=d, page=page, interleaved=interleaved)
    if edit is not None:
        table, lens = edit(table.cpu(), lens.cpu())
        table, lens = table.to(dev), lens.to(dev)
    starts = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device=dev)
    total = sum(new) + pad
    wide = (torch.randn((total, qh * d + stride), generator=g) * 1.5).to(dtype).to(dev)
    q = wide[:, :qh * d].unflatten(1, (qh, d))
    out = torch.full((total, qh * d), 7.0, dtype=dtype, device=dev)
    before = values(out)
    print(f"prompt8 new={new} old={old} layout={layout} {dtype} page={page}", flush=True)
    assert paged.prompt_attention(q, keys, vals, table, lens, starts, scale=scale, out=out, scales=scales) is out
    torch.cuda.synchronize()
    args = values(q), cache8_values(keys, scales[0]), cache8_values(vals, scales[1])
    rest = table.cpu().numpy(), lens.cpu().numpy(), starts.cpu().numpy(), before, scale
    ref = o.prompt_attention(*args, *rest)
    ref_abs = o.prompt_attention(args[0], args[1], np.abs(args[2]), *rest)
    bound = attention_bound(args[0], *(np.where(np.abs(a) < 1e6, a, 0.0) for a in args[1:]), ref, ref_abs,
                            d ** -0.5 if scale is None else scale, dtype, True)
    _close(out, ref, bound, "prompt8")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_prompt_layouts(dev, layout, dtype):
    _prompt(dev, [33, 1, 0, 70], [0, 9, 5, 40], layout, dtype, 16, pad=5)


@pytest.mark.parametrize("page", [16, 64, 512])
@pytest.mark.parametrize("new, old", [([1], [0]), ([1], [130]), ([31, 32, 33, 63, 64, 65], [0] * 6), ([5, 129], [300, 64]),
                                      ([2, 3, 1, 1, 200], [500, 0, 0, 77, 1])])
def test_prompt_lengths(dev, new, old, page):
    _prompt(dev, new, old, (8, 2, 128), torch.bfloat16, page)


@pytest.mark.parametrize("layout, dtype", [((32, 8, 128), torch.bfloat16), ((32, 8, 128), torch.float16),
                                           ((28, 4, 128), torch.bfloat16), ((36, 12, 64), torch.bfloat16)])
def test_prompt_large(dev, layout, dtype):
    """Enough rows for the large tiles, with ends inside tiles and blocks."""
    _prompt(dev, [421, 77, 203], [0, 150, 9], layout, dtype, 32, pad=3)


def test_prompt_many_sequences_strides_and_scale(dev):
    rng = np.random.default_rng(4)
    new = [int(n) for n in rng.integers(0, 6, 140)]
    new[0] = new[64] = new[139] = 0
    _prompt(dev, new, [int(n) for n in rng.integers(0, 40, 140)], (4, 2, 64), torch.bfloat16, 16)
    _prompt(dev, [40, 3, 20], [0, 8, 100], (8, 4, 128), torch.bfloat16, 32, stride=512, interleaved=True)
    _prompt(dev, [40, 3, 20], [0, 8, 100], (8, 4, 64), torch.float16, 32, scale=-0.4)


def test_prompt_rows_without_keys(dev):
    def edit(table, lens):
        table[0, 1] = -1
        table[1, :] = 10 ** 9
        table[2, 0] = -3
        lens[3] = 12
        lens[4] = -4
        return table, lens

    _prompt(dev, [20, 10, 70, 30, 5], [60, 20, 0, 0, 0], (8, 2, 128), torch.bfloat16, 16, edit=edit)
    _prompt(dev, [300, 290, 170, 200, 90], [60, 20, 0, 0, 0], (32, 8, 128), torch.bfloat16, 16, edit=edit)


@pytest.mark.parametrize("tokens", [90, 700])
def test_prompt_values_behind_a_token(dev, tokens):
    """A row of NaN reaches the tokens at and behind it, and none before it."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(9)
    qh, kh, d, bad = 32, 8, 128, 37
    keys, vals, scales, table, lens = cache8(dev, g, [tokens], kh=kh, d=d, page=16)
    q = torch.randn((tokens, qh, d), generator=g).bfloat16().to(dev)
    starts = torch.tensor([0, tokens], dtype=torch.int32, device=dev)
    vals.view(torch.uint8)[int(table[0, bad // 16]), :, bad % 16] = 0x7f
    got = paged.prompt_attention(q, keys, vals, table, lens, starts, scales=scales)
    assert torch.isnan(got[bad:]).all()
    args = values(q), cache8_values(keys, scales[0]), cache8_values(vals, scales[1])
    table_, lens_ = table.cpu().numpy(), np.array([bad])
    first = np.array([0, bad])
    before = np.zeros((bad, qh * d))
    ref = o.prompt_attention(args[0][:bad], *args[1:], table_, lens_, first, before)
    ref_abs = o.prompt_attention(args[0][:bad], args[1], np.abs(args[2]), table_, lens_, first, before)
    bound = attention_bound(args[0], *(np.where(np.abs(a) < 1e6, a, 0.0) for a in args[1:]), ref, ref_abs, d ** -0.5, torch.bfloat16, True)
    _close(got[:bad], ref, bound, "before the row")


@pytest.mark.parametrize("layout, new, old", [((32, 8, 128), [1500, 700], [0, 9]), ((36, 12, 64), [1300, 200, 450], [30, 0, 700])])
def test_prompt_whole_tiles(dev, layout, new, old):
    """More tokens than the halved tiles are for, with parts of a tile's keys joined."""
    from moss_tts._runtime import paged
    from paged_helpers import attend_all

    g = torch.Generator().manual_seed(7)
    qh, kh, d = layout
    keys, vals, scales, table, lens = cache8(dev, g, [a + b for a, b in zip(new, old)], kh=kh, d=d, page=64)
    q = (torch.randn((sum(new), qh, d), generator=g) * 1.5).bfloat16().to(dev)
    starts = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device=dev)
    out = paged.prompt_attention(q, keys, vals, table, lens, starts, scales=scales)
    wide = [torch.nan_to_num(torch.from_numpy(np.where(np.abs(cache8_values(*t)) < 1e6, cache8_values(*t), 0.0))).to(dev)
            for t in ((keys, scales[0]), (vals, scales[1]))]
    rest = table, lens, starts.tolist(), torch.zeros_like(out), d ** -0.5
    ref, ref_abs = attend_all(q, *wide, *rest), attend_all(q, wide[0], wide[1].abs(), *rest)
    bound = attention_bound(values(q), values(wide[0]), values(wide[1]), values(ref), values(ref_abs), d ** -0.5, torch.bfloat16, True)
    _close(out, values(ref), bound, "prompt8")
