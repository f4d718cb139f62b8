"""GPU: attention, rotary embedding and page writes over a paged cache against the 64-bit definitions
(``oracle.paged``), at the sizes and masks where they can go wrong.  Rows that no sequence owns hold NaN throughout."""
import numpy as np
import pytest
import torch

from oracle import paged as o
from paged_helpers import attention_bound, cache, values

pytestmark = pytest.mark.gpu

LAYOUTS = [(32, 8, 128), (4, 4, 64), (28, 4, 128), (16, 2, 64), (16, 1, 128), (40, 2, 128), (3, 3, 128)]
DTYPES = [torch.bfloat16, torch.float16]


def _close(got, ref, bound, what):
    err = np.abs(values(got).reshape(ref.shape) - ref)
    assert np.isfinite(values(got)).all(), f"{what}: not finite"
    assert (err <= bound).all(), f"{what}: {int((err > bound).sum())} off, worst {float((err / bound).max()):.3g} of the bound"


def _decode(dev, lengths, layout, dtype, page, *, seed=0, scale=None, edit=None, stride=0, interleaved=False, ws=False):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(seed)
    qh, kh, d = layout
    keys, vals, table, lens = cache(dev, g, lengths, kh=kh, d=d, page=page, dtype=dtype, interleaved=interleaved)
    if edit is not None:
        table, lens = edit(table.cpu(), lens.cpu())
        table, lens = table.to(dev), lens.to(dev)
    wide = (torch.randn((len(lengths), qh * d + stride), generator=g) * 1.5).to(dtype).to(dev)
    q = wide[:, :qh * d].unflatten(1, (qh, d))
    print(f"decode lengths={lengths} layout={layout} {dtype} page={page}", flush=True)
    w = paged.decode_workspace(q, keys, table).fill_(float("nan")) if ws else None
    out = paged.decode_attention(q, keys, vals, table, lens, scale=scale, ws=w)
    torch.cuda.synchronize()
    args = values(q), values(keys), values(vals)
    t, n = table.cpu().numpy(), lens.cpu().numpy()
    ref = o.decode_attention(*args, t, n, scale)
    ref_abs = o.decode_attention(args[0], args[1], np.abs(args[2]), t, n, scale)
    bound = attention_bound(*args, ref, ref_abs, d ** -0.5 if scale is None else scale, dtype, False)
    _close(out, ref, bound, "decode")
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_decode_layouts(dev, layout, dtype):
    _decode(dev, [1, 77, 0, 128, 300], layout, dtype, 16)


@pytest.mark.parametrize("page", [16, 32, 64, 256, 4096])
@pytest.mark.parametrize("lengths", [[1], [15, 16, 17, 31, 32, 33], [0], [127, 129, 640, 1000, 255, 2], [0, 0, 500, 0]])
def test_decode_lengths(dev, lengths, page):
    _decode(dev, lengths, (8, 2, 128), torch.bfloat16, page, ws=True)


def test_decode_many_sequences(dev):
    """More sequences than a wave counts at once, some empty."""
    rng = np.random.default_rng(3)
    lengths = [int(n) for n in rng.integers(0, 60, 150)]
    lengths[0] = lengths[63] = lengths[64] = lengths[149] = 0
    _decode(dev, lengths, (4, 2, 64), torch.bfloat16, 16)


def test_decode_strides(dev):
    for stride in (8, 1024):
        _decode(dev, [40, 3, 200], (8, 4, 128), torch.bfloat16, 32, stride=stride, interleaved=True)


def test_decode_scale(dev):
    for scale in (0.0, 1.0, -0.3):
        _decode(dev, [40, 3, 200], (8, 4, 64), torch.float16, 32, scale=scale)


def test_decode_pages_that_are_none(dev):
    """Entries outside the cache are rows that take no part; all of them: zeros.  A length past the table is cut."""
    def edit(table, lens):
        table[0, 1] = -5
        table[1, 0] = 2 ** 31 - 1
        table[1, 3] = 10 ** 6
        table[2, :] = -(2 ** 31)
        return table, lens

    _decode(dev, [100, 130, 90], (8, 2, 128), torch.bfloat16, 16, edit=edit)

    def longer(table, lens):  # the rows behind a sequence have no page: -1 entries
        lens[0] = 2 ** 31 - 1
        lens[1] = -7
        return table, lens

    _decode(dev, [64, 30, 9], (8, 2, 128), torch.bfloat16, 16, edit=longer)


def test_decode_large_scores(dev):
    """Scores far apart: one row takes all the weight, rows before it must be forgotten exactly."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(1)
    keys, vals, table, lens = cache(dev, g, [700], kh=1, d=128, page=16, dtype=torch.bfloat16)
    q = torch.ones((1, 2, 128), dtype=torch.bfloat16, device=dev)
    row = 650
    keys[table[0, row // 16].long(), 0, row % 16] = 100.0
    out = paged.decode_attention(q, keys, vals, table, lens)
    v = vals[table[0, row // 16].long(), 0, row % 16]
    assert torch.equal(out.view(2, 128), torch.stack([v, v]))


def test_decode_repeats_bit_for_bit(dev):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(5)
    keys, vals, table, lens = cache(dev, g, [900, 20, 3000], kh=2, d=128, page=64, dtype=torch.bfloat16)
    q = torch.randn((3, 8, 128), generator=g).bfloat16().to(dev)
    first = paged.decode_attention(q, keys, vals, table, lens)
    for _ in range(3):
        assert torch.equal(paged.decode_attention(q, keys, vals, table, lens), first)


def _prompt(dev, new, old, layout, dtype, page, *, seed=0, pad=0, edit=None, stride=0, scale=None, interleaved=False):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(seed)
    qh, kh, d = layout
    lengths = [a + b for a, b in zip(new, old)]
    keys, vals, table, lens = cache(dev, g, lengths, kh=kh, d=d, page=page, dtype=dtype, interleaved=interleaved)
    if edit is not None:
        table, lens = edit(table.cpu(), lens.cpu())
        table, lens = table.to(dev), lens.to(dev)
    starts = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device=dev)
    total = sum(new) + pad
    wide = (torch.randn((total, qh * d + stride), generator=g) * 1.5).to(dtype).to(dev)
    q = wide[:, :qh * d].unflatten(1, (qh, d))
    out = torch.full((total, qh * d), 7.0, dtype=dtype, device=dev)
    before = values(out)
    print(f"prompt new={new} old={old} layout={layout} {dtype} page={page}", flush=True)
    assert paged.prompt_attention(q, keys, vals, table, lens, starts, scale=scale, out=out).data_ptr() == out.data_ptr()
    torch.cuda.synchronize()
    args = values(q), values(keys), values(vals)
    rest = table.cpu().numpy(), lens.cpu().numpy(), starts.cpu().numpy(), before, scale
    ref = o.prompt_attention(*args, *rest)
    ref_abs = o.prompt_attention(args[0], args[1], np.abs(args[2]), *rest)
    bound = attention_bound(*args, ref, ref_abs, d ** -0.5 if scale is None else scale, dtype, True)
    _close(out, ref, bound, "prompt")
    return out


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


def test_prompt_many_sequences(dev):
    rng = np.random.default_rng(4)
    new = [int(n) for n in rng.integers(0, 6, 140)]
    new[0] = new[64] = new[139] = 0
    old = [int(n) for n in rng.integers(0, 40, 140)]
    _prompt(dev, new, old, (4, 2, 64), torch.bfloat16, 16)


def test_prompt_strides_and_scale(dev):
    _prompt(dev, [40, 3, 20], [0, 8, 100], (8, 4, 128), torch.bfloat16, 32, stride=512, interleaved=True)
    _prompt(dev, [40, 3, 20], [0, 8, 100], (8, 4, 64), torch.float16, 32, scale=-0.4)


def test_prompt_rows_without_keys(dev):
    """Pages that are none inside a prefix and under the new tokens, and more new tokens than the length says."""
    def edit(table, lens):
        table[0, 1] = -1
        table[1, :] = 10 ** 9
        table[2, 0] = -3
        lens[3] = 12
        lens[4] = -4
        return table, lens

    _prompt(dev, [20, 10, 70, 30, 5], [60, 20, 0, 0, 0], (8, 2, 128), torch.bfloat16, 16, edit=edit)
    _prompt(dev, [300, 290, 170, 200, 90], [60, 20, 0, 0, 0], (32, 8, 128), torch.bfloat16, 16, edit=edit)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("layout, dtype", [((32, 8, 128), torch.bfloat16), ((4, 4, 64), torch.float16),
                                           ((28, 4, 128), torch.float16), ((5, 1, 64), torch.bfloat16)])
@pytest.mark.parametrize("normed", [True, False])
def test_rope(dev, layout, dtype, f32, normed):
    """Prompts that begin and continue, a single token, an empty slot, padding, a token without a position, pages that
    are none; rows that are not written keep their bits."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(2)
    qh, kh, d = layout
    new, old = [20, 1, 0, 35, 6, 3], [0, 47, 9, 14, 0, 0]
    lengths = [a + b for a, b in zip(new, old)]
    keys, vals, table, lens = cache(dev, g, lengths, kh=kh, d=d, page=16, dtype=dtype, poison=3.0, interleaved=normed)
    table[3, 2] = -1
    table[5, 0] = 2 ** 30
    lens[4] = 2  # its first four tokens stand before the sequence's first row
    starts = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device=dev)
    total = sum(new) + 4
    width = (qh + 2 * kh) * d
    qkv = (torch.randn((total, width + 64), generator=g) * 2).to(dtype).to(dev)[:, :width]
    qw, kw = ((torch.randn(d, generator=g) * 0.3 + 1).to(dtype).to(dev) if normed else None for _ in range(2))
    angle = torch.arange(40, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(d, dtype=torch.float64) % (d // 2) / (d // 2))
    cos, sin = (t.to(torch.float32 if f32 else dtype).to(dev) for t in (angle.cos(), angle.sin()))
    q = torch.full((total, qh, d), 5.0, dtype=dtype, device=dev)
    before = values(q)
    w = [None if t is None else values(t) for t in (qw, kw)]
    ref = o.qk_rope(values(qkv), *w, values(cos), values(sin), values(keys), values(vals), table.cpu().numpy(),
                    lens.cpu().numpy(), starts.cpu().numpy(), 1e-6, before)
    assert paged.qk_rope(qkv, qw, kw, cos, sin, keys, vals, table, lens, 1e-6, starts=starts, out=q).data_ptr() == q.data_ptr()
    # fp32 steps: the mean (D squares), the root, three products, two products and a sum, each off by 2^-24 of its terms,
    # which are at most 1.5 times the row's largest result; then one rounding
    half = torch.finfo(dtype).eps / 2
    for name, got, want in (("q", q, ref[0]), ("keys", keys, ref[1])):
        top = np.abs(want).max(-1, keepdims=True)
        _close(got, want, half * np.abs(want) + (d / 2 + 16) * 2.0 ** -24 * 1.5 * top, name)
    assert np.array_equal(values(vals), ref[2])
    assert np.array_equal(values(q)[sum(new):], before[sum(new):])


def test_rope_without_starts(dev):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(6)
    keys, vals, table, lens = cache(dev, g, [1, 40, 33, 0], kh=2, d=128, page=32, dtype=torch.bfloat16, poison=0.0)
    qkv = torch.randn((4, 8 * 128), generator=g).bfloat16().to(dev)
    cos, sin = (torch.randn((64, 128), generator=g).to(dev) for _ in range(2))
    k2, v2 = keys.clone(), vals.clone()
    q = paged.qk_rope(qkv, None, None, cos, sin, keys, vals, table, lens, 1e-6)
    starts = torch.arange(5, dtype=torch.int32, device=dev)
    q2 = paged.qk_rope(qkv, None, None, cos, sin, k2, v2, table, lens, 1e-6, starts=starts)
    assert torch.equal(q, q2) and torch.equal(keys, k2) and torch.equal(vals, v2)
    want = o.qk_rope(values(qkv), None, None, values(cos), values(sin), values(keys), values(vals), table.cpu().numpy(),
                     lens.cpu().numpy(), np.arange(5), 1e-6, np.zeros((4, 4, 128)))
    assert np.array_equal(values(vals), want[2])
    assert (np.abs(values(q) - want[0]) <= 2.0 ** -8 * np.abs(want[0]) + 2.0 ** -16).all()


def test_cache_past_32_bit_offsets(dev):
    """Pages whose first element lies past 2^32 elements: written by qk_rope, read by both attentions."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(8)
    kh, page, d = 2, 64, 128
    pages = 2 ** 32 // (kh * page * d) + 40
    keys, vals = (torch.empty((pages, kh, page, d), dtype=torch.bfloat16, device=dev) for _ in range(2))
    lengths, new = [150, 70], [150, 1]
    table = torch.tensor([[pages - 1, pages - 3, pages - 7], [0, pages - 2, -1]], dtype=torch.int32, device=dev)
    for p in (pages - 1, pages - 2, pages - 3, pages - 7, 0):
        keys[p], vals[p] = (torch.randn((kh, page, d), generator=g).bfloat16().to(dev) for _ in range(2))
    lens = torch.tensor(lengths, dtype=torch.int32, device=dev)
    starts = torch.tensor([0, 150, 151], dtype=torch.int32, device=dev)
    qkv = torch.randn((151, (4 + 2 * kh) * d), generator=g).bfloat16().to(dev)
    cos, sin = torch.ones((256, d), device=dev), torch.zeros((256, d), device=dev)
    q = paged.qk_rope(qkv, None, None, cos, sin, keys, vals, table, lens, 1e-6, starts=starts)
    assert torch.equal(q.flatten(1), qkv[:, :4 * d])
    used = table[table >= 0].long()
    small = torch.full((2, 3), -1, dtype=torch.int32)
    small[table.cpu() >= 0] = torch.arange(len(used), dtype=torch.int32)
    k, v = keys[used].contiguous(), vals[used].contiguous()
    out = paged.prompt_attention(q, keys, vals, table, lens, starts)
    assert torch.equal(out, paged.prompt_attention(q, k, v, small.to(dev), lens, starts))
    last = q[[149, 150]].contiguous()
    out = paged.decode_attention(last, keys, vals, table, lens)
    assert torch.equal(out, paged.decode_attention(last, k, v, small.to(dev), lens))
    ref = o.decode_attention(values(last), values(k), values(v), small.numpy(), lens.cpu().numpy())
    assert (np.abs(values(out) - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -10).all()


def test_graph_follows_growing_sequences(dev):
    """One captured step (rope, page write, attention) replayed as the sequences grow, against eager calls; eager work
    and synchronizations between the replays."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(9)
    kh, qh, d, page = 2, 8, 128, 16
    lengths = [5, 15, 100, 0]
    room = [n + 40 for n in lengths]
    keys, vals, table, _ = cache(dev, g, room, kh=kh, d=d, page=page, dtype=torch.bfloat16, poison=0.0)
    lens = torch.tensor(lengths, dtype=torch.int32, device=dev)
    qkv = torch.zeros((4, (qh + 2 * kh) * d), dtype=torch.bfloat16, device=dev)
    cos, sin = (torch.randn((256, d), generator=g).to(dev) for _ in range(2))

    def step(k, v):
        q = paged.qk_rope(qkv, None, None, cos, sin, k, v, table, lens, 1e-6)
        return paged.decode_attention(q, k, v, table, lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(keys, vals)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(keys, vals)
    k2, v2 = keys.clone(), vals.clone()
    for i in range(4):
        lens += 9 if i == 2 else 1
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step(k2, v2))
        torch.cuda.synchronize()
        assert torch.equal(keys, k2) and torch.equal(vals, v2)


def test_calls_on_two_streams(dev):
    """Calls that overlap on two streams, each with its own workspace, give what they give alone."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(10)
    sets = []
    for n in (700, 5000):
        keys, vals, table, lens = cache(dev, g, [n, n // 3], kh=2, d=128, page=16, dtype=torch.bfloat16)
        sets.append((torch.randn((2, 8, 128), generator=g).bfloat16().to(dev), keys, vals, table, lens))
    alone = [paged.decode_attention(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(paged.decode_attention(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in outs[i])


def test_prompt_graph_follows_its_batch(dev):
    """A captured prompt pass of 60 packed rows and its rope, replayed with other starts and lengths: more and fewer tokens,
    tiles that are cut and tiles that are not, padding; eager work and synchronizations between the replays."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(12)
    kh, qh, d, page, total = 2, 8, 128, 16, 60
    keys, vals, table, lens = cache(dev, g, [3000, 900, 500], kh=kh, d=d, page=page, dtype=torch.bfloat16, poison=0.0)
    starts = torch.tensor([0, 1, 20, 60], dtype=torch.int32, device=dev)
    qkv = torch.randn((total, (qh + 2 * kh) * d), generator=g).bfloat16().to(dev)
    cos, sin = (torch.randn((4096, d), generator=g).to(dev) for _ in range(2))
    out = torch.zeros((total, qh * d), dtype=torch.bfloat16, device=dev)

    def step(k, v, q, o):
        paged.qk_rope(qkv, None, None, cos, sin, k, v, table, lens, 1e-6, starts=starts, out=q)
        return paged.prompt_attention(q, k, v, table, lens, starts, out=o)

    q = torch.zeros((total, qh, d), dtype=torch.bfloat16, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(keys, vals, q, out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(keys, vals, q, out)
    k2, v2, q2, o2 = (t.clone() for t in (keys, vals, q, out))
    for at, n in (([0, 1, 20, 60], [3000, 900, 500]), ([0, 0, 40, 41], [0, 40, 17]), ([0, 1, 2, 3], [2999, 898, 499]),
                  ([0, 60, 60, 60], [60, 0, 3]), ([0, 0, 0, 0], [1, 2, 3]), ([0, 2, 3, 40], [2048, 64, 500])):
        starts.copy_(torch.tensor(at, dtype=torch.int32))
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(torch.bfloat16))
        for t in (q, out, q2, o2):
            t.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        step(k2, v2, q2, o2)
        torch.cuda.synchronize()
        for a, b in ((q, q2), (out, o2), (keys, k2), (vals, v2)):
            assert torch.equal(a, b)
        assert (out[at[-1]:] == 9.0).all() and (q[at[-1]:] == 9.0).all()


def test_prompt_calls_on_two_streams(dev):
    """Prompts whose tiles are cut, on two streams, with workspaces of their own."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(13)
    sets = []
    for old, new in (([3000, 10], [2, 30]), ([1500, 700], [20, 1])):
        keys, vals, table, lens = cache(dev, g, [a + b for a, b in zip(old, new)], kh=2, d=128, page=32, dtype=torch.bfloat16)
        starts = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device=dev)
        sets.append((torch.randn((sum(new), 8, 128), generator=g).bfloat16().to(dev), keys, vals, table, lens, starts))
    alone = [paged.prompt_attention(*s) for s in sets]
    kept = [paged.prompt_workspace(s[0], s[1], s[3]) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[], []]
    for n in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(paged.prompt_attention(*sets[i], ws=kept[i] if n % 2 else None))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in outs[i])


def test_pages_that_sequences_share(dev):
    """A prefix of whole pages that three sequences read, and one page twice in a sequence."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(14)
    keys, vals, _, _ = cache(dev, g, [160], kh=2, d=64, page=16, dtype=torch.bfloat16)
    rows = [int(p) for p in torch.where(torch.isfinite(keys[:, 0, 0, 0].float()))[0]]
    table = torch.tensor([rows[:4] + [rows[4], rows[4]], rows[:4] + [rows[5], -1], rows[:4] + [rows[6], rows[7]]],
                         dtype=torch.int32, device=dev)
    lens = torch.tensor([96, 70, 90], dtype=torch.int32, device=dev)
    q = torch.randn((3, 8, 64), generator=g).bfloat16().to(dev)
    k, v = values(keys), values(vals)
    ref = o.decode_attention(values(q), k, v, table.cpu().numpy(), lens.cpu().numpy())
    ref_abs = o.decode_attention(values(q), k, np.abs(v), table.cpu().numpy(), lens.cpu().numpy())
    live_k, live_v = np.nan_to_num(k), np.nan_to_num(v)
    got = paged.decode_attention(q, keys, vals, table, lens)
    _close(got, ref, attention_bound(values(q), live_k, live_v, ref, ref_abs, 0.125, q.dtype, False), "decode")
    starts = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev)
    got = paged.prompt_attention(q, keys, vals, table, lens, starts)
    _close(got, ref, attention_bound(values(q), live_k, live_v, ref, ref_abs, 0.125, q.dtype, True), "prompt")


def test_refusals(dev):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(0)
    keys, vals, table, lens = cache(dev, g, [20, 5], kh=2, d=64, page=16, dtype=torch.bfloat16)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=dev)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    paged.decode_attention(q, keys, vals, table, lens)

    def refused(match, fn, *a, **k):
        with pytest.raises(ValueError, match=match):
            fn(*a, **k)

    d = paged.decode_attention
    refused("q must be", d, q.float(), keys, vals, table, lens)
    refused("q must be a CUDA", d, q.cpu(), keys, vals, table, lens)
    refused("keys must be a", d, q, keys.half(), vals.half(), table, lens)
    refused("matching", d, q, keys, vals[:, :1], table, lens)
    refused("multiple of the KV heads", d, q[:, :3], keys, vals, table, lens)
    refused("multiple of the KV heads", d, q[:1], keys, vals, table, lens)
    refused("contiguous", d, q.transpose(1, 2).contiguous().transpose(1, 2), keys, vals, table, lens)
    refused("power of two", d, q, keys[:, :, :8].contiguous(), vals[:, :, :8].contiguous(), table, lens)
    refused("contiguous", d, q, keys.transpose(1, 2).contiguous().transpose(1, 2), vals, table, lens)
    refused("head dim must be", d, torch.zeros((2, 4, 32), dtype=torch.bfloat16, device=dev), keys[..., :32].contiguous(),
            vals[..., :32].contiguous(), table, lens)
    refused("overlap", d, q, keys[:1].expand(4, -1, -1, -1), vals[:1].expand(4, -1, -1, -1), table, lens)
    refused("table must be", d, q, keys, vals, table.long(), lens)
    refused("one length", d, q, keys, vals, table, lens[:1])
    refused("lengths must be", d, q, keys, vals, table, lens.long())
    refused("scale", d, q, keys, vals, table, lens, scale=float("nan"))
    refused("workspace too small", d, q, keys, vals, table, lens, ws=torch.zeros(4, device=dev))
    refused("out must not overlap", d, q, keys, vals, table, lens, out=q.view(2, 256))
    refused("out must hold", d, q, keys, vals, table, lens, out=q.new_empty((2, 128)))
    refused("out must not overlap", paged.prompt_attention, q, keys, vals, table, lens, starts, out=keys.view(-1)[:512].view(2, 256))
    refused("starts required", paged.prompt_attention, q, keys, vals, table, lens, None)
    refused("starts must hold", paged.prompt_attention, q, keys, vals, table, lens, starts[:2])
    qkv = torch.zeros((2, 8 * 64), dtype=torch.bfloat16, device=dev)
    cos = torch.zeros((32, 64), device=dev)
    r = paged.qk_rope
    r(qkv, None, None, cos, cos, keys, vals, table, lens, 1e-6)
    refused("both head-norm weights", r, qkv, cos[0].bfloat16(), None, cos, cos, keys, vals, table, lens, 1e-6)
    refused("query heads", r, qkv[:, :7 * 64].contiguous(), None, None, cos, cos, keys, vals, table, lens, 1e-6)
    refused("query heads", r, qkv[:, :4 * 64].contiguous(), None, None, cos, cos, keys, vals, table, lens, 1e-6)
    refused("one token a sequence", r, qkv[:1], None, None, cos, cos, keys, vals, table, lens, 1e-6)
    refused("cos must be", r, qkv, None, None, cos.double(), cos.double(), keys, vals, table, lens, 1e-6)
    refused("sin must be", r, qkv, None, None, cos, cos.bfloat16(), keys, vals, table, lens, 1e-6)
    refused("share memory", r, qkv, None, None, cos, cos, keys, keys, table, lens, 1e-6)
    refused("share memory", r, qkv, None, None, cos, cos, keys[:2], keys[1:3], table, lens, 1e-6)
    refused("eps", r, qkv, None, None, cos, cos, keys, vals, table, lens, -1.0)
    refused("16-byte", r, qkv.view(-1)[4:4 + 512].view(1, 512), None, None, cos, cos, keys, vals, table[:1], lens[:1], 1e-6)


@pytest.mark.parametrize("new, old", [([1], [2500]), ([3, 40], [1500, 0]), ([150], [1900]), ([1, 1, 1, 300], [4000, 30, 1200, 700])])
@pytest.mark.parametrize("layout", [(8, 2, 128), (16, 1, 128), (4, 4, 64)])
def test_prompt_cut_tiles(dev, new, old, layout):
    """A few new tokens behind a long prefix: tiles that are cut into parts and joined."""
    _prompt(dev, new, old, layout, torch.bfloat16, 16, pad=2)


def test_prompt_starts_that_do_not_rise(dev):
    """Starts that name the same tokens many times over, fall or lie outside: no write past the output or the workspace,
    whose end is watched."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(3)
    n = 40
    keys, vals, table, lens = cache(dev, g, [1500] * n, kh=2, d=128, page=64, dtype=torch.bfloat16)
    q = torch.randn((2, 8, 128), generator=g).bfloat16().to(dev)
    need = paged.prompt_workspace(q, keys, table).numel()
    ws = torch.full((need + 4096,), 3.0, device=dev)
    buffer = torch.full((4, 1024), 3.0, dtype=torch.bfloat16, device=dev)
    for starts in ([0, 1] * (n // 2) + [0], [2] * n + [-5], [-2 ** 31, 2 ** 31 - 1] * (n // 2) + [7], list(range(n, -1, -1))):
        paged.prompt_attention(q, keys, vals, table, lens, torch.tensor(starts, dtype=torch.int32, device=dev),
                               out=buffer[1:3], ws=ws[:need])
        torch.cuda.synchronize()
        assert (ws[need:] == 3.0).all() and (buffer[[0, 3]] == 3.0).all()


@pytest.mark.parametrize("new, old, layout", [([40, 70], [0, 30], (8, 2, 128)), ([130], [5], (4, 4, 64)), ([700], [100], (32, 8, 128))])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_prompt_values_behind_a_token(dev, new, old, layout, what):
    """NaN and infinities in K and V of tokens that come later reach no earlier token; the later ones see them."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(11)
    qh, kh, d = layout
    lengths = [a + b for a, b in zip(new, old)]
    keys, vals, table, lens = cache(dev, g, lengths, kh=kh, d=d, page=16, dtype=torch.bfloat16)
    starts = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device=dev)
    q = torch.randn((sum(new), qh, d), generator=g).bfloat16().to(dev)
    clean = paged.prompt_attention(q, keys, vals, table, lens, starts)
    spread = values(paged.prompt_attention(q, keys, vals.abs(), table, lens, starts))  # sum p |v|
    bad = [n - n // 3 for n in new]  # the new token of each sequence whose row is bad
    for b, t in enumerate(bad):
        row = old[b] + t
        vals[table[b, row // 16].long(), :, row % 16, ::3] = what
        if b:
            keys[table[b, row // 16].long(), :, row % 16, 5] = what
    got = paged.prompt_attention(q, keys, vals, table, lens, starts)
    torch.cuda.synchronize()
    for b, t in enumerate(bad):
        at = int(starts[b])
        x, y, a = values(got[at:at + t]), values(clean[at:at + t]), spread[at:at + t]
        # The rows of tiles without such a key are the same.  The others are summed without rounding P, by which each
        # weight differs by at most 2^-8 of itself and the output by twice that of sum p |v|; both are rounded once more,
        # by 2^-8, and scores summed in another order move a weight by less than 2^-12.
        assert np.isfinite(x).all()
        assert (np.abs(x - y) <= (2.0 ** -7 + 2.0 ** -11) * a * (1 + 2.0 ** -6) + 2.0 ** -8 * (np.abs(x) + np.abs(y))).all()
        after = got[at + t:at + new[b]].view(-1, qh, d)[..., ::3]
        assert not torch.isfinite(after).any()
