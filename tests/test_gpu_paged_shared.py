"""GPU: decode attention of sequences that share a prefix, against the definition in 64 bits of every sequence alone."""
import numpy as np
import pytest
import torch

from oracle import paged as o
from paged_helpers import attention_bound, cache, cache8, cache8_values, values

pytestmark = pytest.mark.gpu

LAYOUTS = [(32, 8, 128), (4, 4, 64), (28, 4, 128), (16, 2, 64), (16, 1, 128), (40, 2, 128), (3, 3, 128)]
DTYPES = [torch.bfloat16, torch.float16]


def _batch(dev, g, groups, shared, lengths, *, kh, d, page, dtype, bits, interleaved=False):
    """A cache whose runs name the same pages for the rows that they share, and hold equal rows where a page is not shared
    whole."""
    if bits == 16:
        keys, vals, table, lens = cache(dev, g, lengths, kh=kh, d=d, page=page, dtype=dtype, interleaved=interleaved)
        parts, scales = [keys, vals], None
    else:
        keys, vals, scales, table, lens = cache8(dev, g, lengths, kh=kh, d=d, page=page, interleaved=interleaved)
        parts = [keys.view(torch.uint8), vals.view(torch.uint8), *scales]
    at = table.cpu().clone()
    first = 0
    for b in range(1, len(groups)):
        if groups[b] < 0 or groups[b] != groups[b - 1]:
            first = b
            continue
        n = max(0, min(shared[b], shared[first], lengths[first], lengths[b]))
        whole = n // page
        for r in range(whole * page, n):
            for t in parts:
                t[at[b, r // page], :, r % page] = t[at[first, r // page], :, r % page]
        at[b, :whole] = at[first, :whole]
    return keys, vals, scales, at.to(dev), lens


BALLAST = 4096


def _with_ballast(groups, shared, lengths, kh):
    """Sharing is taken up when it saves enough rows: a run behind the batch that saves enough by itself."""
    n = 1 + -(-131072 // (kh * BALLAST))
    return groups + [10 ** 6] * n, shared + [BALLAST] * n, lengths + [BALLAST + 3] + [2 + i for i in range(1, n)], n


def _check(dev, groups, shared, lengths, layout, dtype, page, *, bits=16, seed=0, scale=None, edit=None, stride=0, interleaved=False,
           ballast=True):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(seed)
    qh, kh, d = layout
    print(f"shared groups={groups} shared={shared} lengths={lengths} layout={layout} {dtype} page={page} bits={bits} ballast={ballast}", flush=True)
    mine = len(groups)
    if ballast:  # its own rows are made as short sequences, whose tables then begin with the first one's pages
        groups, shared, lengths, n = _with_ballast(groups, shared, lengths, kh)
    keys, vals, scales, table, lens = _batch(dev, g, groups[:mine], shared[:mine], lengths, kh=kh, d=d, page=page, dtype=dtype, bits=bits,
                                             interleaved=interleaved)
    if ballast:
        whole = BALLAST // page
        wide_table = torch.full((len(groups), table.shape[1] + 1), -1, dtype=torch.int32, device=dev)
        wide_table[:, :-1] = table
        for b in range(mine + 1, len(groups)):
            wide_table[b, whole] = table[b, 0]
            wide_table[b, :whole] = table[mine, :whole]
            lens[b] += BALLAST
        table = wide_table
    ids, most = (torch.tensor(t, dtype=torch.int32) for t in (groups, shared))
    if edit is not None:
        parts = [t.cpu() for t in (table, lens, ids, most)]
        edit(*(t[:mine] for t in parts))
        table, lens, ids, most = parts
    table, lens, ids, most = (t.to(dev) for t in (table, lens, ids, most))
    wide = (torch.randn((len(lengths), qh * d + stride), generator=g) * 1.5).to(dtype).to(dev)
    q = wide[:, :qh * d].unflatten(1, (qh, d))
    ws = paged.shared_decode_workspace(q, keys, table).fill_(float("nan"))
    out = paged.shared_decode_attention(q, keys, vals, table, lens, ids, most, scale=scale, ws=ws, scales=scales)
    torch.cuda.synchronize()
    if bits == 16:
        args = values(q), values(keys), values(vals)
    else:
        args = values(q), cache8_values(keys, scales[0]), cache8_values(vals, scales[1])
    t, n = table.cpu().numpy(), lens.cpu().numpy()
    ref = o.decode_attention(*args, t, n, scale)
    ref_abs = o.decode_attention(args[0], args[1], np.abs(args[2]), t, n, scale)
    bound = attention_bound(args[0], *(np.where(np.abs(a) < 1e6, a, 0.0) for a in args[1:]), ref, ref_abs,
                            d ** -0.5 if scale is None else scale, dtype, True)
    err = np.abs(values(out) - ref)
    assert np.isfinite(values(out)).all()
    assert (err <= bound).all(), f"{int((err > bound).sum())} off, worst {float((err / bound).max()):.3g} of the bound, rows {sorted(set(np.argwhere(err > bound)[:, 0].tolist()))}"
    return out


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_layouts(dev, layout, dtype, bits):
    _check(dev, [0, 0, 0, -1, 5, 5, 2], [96, 96, 96, 70, 32, 32, 16], [120, 97, 300, 70, 33, 200, 20], layout, dtype, 16, bits=bits)


@pytest.mark.parametrize("ballast", [True, False])
@pytest.mark.parametrize("page", [16, 64, 512])
@pytest.mark.parametrize("groups, shared, lengths", [
    ([0, 0], [16, 16], [17, 17]),                                   # the least prefix
    ([0, 0], [15, 15], [20, 20]),                                   # less than 16 rows: none
    ([0, 0, 0], [100, 100, 100], [101, 130, 100]),                  # not whole 16 rows; a sequence that ends with it
    ([0, 0, 0], [200, 200, 200], [200, 200, 200]),                  # nothing of its own
    ([0, 0, 0], [208, 208, 208], [208, 208, 208]),
    ([1, 1, 1, 1], [640, 64, 320, 0], [700, 650, 320, 9]),          # shares of different lengths
    ([1, 1, 1], [640, 640, 640], [1000, 30, 0]),                    # shorter than the prefix, empty
    ([1, 1, 1], [640, 640, 640], [20, 700, 650]),                   # the first one is short: few rows shared
    ([1, 1, 1], [640, 640, 640], [0, 700, 650]),                    # the first one is empty: none
    ([3, 3, -1, -1, 3, 3], [64, 64, 64, 64, 128, 128], [70, 80, 90, 100, 140, 150]),  # one number twice: two runs
    ([-1, -1, -1], [64, 64, 64], [70, 80, 90]),
    ([0], [64], [300]),
    ([7] * 9, [1500] * 9, [1501, 1600, 2000, 1700, 1500, 1900, 1555, 1800, 1501]),
])
def test_runs(dev, groups, shared, lengths, page, ballast):
    _check(dev, groups, shared, lengths, (8, 2, 128), torch.bfloat16, page, ballast=ballast)


@pytest.mark.parametrize("bits", [16, 8])
def test_many_sequences(dev, bits):
    """Runs that end at, begin at and pass the batch's 64th sequences; tiles of both heights."""
    rng = np.random.default_rng(2)
    groups = [0] * 40 + [1] * 24 + [2] * 3 + [-1] * 2 + [3] * 80 + [4]
    shared = [160] * 40 + [48] * 24 + [32] * 3 + [0] * 2 + [96] * 80 + [0]
    lengths = [s + int(rng.integers(1, 50)) for s in shared]
    _check(dev, groups, shared, lengths, (4, 2, 64), torch.bfloat16, 16, bits=bits)
    _check(dev, groups, shared, lengths, (32, 8, 128), torch.bfloat16, 16, bits=bits)


def test_strides_and_scale(dev):
    for kwargs in (dict(stride=8, interleaved=True), dict(scale=0.0), dict(scale=1.0), dict(scale=-0.3), dict(interleaved=True, bits=8)):
        _check(dev, [0, 0, 0], [64, 64, 64], [70, 100, 300], (8, 4, 128), torch.bfloat16, 32, **kwargs)


def test_pages_that_are_none(dev):
    """Inside the prefix, for all of a run; behind it; nothing left of a sequence."""
    def edit(table, lens, ids, most):
        table[:3, 1] = -5
        table[1, 5] = 2 ** 31 - 1
        table[3:, :] = -(2 ** 31)

    _check(dev, [0, 0, 0, 1, 1], [64, 64, 64, 32, 32], [70, 130, 90, 40, 50], (8, 2, 128), torch.bfloat16, 16, edit=edit)


def test_device_values_past_everything(dev):
    """Lengths and shared rows that no table holds, negative ones."""
    def edit(table, lens, ids, most):
        most[:] = torch.tensor([2 ** 31 - 1, 2 ** 31 - 1, -5, -(2 ** 31)], dtype=torch.int32)
        lens[1] = 2 ** 31 - 1
        lens[2] = -1
        ids[:] = 2 ** 31 - 1
        table[1] = table[0]

    _check(dev, [0, 0, 0, 0], [0, 0, 0, 0], [64, 64, 20, 30], (8, 2, 128), torch.bfloat16, 16, edit=edit)


def test_without_runs(dev):
    """Sequences that share nothing have no rounded weights: the decode attention's own bound holds."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(1)
    keys, vals, table, lens = cache(dev, g, [900, 20, 3000, 0], kh=2, d=128, page=64, dtype=torch.bfloat16)
    q = torch.randn((4, 8, 128), generator=g).bfloat16().to(dev)
    args, rest = (values(q), values(keys), values(vals)), (table.cpu().numpy(), lens.cpu().numpy())
    ref, ref_abs = o.decode_attention(*args, *rest), o.decode_attention(args[0], args[1], np.abs(args[2]), *rest)
    bound = attention_bound(*args, ref, ref_abs, 128 ** -0.5, torch.bfloat16, False)
    none = torch.full((4,), -1, dtype=torch.int32, device=dev)
    for ids, most in ((none, lens), (torch.arange(4, dtype=torch.int32, device=dev), lens), (torch.zeros_like(none), torch.zeros_like(none))):
        out = paged.shared_decode_attention(q, keys, vals, table, lens, ids, most)
        assert (np.abs(values(out) - ref) <= bound).all()


def _long_run(dev, g, kh, d, page=16):
    """Nine sequences over 2048 shared rows: enough to be shared with 8 KV heads."""
    groups, shared, lengths = [0] * 9, [2048] * 9, [2049 + 40 * i for i in range(9)]
    keys, vals, _, table, lens = _batch(dev, g, groups, shared, lengths, kh=kh, d=d, page=page, dtype=torch.bfloat16, bits=16)
    ids, most = (torch.tensor(t, dtype=torch.int32, device=dev) for t in (groups, shared))
    return keys, vals, table, lens, ids, most


def test_captured(dev):
    """A graph that follows lengths, groups and shared rows; beside an eager call on another stream; bit for bit."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(3)
    keys, vals, table, lens, ids, most = _long_run(dev, g, 8, 128)
    q = torch.randn((9, 32, 128), generator=g).bfloat16().to(dev)
    args = q, keys, vals, table, lens, ids, most
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.shared_decode_attention(*args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.shared_decode_attention(*args)
    for i, (a, b) in enumerate([([0] * 9, [2048] * 9), ([-1] * 9, [0] * 9), ([0, 0] + [1] * 7, [2048] * 2 + [1900] * 7),
                                ([2] * 9, [2048, 300, 320, 0, 100, 2048, 2048, 2000, 9])] * 2):
        ids.copy_(torch.tensor(a, dtype=torch.int32))
        most.copy_(torch.tensor(b, dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=g).bfloat16())
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = paged.shared_decode_attention(*args)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i
        # either rounds its output (2^-8), the prefix's weights besides
        plain = paged.decode_attention(*args[:5]).double()
        assert float((out.double() - plain).norm() / plain.norm()) < 2.0 ** -8 * 1.5


def test_values_that_are_not_finite(dev):
    """A row of NaN in the shared rows reaches the sequences that take it and no other; rows behind a short sequence's end
    hold anything."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(4)
    keys, vals, table, lens, ids, most = _long_run(dev, g, 8, 64)
    lens[1] = 60      # ends within the shared rows, before the row
    most[2] = 96      # takes them from its own table from here on, which names the same page
    ids[8] = -1
    table[2, 6:] = table[2, 128:134].repeat(1 + table.shape[1] // 6)[:table.shape[1] - 6]
    table[8, 6] = table[8, 128]
    vals[int(table[0, 100 // 16]), :, 100 % 16] = float("nan")
    q = torch.randn((9, 32, 64), generator=g).bfloat16().to(dev)
    lens[2] = 150
    out = paged.shared_decode_attention(q, keys, vals, table, lens, ids, most)
    want = paged.decode_attention(q, keys, vals, table, lens)
    for b in (0, 3, 4, 5, 6, 7):
        assert torch.isnan(out[b]).all() and torch.isnan(want[b]).all()
    for b in (1, 2, 8):
        assert float((out[b].double() - want[b].double()).norm() / want[b].double().norm()) < 2.0 ** -8 * 1.5


def test_refusals(dev):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(0)
    keys, vals, table, lens = cache(dev, g, [20, 30], kh=2, d=64, page=16, dtype=torch.bfloat16)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=dev)
    ids = torch.zeros(2, dtype=torch.int32, device=dev)
    args = q, keys, vals, table, lens
    paged.shared_decode_attention(*args, ids, ids.clone())
    for bad in (ids.long(), ids[:1], ids.cpu(), None, 3, torch.zeros(4, dtype=torch.int32, device=dev)[::2]):
        with pytest.raises(ValueError):
            paged.shared_decode_attention(*args, bad, ids)
        with pytest.raises(ValueError):
            paged.shared_decode_attention(*args, ids, bad)
    out = torch.zeros((2, 256), dtype=torch.bfloat16, device=dev)
    need = paged.shared_decode_workspace(q, keys, table)
    for bad in (dict(out=out[:1]), dict(out=out.half()), dict(ws=need[:-1]), dict(ws=need.cpu()), dict(scale=float("inf")),
                dict(out=q.view(2, 256)), dict(out=vals.flatten()[:512].view(2, 256))):
        with pytest.raises(ValueError):
            paged.shared_decode_attention(*args, ids, ids.clone(), **bad)
    whole = torch.zeros(need.numel() + 64, device=dev)
    with pytest.raises(ValueError, match="overlap"):
        paged.shared_decode_attention(*args, whole[:2].view(torch.int32), ids, ws=whole[:need.numel()])
    with pytest.raises(ValueError, match="overlap"):
        paged.shared_decode_attention(*args, ids, whole[4:6].view(torch.int32), ws=whole[:need.numel()])
