"""GPU: what serving from a large pool of pages runs and small caches do not: loads past the last-level cache, from 8 bits and over
shared prefixes; and the 8-bit write with tables in the 16-bit type, code for code over head sizes, norms and heads."""
import numpy as np
import pytest
import torch

from oracle import paged as o
from paged_helpers import cache8, values
from shared_helpers import prefix_taken, shared_workspace
from test_gpu_paged8 import KIND, _tables
from test_gpu_paged_shared import _batch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _moved(dev, parts, table):
    """The same pages in a pool of more than 256 MB, whose other pages hold NaN and bytes that are no scale, and a table that has
    room for all of them."""
    kh, page, d = parts[0].shape[1:]
    eight = len(parts) == 4
    pages = (300 << 20) // ((2 if eight else 4) * kh * page * d)
    b = table.shape[0]
    wide = torch.full((b, max(pages // b + 1, table.shape[1])), -1, dtype=torch.int32, device=dev)
    step = (pages - 5) // len(parts[0])
    assert step >= 1 and b * wide.shape[1] >= pages
    wide[:, :table.shape[1]] = torch.where(table >= 0, table * step + 5, table)
    out = []
    for t in parts:
        raw = t.view(torch.uint8) if eight else t
        pool = torch.full((pages, *raw.shape[1:]), (0x7f if raw.dim() == 4 else 255) if eight else float("nan"), dtype=raw.dtype, device=dev)
        pool[5:5 + step * len(raw):step] = raw
        out.append(pool.view(t.dtype))
    return out, wide


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", [(32, 8, 128), (16, 8, 64)])
def test_decode_from_8_bits_past_the_cache(dev, layout, dtype):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(22)
    qh, kh, d = layout
    keys, vals, scales, table, lens = cache8(dev, g, [3000, 77, 0, 1000], kh=kh, d=d, page=64, width=50)
    q = torch.randn((4, qh, d), generator=g).to(dtype).to(dev)
    print(f"decode8 past the cache {layout} {dtype}", flush=True)
    want = paged.decode_attention(q, keys, vals, table, lens, scales=scales)
    (k2, v2, *s2), wide = _moved(dev, [keys, vals, *scales], table)
    got = paged.decode_attention(q, k2, v2, wide, lens, scales=tuple(s2))
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.isfinite(got).all() and got[0].any()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout, count, prefix", [((32, 8, 128), 9, 2048), ((16, 8, 64), 9, 2048),      # tiles of 64 rows
                                                   ((32, 8, 128), 131, 160), ((16, 8, 64), 260, 96)])    # of 128
def test_shared_past_the_cache(dev, layout, count, prefix, dtype, bits):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(23)
    qh, kh, d = layout
    groups, shared = [0] * count, [prefix] * count
    lengths = [prefix + 1 + 7 * i % 90 for i in range(count)]
    keys, vals, scales, table, lens = _batch(dev, g, groups, shared, lengths, kh=kh, d=d, page=16, dtype=dtype, bits=bits)
    q = torch.randn((count, qh, d), generator=g).to(dtype).to(dev)
    ids, most = (torch.tensor(t, dtype=torch.int32, device=dev) for t in (groups, shared))
    print(f"shared past the cache {layout} count={count} {dtype} bits={bits}", flush=True)
    want = paged.shared_decode_attention(q, keys, vals, table, lens, ids, most, scales=scales)
    (k2, v2, *s2), wide = _moved(dev, [keys, vals, *(scales or ())], table)
    s2 = tuple(s2) or None
    ws = shared_workspace(q, k2, wide)
    got = paged.shared_decode_attention(q, k2, v2, wide, lens, ids, most, scales=s2, ws=ws)
    alone = paged.decode_attention(q, keys, vals, table, lens, scales=scales)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and prefix_taken(ws, q, keys)
    # either rounds its output
    half = torch.finfo(dtype).eps / 2
    assert float((got.double() - alone.double()).norm() / alone.double().norm()) < 3 * half


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d, kh, qh", [(64, 1, 1), (64, 3, 6), (128, 3, 3), (64, 8, 16), (128, 8, 32)])
@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("table", ["fp32", "own"])
def test_written_codes(dev, d, kh, qh, dtype, normed, table):
    """Every key's and value's code and byte is the definition's: the kernel's 64-bit steps are off by 2^-44 of |x cos| + |y sin|,
    and a border lies within that of one value in 10^10."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(31)
    n, page = 16 * max(1, 64 // kh), 16
    qkv = (torch.randn((n, (qh + 2 * kh) * d), generator=g) * torch.exp2(torch.randint(-6, 7, (n, 1), generator=g).float())).to(dtype).to(dev)
    qw, kw = ((torch.randn(d, generator=g) * 0.3 + 1).to(dtype).to(dev) for _ in range(2)) if normed else (None, None)
    cos, sin = _tables(g, n, d, dev)
    if table == "own":
        cos, sin = cos.to(dtype), sin.to(dtype)
    keys, vals = (torch.zeros((n // page, kh, page, d), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2))
    scales = tuple(torch.zeros((n // page, kh, page), dtype=torch.uint8, device=dev) for _ in range(2))
    pages = torch.arange(n // page, dtype=torch.int32, device=dev)[None]
    eps = float(np.float32(1e-6))
    print(f"write8 d={d} kh={kh} qh={qh} {dtype} normed={normed} table={table}", flush=True)
    q = paged.qk_rope(qkv, qw, kw, cos, sin, keys, vals, pages, torch.tensor([n], dtype=torch.int32, device=dev), eps,
                      starts=torch.tensor([0, n], dtype=torch.int32, device=dev), scales=scales)
    torch.cuda.synchronize()
    x = values(qkv).reshape(n, -1, d)
    c, s = values(cos)[:, None], values(sin)[:, None]

    def turned(v, weight):
        if weight is not None:
            v = v / np.sqrt((v * v).mean(-1, keepdims=True) + eps) * values(weight)
        return v * c + np.concatenate((-v[..., d // 2:], v[..., :d // 2]), -1) * s

    for t, scale, rows in ((keys, scales[0], turned(x[:, qh:qh + kh], kw)), (vals, scales[1], x[:, qh + kh:])):
        codes = t.view(torch.uint8).cpu().numpy().transpose(0, 2, 1, 3).reshape(n, kh, d)
        byte = scale.cpu().numpy().transpose(0, 2, 1).reshape(n, kh)
        got = o.cache_values(codes, byte)
        for i in range(n):
            for h in range(kh):
                want, want_byte = o.quantize_row(rows[i, h], KIND[dtype])
                assert byte[i, h] == want_byte and np.array_equal(got[i, h], want), (i, h)
    ref = turned(x[:, :qh], qw)
    # fp32 from the inputs to one rounding: a sum of d / 2 products a lane and some steps
    half = torch.finfo(dtype).eps / 2
    top = np.abs(ref).max(-1, keepdims=True)
    floor = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert (np.abs(values(q) - ref) <= half * np.abs(ref) + (d / 2 + 16) * 2.0 ** -24 * 1.5 * top + floor).all()
