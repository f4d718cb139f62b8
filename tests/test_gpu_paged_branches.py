"""GPU: the code that paged calls take only from some size on: prompts in tiles of 128 rows, sequences of more than 64
decode shares, batches of more than 64 sequences whose work is cut, caches that are read past the last-level cache."""
import numpy as np
import pytest
import torch

import test_gpu_paged as small
from paged_helpers import attend_all, attention_bound, cache, values

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _tall(tokens, layout):
    """A call of so many tokens is taken in tiles of 128 rows: the workspace of a wide table shows it."""
    from moss_tts._runtime import native

    qh, kh, d = layout
    nbytes = native.lib().moss_paged_prompt_workspace_bytes(1, 1000, 16, tokens, qh, kh, d)
    assert nbytes == 2 * max(256 // kh, 1) * kh * 128 * (d + 2) * 4, "not in tiles of 128 rows"


def _prompt(dev, new, old, layout, dtype, page, *, pad=0, edit=None, interleaved=False, stride=0):
    """A prompt call in tiles of 128 rows against the 64-bit reference."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(21)
    qh, kh, d = layout
    lengths = [a + b for a, b in zip(new, old)]
    keys, vals, table, lens = cache(dev, g, lengths, kh=kh, d=d, page=page, dtype=dtype, interleaved=interleaved)
    if edit is not None:
        table, lens = edit(table.cpu(), lens.cpu())
        table, lens = table.to(dev), lens.to(dev)
    at = [0, *np.cumsum(new).tolist()]
    starts = torch.tensor(at, dtype=torch.int32, device=dev)
    total = sum(new) + pad
    wide = (torch.randn((total, qh * d + stride), generator=g) * 1.5).to(dtype).to(dev)
    q = wide[:, :qh * d].unflatten(1, (qh, d))
    _tall(total, layout)
    ws = paged.prompt_workspace(q, keys, table)
    if ws is not None:
        ws.fill_(float("nan"))
    out = torch.full((total, qh * d), 7.0, dtype=dtype, device=dev)
    before = out.clone()
    print(f"prompt new={new} old={old} layout={layout} {dtype} page={page}", flush=True)
    paged.prompt_attention(q, keys, vals, table, lens, starts, out=out, ws=ws)
    torch.cuda.synchronize()
    rest = table, lens, at, before, d ** -0.5
    ref = values(attend_all(q, keys, vals, *rest))
    ref_abs = values(attend_all(q, keys, vals.abs(), *rest))
    largest = [np.array([t.nan_to_num(nan=0.0).abs().max().item()]) for t in (keys, vals)]
    small._close(out, ref, attention_bound(values(q), *largest, ref, ref_abs, d ** -0.5, dtype, True), "prompt")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout, new, old, page", [
    ((512, 128, 64), [171, 70, 1, 58], [0, 150, 9, 700], 16),   # ends inside tiles and blocks, continued prompts
    ((448, 64, 128), [300, 0, 13], [0, 4, 45], 32),             # groups that do not divide a tile
    ((128, 128, 64), [1025, 30], [3, 0], 64),                   # heads that share nothing
    ((1024, 64, 64), [130, 5], [0, 3000], 64),                  # a prefix that is cut into parts
    ((256, 64, 128), [520, 7, 1], [0, 4000, 70], 128),
    ((32, 8, 128), [4200], [0], 64),
])
def test_prompt_tall_tiles(dev, layout, new, old, page, dtype):
    _prompt(dev, new, old, layout, dtype, page, pad=3)


def test_prompt_tall_tiles_strides(dev):
    _prompt(dev, [171, 70, 1, 58], [0, 150, 9, 700], (512, 128, 64), torch.bfloat16, 16, interleaved=True, stride=512)


@pytest.mark.parametrize("layout, dtype", [((512, 128, 64), torch.float16), ((1024, 128, 128), torch.bfloat16)])
def test_prompt_tall_tiles_rows_without_keys(dev, layout, dtype):
    """Pages that are none inside a prefix and under the new tokens, and more new tokens than the length says."""
    def edit(table, lens):
        table[0, 1] = -1
        table[0, 7] = 2 ** 31 - 1
        table[1, :] = 10 ** 9
        table[2, 0] = -3
        lens[3] = 12
        lens[4] = -4
        return table, lens

    _prompt(dev, [200, 60, 70, 30, 5], [60, 20, 0, 0, 0], layout, dtype, 16, edit=edit)


@pytest.mark.parametrize("layout, new, old", [((512, 128, 64), [150, 170], [0, 30]), ((256, 64, 128), [560], [100])])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_prompt_tall_tiles_values_behind_a_token(dev, layout, new, old, what):
    _tall(sum(new), layout)
    small.test_prompt_values_behind_a_token(dev, new, old, layout, what)


def test_prompt_many_sequences_cut(dev):
    """More sequences than a wave counts at once, a few new tokens of some behind long prefixes on both sides of the 64th."""
    rng = np.random.default_rng(7)
    new = [int(n) for n in rng.integers(0, 4, 130)]
    old = [int(n) for n in rng.integers(0, 40, 130)]
    for b, n in ((0, 1500), (5, 4000), (63, 1000), (64, 2500), (100, 3000), (129, 1100)):
        new[b], old[b] = 1 + b % 3, n
    small._prompt(dev, new, old, (8, 2, 64), torch.bfloat16, 16, pad=2)


def test_prompt_tall_tiles_many_sequences_cut(dev):
    rng = np.random.default_rng(8)
    new = [int(n) for n in rng.integers(1, 4, 130)]
    old = [int(n) for n in rng.integers(0, 40, 130)]
    new[90], old[90] = 2, 9000
    _prompt(dev, new, old, (1024, 64, 64), torch.bfloat16, 16, pad=1)


@pytest.mark.parametrize("layout, dtype, lengths", [
    ((8, 2, 128), torch.bfloat16, [20000, 5, 0, 8321, 300]),   # 157 and 66 shares of one unit
    ((12, 12, 64), torch.float16, [10000, 8200]),
    ((4, 2, 64), torch.bfloat16, [110000, 40]),                # 860 units: shares of two
])
def test_decode_many_shares(dev, layout, dtype, lengths):
    small._decode(dev, lengths, layout, dtype, 64, ws=True)


@pytest.mark.parametrize("layout, dtype", [((4, 2, 64), torch.bfloat16), ((32, 8, 128), torch.float16)])
def test_decode_many_sequences_of_many_shares(dev, layout, dtype):
    rng = np.random.default_rng(5)
    lengths = [int(n) for n in rng.integers(0, 200, 130)]
    for b, n in ((0, 0), (5, 4000), (63, 1000), (64, 2500), (65, 0), (100, 3000), (129, 1100)):
        lengths[b] = n
    small._decode(dev, lengths, layout, dtype, 16, ws=True)


@pytest.mark.parametrize("layout, dtype", [((32, 8, 128), torch.bfloat16), ((16, 8, 64), torch.float16)])
def test_decode_reads_past_the_cache(dev, layout, dtype):
    """Pages of more than 256 MB that the table has room for: the same bits as from a small cache."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(22)
    qh, kh, d = layout
    lengths, page = [3000, 77, 0, 1000], 64
    keys, vals, table, lens = cache(dev, g, lengths, kh=kh, d=d, page=page, dtype=dtype, width=50)
    q = torch.randn((4, qh, d), generator=g).to(dtype).to(dev)
    want = paged.decode_attention(q, keys, vals, table, lens)
    pages = (300 << 20) // (4 * kh * page * d)
    wide = torch.full((4, pages // 4 + 1), -1, dtype=torch.int32, device=dev)
    wide[:, :50] = torch.where(table >= 0, table * 9 + 5, table)
    k2, v2 = (torch.full((pages, kh, page, d), float("nan"), dtype=dtype, device=dev) for _ in range(2))
    k2[5:5 + 9 * len(keys):9], v2[5:5 + 9 * len(vals):9] = keys, vals
    got = paged.decode_attention(q, k2, v2, wide, lens)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.isfinite(got).all()
