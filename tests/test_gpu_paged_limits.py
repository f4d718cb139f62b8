"""GPU: paged calls at the ends of what their arguments can say."""
import numpy as np
import pytest
import torch

from oracle import paged as o
from paged_helpers import cache, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [True, False])
def test_rope_lengths_past_the_table(dev, packed):
    """A length that the table's row cannot hold counts as the rows that it can, in qk_rope as in the attentions: the new
    tokens are the last of those rows, and attend themselves."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(31)
    qh, kh, d, page = 8, 2, 64, 16
    keys, vals, table, lens = cache(dev, g, [32, 32, 32, 32, 20], kh=kh, d=d, page=page, dtype=torch.bfloat16, width=2)
    lens.copy_(torch.tensor([40, 33, 2 ** 31 - 1, -5, 20], dtype=torch.int32))
    new = [8, 1, 3, 2, 4] if packed else [1] * 5
    at = np.concatenate(([0], np.cumsum(new)))
    starts = torch.from_numpy(at.astype(np.int32)).to(dev)
    qkv = torch.randn((sum(new), (qh + 2 * kh) * d), generator=g).bfloat16().to(dev)
    cos, sin = (torch.randn((64, d), generator=g).to(dev) for _ in range(2))
    rest = table.cpu().numpy(), lens.cpu().numpy(), at
    want = o.qk_rope(values(qkv), None, None, values(cos), values(sin), values(keys), values(vals), *rest, 1e-6,
                     np.zeros((sum(new), qh, d)))
    q = paged.qk_rope(qkv, None, None, cos, sin, keys, vals, table, lens, 1e-6, starts=starts if packed else None)
    torch.cuda.synchronize()
    # two products and a sum in fp32, each off by 2^-24 of terms of at most 20; one rounding
    for got, ref in ((values(q), want[0]), (values(keys), want[1])):
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        assert (np.abs(got - ref)[~np.isnan(ref)] <= (2.0 ** -8 * np.abs(ref) + 2.0 ** -18)[~np.isnan(ref)]).all()
    assert np.array_equal(values(vals), want[2], equal_nan=True)
    if packed:
        out = paged.prompt_attention(q, keys, vals, table, lens, starts)
        ref = o.prompt_attention(values(q), values(keys), values(vals), *rest, np.zeros((sum(new), qh * d)))
    else:
        out = paged.decode_attention(q, keys, vals, table, lens)
        ref = o.decode_attention(values(q), values(keys), values(vals), *rest[:2])
    # the terms of a score sum to at most 2^9 here, so fp32 moves a weight by less than (64 + 8) 2^-24 2^9 < 2^-8, and its
    # rounding by 2^-8; an error r in every weight moves the output by at most 2 r times a value, which is at most 5
    assert (np.abs(values(out) - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -6 * 5).all()


def test_rope_refuses_more_tokens_than_a_grid_holds(dev):
    """A launch of 256 threads a token ends at 2^32 threads."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(32)
    keys, vals, table, lens = cache(dev, g, [20], kh=1, d=64, page=16, dtype=torch.bfloat16)
    qkv = torch.empty((1 << 24, 3 * 64), dtype=torch.bfloat16, device=dev)
    cos = torch.zeros((32, 64), device=dev)
    starts = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="2\\^24"):
        paged.qk_rope(qkv, None, None, cos, cos, keys, vals, table, lens, 1e-6, starts=starts)


def test_outputs_over_what_the_kernels_read(dev):
    """An output or a workspace over the table, the lengths, the starts, the head-norm weights or the cos / sin tables is
    refused: the kernels would find their work changed while they run."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(33)
    qh, kh, d, n = 4, 2, 64, 2
    keys, vals, table, lens = cache(dev, g, [20, 700], kh=kh, d=d, page=16, dtype=torch.bfloat16)
    q = torch.zeros((n, qh, d), dtype=torch.bfloat16, device=dev)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    memory = torch.zeros(1 << 20, device=dev)
    width = table.shape[1]

    def over(t, at):  # a copy of t that lies in `memory` from element `at` on
        part = memory[at:at + t.numel() * t.element_size() // 4].view(t.dtype).view(t.shape)
        return part.copy_(t)

    out = memory[:n * qh * d // 2].view(torch.bfloat16).view(n, qh * d)
    last = out.numel() // 2 - 1  # the last word of the output
    need = paged.decode_workspace(q, keys, table).numel()
    assert torch.isfinite(paged.decode_attention(q, keys, vals, table, lens, out=out, ws=memory[1024:1024 + need])).all()
    for at in (0, last):
        for args in ((over(table, at), lens), (table, over(lens, at))):
            for more in ((), (starts,)):
                fn = paged.prompt_attention if more else paged.decode_attention
                with pytest.raises(ValueError, match="out must not overlap"):
                    fn(q, keys, vals, *args, *more, out=out)
                size = (paged.prompt_workspace if more else paged.decode_workspace)(q, keys, table).numel()
                with pytest.raises(ValueError, match="ws must not overlap"):
                    fn(q, keys, vals, *args, *more, ws=memory[:max(size, 1024)])
        with pytest.raises(ValueError, match="out must not overlap"):
            paged.prompt_attention(q, keys, vals, table, lens, over(starts, at), out=out)
    # a table whose rows lie apart: its last row counts
    wide = memory[4096 - width - 3:4096 + width - 3].view(torch.int32).as_strided((2, width), (width, 1), 4096 - width - 3)
    wide.copy_(table)
    with pytest.raises(ValueError, match="out must not overlap"):
        paged.decode_attention(q, keys, vals, wide, lens, out=memory[4096:4096 + n * qh * d // 2].view(torch.bfloat16).view(n, -1))

    qkv = torch.zeros((n, (qh + 2 * kh) * d), dtype=torch.bfloat16, device=dev)
    weight = torch.ones(d, dtype=torch.bfloat16, device=dev)
    cos = torch.zeros((1024, d), device=dev)
    plain = dict(q_weight=weight, k_weight=weight, cos=cos, sin=cos, table=table, lengths=lens, starts=starts)
    rope_out = out.view(n, qh, d)
    paged.qk_rope(qkv, keys=keys, values=vals, eps=1e-6, out=rope_out, **plain)
    torch.cuda.synchronize()
    for name, t in plain.items():
        with pytest.raises(ValueError, match="out must not overlap"):
            paged.qk_rope(qkv, keys=keys, values=vals, eps=1e-6, out=rope_out,
                          **dict(plain, **{name: over(t, 4 * (last // 4))}))
