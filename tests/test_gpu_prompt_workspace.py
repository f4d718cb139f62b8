"""GPU: prompt attention with a kept workspace of each form's size, where the forms' sizes differ."""
import numpy as np
import pytest
import torch

from paged_helpers import attend_all, attention_bound, cache, cache8, cache8_values, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("bits", [16, 8])
def test_kept_workspaces(dev, monkeypatch, bits, compiled):
    from moss_tts._runtime import native, paged

    if not compiled:
        monkeypatch.setattr(native, "calls", lambda: native._NoCalls)
    g = torch.Generator().manual_seed(11)
    qh, kh, d, new, old = 32, 8, 128, [1900, 300, 1], [0, 1200, 2900]  # 552 whole tiles, some cut into parts
    lengths = [a + b for a, b in zip(new, old)]
    if bits == 16:
        keys, vals, table, lens = cache(dev, g, lengths, kh=kh, d=d, page=64, dtype=torch.bfloat16)
        scales, pages = None, [torch.nan_to_num(t.double()) for t in (keys, vals)]
    else:
        keys, vals, scales, table, lens = cache8(dev, g, lengths, kh=kh, d=d, page=64)
        pages = [np.nan_to_num(cache8_values(*t), posinf=0.0) for t in ((keys, scales[0]), (vals, scales[1]))]
        pages = [torch.from_numpy(np.where(np.abs(t) < 1e6, t, 0.0)).to(dev) for t in pages]
    q = (torch.randn((sum(new), qh, d), generator=g) * 1.5).bfloat16().to(dev)
    starts = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device=dev)
    shape = len(new), table.shape[1], 64, sum(new), qh, kh, d
    plain, eight = native.lib().moss_paged_prompt_workspace_bytes(*shape), native.lib().moss_paged_prompt_workspace_bytes_fp8(*shape)
    assert eight == 2 * plain
    assert 4 * paged.prompt_workspace(q, keys, table).numel() == (plain if bits == 16 else eight)
    rest = table, lens, starts.tolist(), torch.zeros((sum(new), qh * d), device=dev), d ** -0.5
    ref, ref_abs = attend_all(q, *pages, *rest), attend_all(q, pages[0], pages[1].abs(), *rest)
    bound = attention_bound(values(q), values(pages[0]), values(pages[1]), values(ref), values(ref_abs), d ** -0.5, torch.bfloat16, True)
    outs = {}
    for nbytes in (None, plain, plain + 16, eight):
        ws = None if nbytes is None else torch.full((nbytes // 4 + 64,), float("nan"), device=dev)[:nbytes // 4]
        print(f"prompt workspace bits={bits} compiled={compiled} bytes={nbytes}", flush=True)
        out = paged.prompt_attention(q, keys, vals, table, lens, starts, scales=scales, ws=ws)
        torch.cuda.synchronize()
        assert (np.abs(values(out) - values(ref)) <= bound).all(), nbytes
        outs[nbytes] = out
    assert torch.equal(outs[None], outs[eight])
    assert torch.equal(outs[plain], outs[plain + 16])
    with pytest.raises(ValueError):
        paged.prompt_attention(q, keys, vals, table, lens, starts, scales=scales, ws=torch.zeros(plain // 4 - 1, device=dev))
