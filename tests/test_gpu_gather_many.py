"""GPU: cached rows of more tokens than one grid holds."""
import pytest
import torch

from paged_helpers import cache, cache8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
def test_tokens_past_a_grid(dev, bits):
    """2^23 tokens of 32 KV heads of 128 are 2^32 threads.  All but the newest of the first sequence stand before its first row
    and give zeros; those behind the last sequence are left."""
    from moss_tts._runtime import paged

    tokens, kh, d = (1 << 23) + 9, 32, 128
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("150 GB of free memory required")
    print(f"gather tokens={tokens} bits={bits}", flush=True)
    g = torch.Generator().manual_seed(0)
    if bits == 16:
        keys, vals, table, lens = cache(dev, g, [20, 3], kh=kh, d=d, page=16, dtype=torch.bfloat16)
        scales = None
    else:
        keys, vals, scales, table, lens = cache8(dev, g, [20, 3], kh=kh, d=d, page=16)
    few = paged.gather(keys, vals, table, lens, torch.tensor([0, 20, 23], dtype=torch.int32, device=dev), 23, scales=scales)
    first = tokens - 5  # tokens of the first sequence
    starts = torch.tensor([0, first, first + 3], dtype=torch.int32, device=dev)
    out = tuple(torch.full((tokens, kh, d), 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
    paged.gather(keys, vals, table, lens, starts, tokens, scales=scales, out=out)
    torch.cuda.synchronize()
    for got, want in zip(out, few):
        assert torch.equal(got[first - 20:first + 3], want)
        assert (got[first + 3:] == 7.0).all()
        step = 1 << 19
        for at in range(0, first - 20, step):
            assert not got[at:min(at + step, first - 20)].any(), at
    del out
    torch.cuda.empty_cache()
