"""GPU: what sequences share counts by what is taken of it: rows that only the first one names save nothing, and are not read on
their own."""
import pytest
import torch

from test_gpu_paged_shared import _batch

pytestmark = pytest.mark.gpu

N, P = 9, 4096


def _out(dev, groups, shared, lengths, bits):
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(3)
    keys, vals, scales, table, lens = _batch(dev, g, [0] * N, [P] * N, lengths, kh=8, d=128, page=16, dtype=torch.bfloat16, bits=bits)
    q = (torch.randn((N, 32, 128), generator=g) * 1.5).bfloat16().to(dev)
    ids, most = (torch.tensor(t, dtype=torch.int32, device=dev) for t in (groups, shared))
    out = paged.shared_decode_attention(q, keys, vals, table, lens, ids, most, scales=scales)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("shared, lengths, same_as", [
    ([P] + [0] * 8, [4200 + i for i in range(N)], None),              # nobody takes what the first one shares
    ([P] + [15] * 8, [4200 + i for i in range(N)], None),             # nor less than 16 rows
    ([P] * N, [4200] + [20 + i for i in range(8)], None),             # short sequences save little
    ([P] + [2048] * 8, [4200 + i for i in range(N)], [2048] * N),     # half of it is shared, and half is read for all
    # the second one ends within its 2050, so it takes all of its 2049 rows: 2064 are read
    ([P] + [2050, 16, 0] + [2048] * 5, [4200, 2049] + [4200] * 7, [2064, 2050, 16, 0] + [2048] * 5),
])
def test_only_what_is_taken(dev, shared, lengths, same_as, bits):
    print(shared, lengths, bits, flush=True)
    got = _out(dev, [0] * N, shared, lengths, bits)
    want = _out(dev, [-1] * N if same_as is None else [0] * N, same_as or [0] * N, lengths, bits)
    assert torch.isfinite(got).all() and torch.equal(got, want)
