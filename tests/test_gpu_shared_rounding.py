"""GPU: a shared prefix costs a sequence no bits: its output is as near to the definition as decode_attention's, whoever stands
beside it in the batch."""
import numpy as np
import pytest
import torch

from oracle import paged as o
from paged_helpers import cache8_values, values
from shared_helpers import prefix_taken, shared_workspace
from test_gpu_paged_shared import _batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout, count, prefix", [((32, 8, 128), 9, 2048), ((16, 8, 64), 9, 2048),      # tiles of 64 rows
                                                   ((32, 8, 128), 131, 160), ((16, 8, 64), 260, 96)])    # of 128
def test_as_near_as_alone(dev, layout, count, prefix, dtype, bits):
    """Both forms take their weights as two 16-bit values, off by 2^-17 at most, and sum in 32 bits: what differs from the 64-bit
    value rounded to the type are outputs near a border, one in 2^8 or fewer of them, in either form.  The norm of the difference goes
    with the root of the error, so four times the other's allows sixteen times its error; weights rounded to 16 bits have 2^6
    (fp16) to 2^9 times it, and leave hardly an output's last bit alone."""
    from moss_tts._runtime import paged

    g = torch.Generator().manual_seed(41)
    qh, kh, d = layout
    groups, shared = [0] * count, [prefix] * count
    lengths = [prefix + 1 + 3 * i % 20 for i in range(count)]
    keys, vals, scales, table, lens = _batch(dev, g, groups, shared, lengths, kh=kh, d=d, page=16, dtype=dtype, bits=bits)
    if bits == 8:  # rows of one size, so that many take part
        for t in scales:
            t[t != 255] = torch.where(t[t != 255] == 0, 0, 120).to(torch.uint8)
    q = (torch.randn((count, qh, d), generator=g) * 0.05).to(dtype).to(dev)
    ids, most = (torch.tensor(t, dtype=torch.int32, device=dev) for t in (groups, shared))
    print(f"rounding {layout} count={count} {dtype} bits={bits}", flush=True)
    ws = shared_workspace(q, keys, table)
    together = paged.shared_decode_attention(q, keys, vals, table, lens, ids, most, scales=scales, ws=ws)
    alone = paged.decode_attention(q, keys, vals, table, lens, scales=scales)
    torch.cuda.synchronize()
    pages = (values(keys), values(vals)) if bits == 16 else (cache8_values(keys, scales[0]), cache8_values(vals, scales[1]))
    ref = o.decode_attention(values(q), *pages, table.cpu().numpy(), lens.cpu().numpy(), None)
    want = values(torch.from_numpy(ref).to(dtype))
    off = [float(np.linalg.norm(values(t) - want) / np.linalg.norm(want)) for t in (together, alone)]
    share = [float((values(t) != want).mean()) for t in (together, alone)]
    print(off, share, flush=True)
    assert prefix_taken(ws, q, keys)
    assert off[0] <= 4 * off[1] + torch.finfo(dtype).eps * 2.0 ** -6, (off, share)
