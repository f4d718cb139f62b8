"""The 64-bit prompt attention of whole tensors (``paged_helpers.attend_all``) against the definition, one token and head
at a time (``oracle.paged``)."""
import numpy as np
import pytest
import torch

from oracle import paged as o
from paged_helpers import attend_all, cache, values


@pytest.mark.parametrize("layout", [(6, 2, 64), (4, 4, 128), (5, 1, 64)])
def test_prompt_reference(layout):
    g = torch.Generator().manual_seed(3)
    qh, kh, d = layout
    new, old = [20, 1, 0, 33, 9, 6], [0, 30, 9, 14, 3, 0]
    keys, vals, table, lens = cache("cpu", g, [a + b for a, b in zip(new, old)], kh=kh, d=d, page=16, dtype=torch.bfloat16)
    table[3, 1] = -1
    table[1, :] = 10 ** 9
    lens[4] = 4
    lens[5] = -3
    starts = np.concatenate(([0], np.cumsum(new)))
    q = torch.randn((sum(new) + 2, qh, d), generator=g)
    before = torch.full((sum(new) + 2, qh * d), 7.0)
    want = o.prompt_attention(values(q), values(keys), values(vals), table.numpy(), lens.numpy(), starts, values(before), -0.3)
    got = attend_all(q, keys, vals, table, lens, starts.tolist(), before, -0.3)
    assert np.abs(got.numpy() - want).max() <= 1e-12
