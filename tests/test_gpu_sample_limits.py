"""GPU: ``sampling.sample`` at the ends of its ranges: rows whose kept weight comes near 2^63, and buffers that share memory."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
VOCAB = 1 << 19
# above 0.9975 the draw of 2^19 entries of full weight passes 9.2 10^18 units of 2^-44
UNIFORM = [0.0, 0.25, 0.9974, 0.998, 0.9995, 0.9999, 1.0 - 2.0 ** -24, 1.0, 1e30, math.inf]


@pytest.mark.parametrize("rows", [3, 20])  # few rows; rows that one workgroup each draws (bf16)
@pytest.mark.parametrize("kind", ["equal", "hot"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_that_sum_to_two_to_the_63(dev, dtype, kind, rows):
    """Every entry weighs 1, so the draw is floor(u entries), and the last entry from u = 1 on: equal logits, and logits
    whose distance a temperature of 1e30 takes away.  All numbers are exact: 2^44 an entry, u of 24 bits."""
    from moss_tts._runtime import sampling

    g = torch.Generator().manual_seed(1)
    x = torch.full((rows, VOCAB), 1.5) if kind == "equal" else torch.randn((rows, VOCAB), generator=g)
    x = x.to(dtype).to(dev)
    temperature = 1.0 if kind == "equal" else 1e30
    for first in range(0, len(UNIFORM), rows):
        u = np.float32((UNIFORM[first:] + UNIFORM * 3)[:rows])
        print(f"sample {kind} {dtype} rows={rows} from u={u[0]}", flush=True)
        got = sampling.sample(x, torch.from_numpy(u).to(dev), temperature=temperature).tolist()
        assert got == [int(min(float(v) * VOCAB, VOCAB - 1)) for v in u]
        # half of the entries by top-p: the ones whose predecessors weigh at most half of all
        kept = VOCAB // 2 + 1
        if kind == "equal":
            got = sampling.sample(x, torch.from_numpy(u).to(dev), top_p=0.5).tolist()
            assert got == [int(min(float(v) * kept, kept - 1)) for v in u]


def test_buffers_that_share_memory(dev):
    """The draw of one row writes its index while others still read: an output or a workspace that lies over the logits, the
    uniform numbers, a setting or each other is refused."""
    from moss_tts._runtime import sampling

    n, vocab = 4, 3000
    need = sampling.sample_workspace(n, vocab, dev).numel()
    memory = torch.zeros(need + 4096, device=dev)
    x, u = torch.zeros((n, vocab), device=dev), torch.zeros(n, device=dev)
    t, k = torch.ones(n, device=dev), torch.zeros(n, dtype=torch.int32, device=dev)
    p, m = torch.ones(n, device=dev), torch.zeros(n, device=dev)
    out = torch.zeros(n, dtype=torch.int64, device=dev)
    plain = dict(temperature=t, top_k=k, top_p=p, min_p=m)
    assert sampling.sample(x, u, **plain, out=out, ws=memory[:need]).tolist() == [0] * n
    inside = memory[need - n:need]
    for name in plain:
        bad = dict(plain, **{name: inside.view(plain[name].dtype)})
        with pytest.raises(ValueError, match="ws must not overlap"):
            sampling.sample(x, u, **bad, out=out, ws=memory[:need])
        over = inside if name == "temperature" else memory[:n]
        with pytest.raises(ValueError, match="out must not overlap"):
            sampling.sample(x, u, **dict(plain, **{name: over.view(plain[name].dtype)}),
                            out=(memory[need - 2 * n:need] if name == "temperature" else memory[:2 * n]).view(torch.int64))
    with pytest.raises(ValueError, match="out must not overlap"):
        sampling.sample(x, inside, **plain, out=memory[need - 2 * n:need].view(torch.int64))
    with pytest.raises(ValueError, match="out must not overlap"):
        sampling.sample(x, u, **plain, out=x.view(torch.int64)[0, :n])
    with pytest.raises(ValueError, match="ws must not overlap"):
        sampling.sample(x, u, **plain, out=memory[need - 2 * n:need].view(torch.int64), ws=memory[:need])


def test_more_rows_than_a_call_takes(dev):
    from moss_tts._runtime import sampling

    rows = 1 << 21
    x, u = torch.zeros((rows + 1, 2), dtype=torch.bfloat16, device=dev), torch.full((rows + 1,), 0.75, device=dev)
    with pytest.raises(ValueError, match="at most 2097152 rows"):
        sampling.sample(x, u)
    assert (sampling.sample(x[:rows], u[:rows]) == 1).all()


@pytest.mark.parametrize("vocab", [9, 3000])
def test_entries_without_weight_are_not_drawn(dev, vocab):
    """u = 0 draws the first entry that weighs anything: 2^-44 of the largest does, 2^-46 does not."""
    from moss_tts._runtime import sampling

    x = torch.full((2, vocab), -math.inf)
    x[:, 3], x[:, 7] = torch.tensor([-44 * math.log(2.0), -46 * math.log(2.0)]), 0.0
    assert sampling.sample(x.to(dev), torch.zeros(2, device=dev)).tolist() == [3, 7]
