"""GPU: logit adjustments of more rows than one grid holds."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_rows_past_a_grid(dev):
    """2^21 rows of two chunks each, of 2^15 tokens and more a row, are 2^32 threads: 34 GB of logits, adjusted in place."""
    from moss_tts._runtime import sampling

    rows, vocab, width = 1 << 21, 8190, 1 << 15
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("48 GB of free memory required")
    print(f"adjust rows={rows} vocab={vocab}", flush=True)
    logits = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=dev)
    said = torch.randint(0, vocab, (1, width), generator=torch.Generator().manual_seed(0), dtype=torch.int32).to(dev)
    row = torch.arange(rows, device=dev)
    lengths = (row * 5 % 7).int()
    ids, bias = torch.tensor([[3, 8189]], dtype=torch.int32, device=dev), torch.tensor([[2.0, 4.0]], device=dev)
    mask = torch.full((1, 256), -1, dtype=torch.int32, device=dev)
    mask[0, 1] = ~(1 << 5)
    out = sampling.adjust(logits, tokens=said.expand(rows, width), lengths=lengths, presence=1.0, bias_ids=ids, bias=bias, mask=mask,
                          out=logits)
    torch.cuda.synchronize()
    assert out is logits
    kinds = torch.zeros((7, vocab), device=dev)  # a row's length decides what it is
    for n in range(7):
        kinds[n, said[0, :n].long()] -= 1.0
    kinds[:, 3] += 2.0
    kinds[:, 8189] += 4.0
    kinds[:, 37] = float("-inf")
    kinds = kinds.bfloat16()
    step = 1 << 15
    for first in range(0, rows, step):
        assert torch.equal(logits[first:first + step], kinds[lengths[first:first + step].long()]), first


def test_refused_by_name(dev):
    """Shapes that no memory holds, of one entry."""
    from moss_tts._runtime import sampling

    x = torch.zeros(1, dtype=torch.bfloat16, device=dev)
    for shape, name in (((1 << 20, 1 << 19), "logits"), (((1 << 21) + 1, 4), "rows"), ((4, (1 << 19) + 1), "entries")):
        with pytest.raises(ValueError, match=name):
            sampling.adjust(x.as_strided(shape, (0, 0)))
