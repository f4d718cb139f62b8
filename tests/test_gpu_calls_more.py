"""GPU: what the compiled calls leave to Python, and where they and Python's checks have to agree."""
import pytest
import torch

from test_gpu_calls import _batch, _call, _same

pytestmark = pytest.mark.gpu


class Named(torch.Tensor):
    """A tensor that its operations hand on as what it is."""


@pytest.mark.parametrize("name, of", [("decode_attention", "q"), ("shared_decode_attention", "q"), ("prompt_attention", "packed"),
                                      ("qk_rope", "qkv")])
def test_subclass_makes_its_outputs(dev, name, of):
    s = _batch(dev, torch.bfloat16, False)
    want = _call(s, name)
    assert type(want) is torch.Tensor
    setattr(s, of, getattr(s, of).as_subclass(Named))
    got = _call(s, name)
    assert type(got) is Named and _same(got.as_subclass(torch.Tensor), want)


def test_subclass_of_logits(dev):
    from moss_tts._runtime import sampling

    x = torch.randn((3, 700), generator=torch.Generator().manual_seed(0)).to(dev)
    mask = torch.full((1, 22), -2, dtype=torch.int32, device=dev)
    got = sampling.adjust(x.as_subclass(Named), mask=mask)
    assert type(got) is Named and _same(got.as_subclass(torch.Tensor), sampling.adjust(x, mask=mask))
