"""GPU: numbers that 32 bits do not hold, through the compiled calls and Python's."""
import pytest
import torch

from test_gpu_calls import _batch, _call

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["compiled", "python"])
def made_by(request, monkeypatch):
    from moss_tts._runtime import native

    if not request.param:
        monkeypatch.setattr(native, "calls", lambda: native._NoCalls)


@pytest.mark.parametrize("name", ["decode_attention", "shared_decode_attention", "prompt_attention"])
def test_scales(dev, made_by, name):
    s = _batch(dev, torch.bfloat16, False)
    _call(s, name, scale=1.0)
    for scale in (1e39, -1e39, 2.0 ** 127, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="finite"):
            _call(s, name, scale=scale)


def test_penalties(dev, made_by):
    from moss_tts._runtime import sampling

    x, tokens = torch.zeros((2, 50), device=dev), torch.zeros((2, 3), dtype=torch.int64, device=dev)
    sampling.adjust(x, tokens=tokens, repetition=1e-30, presence=3e38, frequency=-3e38)
    for name in ("repetition", "presence", "frequency"):
        for value in (1e39, -1e39, float("inf"), float("nan")):
            with pytest.raises(ValueError):
                sampling.adjust(x, tokens=tokens, **{name: value})
    for value in (1e-50, 0.0, -1.0):  # the first is 0 in 32 bits
        with pytest.raises(ValueError, match="positive"):
            sampling.adjust(x, tokens=tokens, repetition=value)
