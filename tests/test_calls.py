"""The compiled calls without a GPU: what is no call of theirs is left to Python, whatever the arguments are."""
import os

import pytest
import torch

from moss_tts import _build

COUNTS = {"decode": 11, "prompt": 10, "qk_rope": 13, "gather": 8, "adjust": 11}
THINGS = [None, 1, 0, -5, 2.5, float("nan"), True, "x", (), (1, 2), [None, None], object(), 1 << 80, torch.zeros(3),
          torch.zeros((2, 4, 64), dtype=torch.bfloat16), torch.zeros((0, 3)), torch.zeros(2, 3).to_sparse(),
          torch.empty((2, 4, 64), dtype=torch.bfloat16, device="meta"), torch.nn.Parameter(torch.zeros(2, 2))]


@pytest.fixture(scope="module", autouse=True)
def built():
    if not (os.path.exists(_build.LIB) and os.path.exists(_build.CALLS)):
        _build.build()


@pytest.mark.parametrize("name", COUNTS)
def test_arguments_of_no_call(name):
    from moss_tts._runtime import native

    function = getattr(native.calls(), name)
    for thing in THINGS:
        assert function(*[thing] * COUNTS[name]) is None
        for i in range(COUNTS[name]):
            args = [torch.zeros((2, 4, 64), dtype=torch.bfloat16)] * COUNTS[name]
            args[i] = thing
            assert function(*args) is None
    for n in range(15):
        if n != COUNTS[name]:
            assert function(*[None] * n) is None


def test_init_needs_the_library():
    from moss_tts._runtime import native

    with pytest.raises(TypeError):
        native.calls().init(1)
    with pytest.raises(TypeError):
        native.calls().init(1, 2)
    with pytest.raises(TypeError):
        native.calls().init("x", print)
