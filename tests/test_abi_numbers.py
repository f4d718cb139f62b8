"""Numbers that are finite as the caller has them and not as the kernels get them, in 32 bits, are refused; without a GPU."""
import pytest

from test_abi_paged import BATCH, CACHE, NULL, Call, F, P, lib  # noqa: F401
from test_abi_paged8 import CACHE8

INF = float("inf")
SCALES = [INF, -INF, float("nan"), 2.0 ** 127, -(2.0 ** 127)]


def _attention(fn, cache, *, more=None, behind=None, need=0):
    return Call(fn, q=P, q_stride=4096, **cache, **BATCH, **(more or {}), B=3, W=4, **(behind or {}), qh=32, kh=8, d=128, scale=F(0.1),
                out=P, workspace=P if need else NULL, workspace_bytes=need, dtype=0, stream=NULL)


@pytest.mark.parametrize("bits", [16, 8])
def test_scales(lib, bits):  # noqa: F811
    cache, end = (CACHE, "") if bits == 16 else (CACHE8, "_fp8")
    calls = [_attention(getattr(lib, "moss_paged_decode_attention" + end), cache, need=lib.moss_paged_decode_workspace_bytes(3, 4, 16, 32, 8, 128)),
             _attention(getattr(lib, "moss_paged_shared_decode_attention" + end), cache, more=dict(groups=P, shared=P),
                        need=lib.moss_paged_shared_workspace_bytes(3, 4, 16, 32, 8, 128)),
             _attention(getattr(lib, "moss_paged_prompt_attention" + end), cache, more=dict(starts=P), behind=dict(T=50))]
    for call in calls:
        for scale in SCALES:
            assert call(scale=F(scale)) == 1, scale


def test_penalties(lib):  # noqa: F811
    call = Call(lib.moss_adjust_rows, logits=P, dtype=0, rows=3, stride=5000, vocab=5000, tokens=P, token_bytes=8, token_row_stride=90,
                token_stride=1, width=90, lengths=P, prompt=P, repetition=NULL, repetition_value=F(1.0), presence=NULL,
                presence_value=F(0.0), frequency=NULL, frequency_value=F(0.0), bias_ids=NULL, bias_ids_stride=0, bias=NULL, bias_stride=0,
                biases=0, mask=NULL, mask_stride=0, out=P, out_stride=5000, stream=NULL)
    for name in ("repetition_value", "presence_value", "frequency_value"):
        for value in (INF, -INF, float("nan")):
            assert call(**{name: F(value)}) == 1, (name, value)
    for value in (0.0, -1.0):
        assert call(repetition_value=F(value)) == 1, value


def test_scales_in_python():
    from moss_tts._runtime import paged

    for scale in (1e39, -1e39, *SCALES):
        with pytest.raises(ValueError, match="finite"):
            paged._scale(scale, 64)
    assert paged._scale(1e30, 64) == 1e30 and paged._scale(-0.0, 64) == 0.0 and paged._scale(None, 64) == 0.125
