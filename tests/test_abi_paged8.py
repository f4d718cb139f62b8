"""The C entries of the 8-bit paged operators and of the logit adjustments without a GPU: argument errors come back as
hipErrorInvalidValue before anything is launched."""
import ctypes

import pytest

from test_abi_paged import BAD_CACHE, BATCH, NULL, ODD, Call, F, P, lib  # noqa: F401

CACHE8 = dict(k=P, v=P, k_scales=P, v_scales=P, k_stride=8 * 16 * 128, v_stride=8 * 16 * 128, k_scale_stride=8 * 16,
              v_scale_stride=8 * 16, pages=10, page_rows=16)
BAD_CACHE8 = BAD_CACHE + [dict(k_scales=NULL), dict(v_scales=NULL), dict(k_scales=ODD), dict(v_scales=ODD), dict(k_scale_stride=127),
                          dict(v_scale_stride=112), dict(k_scale_stride=136), dict(k_stride=8 * 16 * 128 + 8),
                          dict(v_stride=8 * 16 * 128 + 8)]


def test_decode_attention(lib):  # noqa: F811
    need = lib.moss_paged_decode_workspace_bytes(3, 4, 16, 32, 8, 128)
    call = Call(lib.moss_paged_decode_attention_fp8, q=P, q_stride=4096, **CACHE8, **BATCH, B=3, W=4, qh=32, kh=8, d=128, scale=F(0.1),
                out=P, workspace=P, workspace_bytes=need, dtype=0, stream=NULL)
    for bad in BAD_CACHE8 + [dict(q=NULL), dict(q=ODD), dict(q_stride=4088), dict(q_stride=4100), dict(scale=F(float("nan"))),
                             dict(out=NULL), dict(out=ODD), dict(workspace=NULL), dict(workspace=ODD), dict(workspace_bytes=need - 1)]:
        assert call(**bad) == 1, bad


def test_qk_rope(lib):  # noqa: F811
    call = Call(lib.moss_paged_qk_rope_fp8, qkv=P, qkv_stride=6144, q_weight=P, k_weight=P, cos=P, sin=P, table_f32=1, table_rows=100,
                q_out=P, **CACHE8, **BATCH, starts=P, B=3, W=4, T=50, qh=32, kh=8, d=128, eps=F(1e-6), dtype=0, stream=NULL)
    for bad in BAD_CACHE8 + [dict(qkv=NULL), dict(qkv_stride=6136), dict(q_weight=NULL), dict(cos=NULL), dict(sin=ODD), dict(table_rows=0),
                             dict(q_out=ODD), dict(T=0), dict(T=1 << 24), dict(eps=F(-1.0)), dict(starts=NULL)]:
        assert call(**bad) == 1, bad


@pytest.mark.parametrize("bits", [16, 8])
def test_gather(lib, bits):  # noqa: F811
    from test_abi_paged import CACHE

    fn, cache = (lib.moss_paged_gather, CACHE) if bits == 16 else (lib.moss_paged_gather_fp8, CACHE8)
    call = Call(fn, **cache, **BATCH, starts=P, B=3, W=4, T=50, kh=8, d=128, k_out=P, v_out=P, dtype=0, stream=NULL)
    bad_cache = [b for b in (BAD_CACHE if bits == 16 else BAD_CACHE8) if "qh" not in b]
    for bad in bad_cache + [dict(starts=NULL), dict(starts=ctypes.c_void_p(4098)), dict(T=0), dict(T=1 << 24), dict(k_out=NULL),
                            dict(v_out=ODD), dict(kh=1025, k_stride=1 << 30, v_stride=1 << 30)]:
        assert call(**bad) == 1, bad


def test_adjust_rows(lib):  # noqa: F811
    H = ctypes.c_void_p(4098)
    call = Call(lib.moss_adjust_rows, logits=P, dtype=0, rows=3, stride=5000, vocab=5000, tokens=P, token_bytes=8, token_row_stride=90,
                token_stride=1, width=90, lengths=P, prompt=P, repetition=P, repetition_value=F(1.0), presence=P, presence_value=F(0.0),
                frequency=P, frequency_value=F(0.0), bias_ids=P, bias_ids_stride=4, bias=P, bias_stride=4, biases=4, mask=P,
                mask_stride=157, out=P, out_stride=5000, stream=NULL)
    for bad in [dict(logits=NULL), dict(out=NULL), dict(logits=ctypes.c_void_p(4097)), dict(logits=H, dtype=2), dict(out=H, dtype=2),
                dict(dtype=3), dict(dtype=-1), dict(rows=0), dict(rows=(1 << 21) + 1), dict(vocab=0), dict(stride=4999), dict(out_stride=4999),
                dict(vocab=(1 << 19) + 1, stride=1 << 20, out_stride=1 << 20, mask_stride=1 << 20), dict(token_bytes=2), dict(tokens=ODD),
                dict(tokens=NULL), dict(width=0), dict(width=(1 << 30) + 1), dict(token_stride=-1), dict(token_row_stride=-1), dict(lengths=H), dict(prompt=H),
                dict(repetition=H), dict(presence=H), dict(frequency=H), dict(bias=NULL), dict(bias_ids=NULL), dict(bias=H),
                dict(bias_ids=H), dict(biases=0), dict(biases=1 << 16, bias_stride=0, bias_ids_stride=0), dict(bias_stride=3),
                dict(bias_ids_stride=3), dict(mask=H), dict(mask_stride=156),
                dict(rows=1 << 21, vocab=1 << 19, stride=1 << 19, out_stride=1 << 19, mask_stride=0)]:
        assert call(**bad) == 1, bad


def test_prompt_attention(lib):  # noqa: F811
    call = Call(lib.moss_paged_prompt_attention_fp8, q=P, q_stride=4096, **CACHE8, **BATCH, starts=P, B=3, W=4, T=50, qh=32, kh=8, d=128,
                scale=F(0.1), out=P, workspace=NULL, workspace_bytes=0, dtype=0, stream=NULL)
    for bad in BAD_CACHE8 + [dict(q=NULL), dict(q=ODD), dict(q_stride=4088), dict(q_stride=4100), dict(scale=F(float("nan"))),
                             dict(out=NULL), dict(out=ODD), dict(starts=NULL), dict(T=0), dict(T=(1 << 20) + 1), dict(workspace=ODD),
                             dict(W=100, table_stride=100)]:
        assert call(**bad) == 1, bad
