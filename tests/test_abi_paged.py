"""The C entries of the paged operators and the row sampler without a GPU: argument errors come back as
hipErrorInvalidValue before anything is launched, and the workspace sizes follow the shapes."""
import ctypes
import os

import pytest

P, ODD, NULL = ctypes.c_void_p(4096), ctypes.c_void_p(4100), None
F = ctypes.c_float


@pytest.fixture(scope="module")
def lib():
    from moss_tts import _build
    from moss_tts._runtime import native

    if not os.path.exists(native.LIB_PATH):
        _build.build()
    return native.lib()


class Call:
    """An entry's arguments by name, in order; ``call(name=value)`` calls it with one or more of them changed."""

    def __init__(self, fn, **args):
        self.fn, self.args = fn, args

    def __call__(self, **changes):
        assert set(changes) <= set(self.args)
        return self.fn(*{**self.args, **changes}.values())


CACHE = dict(k=P, v=P, k_stride=8 * 16 * 128, v_stride=8 * 16 * 128, pages=10, page_rows=16)
BATCH = dict(table=P, table_stride=4, lengths=P)
BAD_CACHE = [dict(k=NULL), dict(v=NULL), dict(k=ODD), dict(v=ODD), dict(k_stride=8 * 16 * 128 - 8), dict(v_stride=8 * 16 * 128 + 4),
             dict(pages=0), dict(page_rows=8), dict(page_rows=24), dict(page_rows=8192), dict(table=NULL), dict(table=ctypes.c_void_p(4097)),
             dict(table_stride=3), dict(lengths=NULL), dict(B=0), dict(B=65536), dict(W=0), dict(W=1 << 27), dict(qh=30), dict(qh=0),
             dict(qh=2048), dict(kh=0), dict(d=96), dict(d=256), dict(dtype=2), dict(dtype=-1)]


def test_decode_attention(lib):
    need = lib.moss_paged_decode_workspace_bytes(3, 4, 16, 32, 8, 128)
    call = Call(lib.moss_paged_decode_attention, q=P, q_stride=4096, **CACHE, **BATCH, B=3, W=4, qh=32, kh=8, d=128, scale=F(0.1),
                out=P, workspace=P, workspace_bytes=need, dtype=0, stream=NULL)
    for bad in BAD_CACHE + [dict(q=NULL), dict(q=ODD), dict(q_stride=4088), dict(q_stride=4100), dict(scale=F(float("nan"))),
                            dict(out=NULL), dict(out=ODD), dict(workspace=NULL), dict(workspace=ODD), dict(workspace_bytes=need - 1)]:
        assert call(**bad) == 1, bad


def test_decode_workspace(lib):
    size = lib.moss_paged_decode_workspace_bytes
    assert size(3, 4, 16, 32, 8, 128) == 3 * 32 * 130 * 4              # 64 rows: one share a sequence
    assert size(1, 64, 16, 32, 8, 128) == 8 * 32 * 130 * 4             # 1024 rows: 8 shares at most
    assert size(64, 1000, 16, 32, 8, 128) == (64 + 192) * 32 * 130 * 4
    for bad in ((0, 4, 16, 32, 8, 128), (3, 0, 16, 32, 8, 128), (3, 4, 17, 32, 8, 128), (3, 4, 16, 31, 8, 128), (3, 4, 16, 32, 8, 80)):
        assert size(*bad) == 0


def test_prompt_attention(lib):
    call = Call(lib.moss_paged_prompt_attention, q=P, q_stride=4096, **CACHE, **BATCH, starts=P, B=3, W=4, T=50, qh=32, kh=8, d=128,
                scale=F(0.1), out=P, workspace=NULL, workspace_bytes=0, dtype=0, stream=NULL)
    for bad in BAD_CACHE + [dict(q=NULL), dict(q=ODD), dict(q_stride=4088), dict(q_stride=4100), dict(scale=F(float("nan"))),
                            dict(out=NULL), dict(out=ODD), dict(starts=NULL), dict(T=0), dict(T=(1 << 20) + 1), dict(workspace=ODD),
                            dict(W=100, table_stride=100)]:            # 1600 rows: a workspace is needed
        assert call(**bad) == 1, bad
    need = lib.moss_paged_prompt_workspace_bytes(3, 100, 16, 50, 32, 8, 128)
    assert need > 0
    assert call(W=100, table_stride=100, workspace=P, workspace_bytes=need - 1) == 1


def test_prompt_workspace(lib):
    size = lib.moss_paged_prompt_workspace_bytes
    assert size(3, 32, 16, 50, 32, 8, 128) == 0                        # 512 rows: no tile is cut
    assert size(1, 33, 16, 1, 32, 8, 128) == 2 * 2 * 8 * 64 * 130 * 4  # two tiles at most, in two parts
    assert size(64, 4000, 16, 100000, 32, 8, 128) == 64 * 8 * 128 * 130 * 4
    assert size(3, 33, 16, 0, 32, 8, 128) == 0


def test_qk_rope(lib):
    call = Call(lib.moss_paged_qk_rope, qkv=P, qkv_stride=6144, q_weight=P, k_weight=P, cos=P, sin=P, table_f32=1, table_rows=100,
                q_out=P, **CACHE, **BATCH, starts=P, B=3, W=4, T=50, qh=32, kh=8, d=128, eps=F(1e-6), dtype=0, stream=NULL)
    for bad in BAD_CACHE + [dict(qkv=NULL), dict(qkv=ODD), dict(qkv_stride=6136), dict(qkv_stride=6148), dict(q_weight=NULL),
                            dict(k_weight=NULL), dict(q_weight=ODD), dict(cos=NULL), dict(sin=ODD), dict(table_rows=0), dict(q_out=NULL),
                            dict(q_out=ODD), dict(T=0), dict(eps=F(-1.0)), dict(starts=NULL)]:  # without starts T must be B
        assert call(**bad) == 1, bad


def test_sample_rows(lib):
    call = Call(lib.moss_sample_rows, logits=P, dtype=0, rows=3, stride=5000, vocab=5000, uniform=P, temperature=NULL,
                temperature_value=F(1.0), top_k=NULL, top_k_value=0, top_p=NULL, top_p_value=F(1.0), min_p=NULL, min_p_value=F(0.0),
                out=P, workspace=P, workspace_bytes=lib.moss_sample_rows_workspace_bytes(3, 5000), stream=NULL)
    for bad in [dict(logits=NULL), dict(logits=ctypes.c_void_p(4097)), dict(dtype=3), dict(dtype=-1), dict(rows=0), dict(stride=4999),
                dict(vocab=0), dict(vocab=(1 << 19) + 1, stride=1 << 20), dict(uniform=NULL), dict(uniform=ctypes.c_void_p(4098)),
                dict(temperature=ctypes.c_void_p(4098)), dict(top_k=ctypes.c_void_p(4098)), dict(out=NULL), dict(out=ODD),
                dict(workspace=NULL), dict(workspace=ODD),
                dict(workspace_bytes=lib.moss_sample_rows_workspace_bytes(3, 5000) - 1)]:
        assert call(**bad) == 1, bad
    assert lib.moss_sample_rows_workspace_bytes(3, 2048) == 0
    assert lib.moss_sample_rows_workspace_bytes(0, 5000) == 0
    assert lib.moss_sample_rows_workspace_bytes(3, (1 << 19) + 1) == 0


def test_sample_workspace_serves_smaller_calls(lib):
    """A workspace for some rows and entries is enough for fewer of either."""
    size = lib.moss_sample_rows_workspace_bytes
    rows = [1, 2, 3, 17, 63, 64, 65, 100, 128, 129, 511, 512, 513, 1023, 1024, 1025, 5000]
    vocabs = [2049, 2560, 4096, 4097, 8191, 8193, 16385, 50000, 65537, 100000, 151936, 262145, 1 << 19]
    for n in rows:
        sizes = [size(n, v) for v in vocabs]
        assert sizes == sorted(sizes)
    for v in vocabs:
        sizes = [size(n, v) for n in rows]
        assert sizes == sorted(sizes)
