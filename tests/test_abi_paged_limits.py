"""The C entries of the paged operators refuse, before anything is launched, what their grids cannot hold."""
import ctypes
import os

import pytest

P, F = ctypes.c_void_p(4096), ctypes.c_float


@pytest.fixture(scope="module")
def lib():
    from moss_tts import _build
    from moss_tts._runtime import native

    if not os.path.exists(native.LIB_PATH):
        _build.build()
    return native.lib()


@pytest.mark.parametrize("tokens", [1 << 24, (1 << 24) + 1, 2 ** 31 - 1])
def test_qk_rope_tokens(lib, tokens):
    """256 threads a token: 2^24 tokens would be 2^32 threads."""
    assert lib.moss_paged_qk_rope(P, 192, None, None, P, P, 1, 100, P, P, P, 16 * 64, 16 * 64, 10, 16, P, 4, P, P, 1, 4, tokens,
                                  1, 1, 64, F(1e-6), 0, None) == 1
