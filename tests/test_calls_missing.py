"""Without the compiled calls, or with those of another torch, Python makes the batch operators' calls by itself."""
import os
import shutil

import pytest
import torch

from moss_tts import _build


@pytest.fixture(scope="module", autouse=True)
def built():
    if not (os.path.exists(_build.LIB) and os.path.exists(_build.CALLS)):
        _build.build()


@pytest.fixture
def calls_at(monkeypatch):
    """``calls`` as a process finds it whose compiled module lies at the path given."""
    from moss_tts._runtime import native

    def use(path):
        monkeypatch.setattr(native, "CALLS_PATH", str(path))
        native.calls.cache_clear()
        return native.calls
    yield use
    monkeypatch.undo()
    native.calls.cache_clear()


def _refused():
    from moss_tts._runtime import paged, sampling

    x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    for call in (lambda: paged.decode_attention(x, x, x, x, x), lambda: paged.shared_decode_attention(x, x, x, x, x, x, x),
                 lambda: paged.prompt_attention(x, x, x, x, x, x), lambda: paged.gather(x, x, x, x, x, 3),
                 lambda: paged.qk_rope(x, None, None, x, x, x, x, x, x, 1e-6), lambda: sampling.adjust(x)):
        with pytest.raises(ValueError):
            call()


def test_absent(calls_at, tmp_path):
    calls = calls_at(tmp_path / "none.so")
    with pytest.warns(RuntimeWarning, match="not built"):
        taken = calls()
    assert taken.decode(*[None] * 11) is None and taken.adjust(*[None] * 11) is None
    _refused()


def test_no_module(calls_at, tmp_path):
    path = tmp_path / "_moss_calls.so"
    path.write_bytes(b"\x7fELF and nothing behind it")
    with pytest.warns(RuntimeWarning):
        calls_at(path)()
    _refused()


def test_another_torchs(calls_at, monkeypatch):
    from moss_tts._runtime import native

    tag = native.calls_tag()
    assert torch.__version__ in tag
    monkeypatch.setattr(native, "calls_tag", lambda: tag + " of another day")
    with pytest.warns(RuntimeWarning, match="another day"):
        calls_at(native.CALLS_PATH)()
    _refused()


def test_a_patch_release_is_the_same_python(monkeypatch):
    from moss_tts._runtime import native

    tag = native.calls_tag()
    monkeypatch.setattr(native.sys, "version_info", (*native.sys.version_info[:2], 99, "final", 0))
    assert native.calls_tag() == tag
    monkeypatch.setattr(native.sys, "version_info", (3, 99, 0, "final", 0))
    assert native.calls_tag() != tag


def test_this_ones(calls_at):
    from moss_tts._runtime import native

    calls = calls_at(native.CALLS_PATH)
    assert calls().built_for == native.calls_tag()


def test_built_without_a_host_compiler(calls_at, monkeypatch, tmp_path):
    """hipcc alone builds the module, as it does the library."""
    from moss_tts._runtime import native

    hipcc, which = _build.hipcc(), shutil.which
    monkeypatch.setattr(_build.shutil, "which", lambda name: None if name in ("g++", "c++") else which(name))
    monkeypatch.setattr(_build, "hipcc", lambda: hipcc)
    monkeypatch.setattr(_build, "CALLS", str(tmp_path / "_moss_calls.so"))
    _build._compile_calls(False)
    calls = calls_at(_build.CALLS)
    assert calls().built_for == native.calls_tag() and calls().decode(*[None] * 11) is None
