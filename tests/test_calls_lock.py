"""The compiled calls and the interpreter's lock, by their source: a device allocation cannot be watched without a GPU."""
import os
import re

from moss_tts import _build


def test_memory_is_asked_for_without_the_interpreters_lock():
    """A device allocation may take long, and stops no other thread: one function asks for memory, and it has let go."""
    with open(os.path.join(_build.CSRC, "host", "calls.cpp")) as f:
        text = re.sub(r"//.*", "", f.read())
    asks = [m.start() for m in re.finditer(r"\bat::(empty|zeros|full|empty_like|new_empty)\w*\(", text)]
    assert len(asks) == 1
    function = re.search(r"at::Tensor fresh\([^{]*\{(.*?)\n\}", text, re.S)
    assert function.start() < asks[0] < function.end()
    assert text.index("Unlocked now;") < asks[0] and "PyEval_SaveThread()" in text and "~Unlocked() { PyEval_RestoreThread(state); }" in text
