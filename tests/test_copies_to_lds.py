"""Copies from global memory to LDS in inline assembly hold the wait states that the compiler cannot add inside a string."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashact_amd", "csrc")
STRING = re.compile(r'"((?:[^"\\]|\\.)*)"')


def _copies(text):
    """The instructions of every assembly string that copies to LDS."""
    for s in STRING.findall(text):
        if "global_load_lds" in s or "buffer_load" in s and " lds" in s:
            yield [i.strip() for i in s.replace("\\t", "").split("\\n")]


def _states(instructions):
    """Wait states that instructions stand for: one each, n + 1 for `s_nop n`."""
    return sum(int(i.split()[1]) + 1 if i.startswith("s_nop") else 1 for i in instructions)


def _check(instructions):
    at = next(i for i, x in enumerate(instructions) if "load" in x)
    to_m0 = max(i for i, x in enumerate(instructions[:at]) if x.startswith("s_mov_b32 m0"))
    assert _states(instructions[to_m0 + 1:at]) >= 1, instructions  # a scalar write of m0, then a copy to LDS
    if not re.search(r"\boff\b", instructions[at]):  # a scalar base, which a vector instruction may have written just before
        assert _states(instructions[:at]) >= 5, instructions


def test_every_copy_waits_for_m0_and_its_base():
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))):
        text = "\n".join(line.split("//", 1)[0] for line in open(path))
        for instructions in _copies(text):
            _check(instructions)
            found += 1
    assert found


@pytest.mark.parametrize("text", [
    r'"s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"',
    r'"s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"',
])
def test_the_check_finds_what_is_missing(text):
    (instructions,) = _copies(text)
    with pytest.raises(AssertionError):
        _check(instructions)
