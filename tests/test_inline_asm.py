"""Wait states that the compiler cannot see to: hipcc inserts them between the
instructions it schedules, not inside an inline asm statement.

gfx9 (gfx950 among it) needs one wait state between a scalar write of M0 and a
load to LDS that takes its address from it; without it the load may go to the
address before."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "s4000-moe-engine_amd" / "csrc"
SOURCES = sorted(p for p in CSRC.iterdir() if p.suffix in (".hip", ".h"))
COMMENT = re.compile(r"//[^\n]*|/\*.*?\*/", re.S)
ASM = re.compile(r"\basm\s+(?:volatile\s*)?\(")
STRING = re.compile(r'\s*"((?:[^"\\]|\\.)*)"')
WRITES_M0 = re.compile(r"s_\w+\s+m0\b")
LOADS_LDS = re.compile(r"buffer_load_\w+\b.*\blds\b|(?:global|scratch)_load_lds_\w+")


def _statements(text):
    """The instructions of every asm statement, in order."""
    text = COMMENT.sub("", text)
    for start in ASM.finditer(text):
        at, body = start.end(), ""
        while True:
            piece = STRING.match(text, at)
            if piece is None:
                break
            body += piece.group(1)
            at = piece.end()
        lines = re.split(r"\\n|;", body.replace("\\t", " "))
        yield [line.strip() for line in lines if line.strip()]


def _unwaited(lines):
    return [(a, b) for a, b in zip(lines, lines[1:])
            if WRITES_M0.match(a) and LOADS_LDS.match(b)]


@pytest.mark.parametrize("path", SOURCES, ids=[p.name for p in SOURCES])
def test_a_load_to_lds_waits_for_its_m0(path):
    for lines in _statements(path.read_text()):
        assert not _unwaited(lines), f"{path.name}: no wait state in {lines}"


def test_the_scan_finds_such_loads():
    found = [lines for p in SOURCES for lines in _statements(p.read_text())
             if any(LOADS_LDS.match(x) for x in lines)]
    assert len(found) >= 3          # the two helpers and the ring's own
    assert all(any(WRITES_M0.match(x) for x in lines) for lines in found)
    bad = 'asm volatile("s_mov_b32 m0, %0\\n\\t"\n "buffer_load_dwordx4 %1, %2, 0 offen lds");'
    (lines,) = _statements(bad)
    assert _unwaited(lines)
    assert _unwaited(["s_add_u32 m0, m0, s3", "global_load_lds_dwordx4 v[0:1], off"])
    assert not _unwaited(["s_mov_b32 m0, s3", "s_nop 0", "global_load_lds_dwordx4 v[0:1], off"])
