"""CPU test of the kernels' inline assembly: a register that a block writes by its name is in the block's list of clobbers, and a
block that moves data between memories tells the compiler that memory changes."""
import re

import pytest

from helpers import ROOT

SOURCES = [p for p in sorted((ROOT / "minicpm-v-4.6-orangepi_amd" / "csrc").iterdir()) if p.suffix in (".hip", ".h")]
WRITTEN = re.compile(r"\b[sv]_\w+ +(m0|vcc|exec|scc)\b")


def blocks(text):
    """Every asm statement, from its name to the parenthesis that closes it."""
    for m in re.finditer(r"\basm\s+volatile\s*\(|\basm\s*\(", text):
        depth, end, quoted = 1, m.end(), False
        while depth:
            c = text[end]
            if c == '"' and text[end - 1] != "\\":
                quoted = not quoted
            if not quoted:
                depth += (c == "(") - (c == ")")
            end += 1
        yield text[m.start():end]


def missing(block):
    strings = re.findall(r'"((?:[^"\\]|\\.)*)"', block)
    code = strings[0].replace("\\n", "\n").replace("\\t", " ")
    want = {m.group(1) for m in WRITTEN.finditer(code)}
    if re.search(r"\b(buffer|global|flat|ds)_(load|store|read|write)\w*.*\blds\b", code):
        want.add("memory")
    return want - set(strings[1:])


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_written_registers_are_declared(path):
    for block in blocks(path.read_text()):
        assert not missing(block), block


def test_what_is_looked_for():
    assert missing('asm volatile("s_mov_b32 m0, %0\\n\\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(a), "v"(f(b, ")")))') == {"m0", "memory"}
    assert missing('asm volatile("s_mov_b32 m0, %0" ::"s"(a) : "m0")') == set()
    assert any("offen lds" in b for p in SOURCES for b in blocks(p.read_text()))
