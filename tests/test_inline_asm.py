"""What the compiler has to be told about the inline assembly in csrc, read
from the sources (no GPU).  Global -> LDS copies set m0 by themselves: a
statement that does not name it lets the compiler keep a value of its own
there across the copy."""
import glob
import os
import re

import pytest

from conftest import PKG

SOURCES = sorted(glob.glob(os.path.join(PKG, "csrc", "*.h*")))


def statements(text):
    """(instructions, constraints) of every asm statement."""
    for m in re.finditer(r"\basm\s+volatile\s*\(", text):
        depth, quoted, i = 1, False, m.end()
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != "\\":
                quoted = not quoted
            depth += 0 if quoted else (c == "(") - (c == ")")
            i += 1
        body = text[m.end():i - 1]
        code = re.match(r'(?:\s*"(?:\\.|[^"\\])*")+', body).group()
        lines = "".join(re.findall(r'"((?:\\.|[^"\\])*)"', code))
        yield re.split(r"(?:\\n|\\t|;)+", lines), body[len(code):]


def test_reads_statements():
    got = list(statements('asm volatile("s_mov_b32 m0, %1\\n\\ts_nop 0" "\\n\\tx (%0)" ::"v"(f(g)),'
                          ' "s"(l) : "memory", "m0");  asm volatile("" ::: "memory");'))
    assert got[0][0] == ["s_mov_b32 m0, %1", "s_nop 0", "x (%0)"] and '"m0"' in got[0][1]
    assert got[1][0] == [""] and len(got) == 2


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_m0_is_named(path):
    for code, rest in statements(open(path).read()):
        if any(re.match(r"s_mov_b32 m0\b", line) for line in code):
            assert '"m0"' in rest, code


def test_finds_the_copies():
    n = sum("lds" in line for p in SOURCES for code, _ in statements(open(p).read())
            for line in code)
    assert n >= 8


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_a_base_from_a_vector_instruction_can_be_read(path):
    """A memory instruction may read a scalar register that a vector
    instruction wrote (readfirstlane, or readlane of a spilled one) only five
    wait states later; inside asm the compiler does not see the reader and
    counts none of them."""
    for code, _ in statements(open(path).read()):
        states = 0
        for line in code:
            if m := re.match(r"(global|buffer|scratch)_\w+\s+(.*)", line):
                vector_only = re.fullmatch(r"%\d+, off", m.group(2))
                assert vector_only or states >= 5, code
            nop = re.match(r"s_nop (\d+)", line)
            states += int(nop.group(1)) + 1 if nop else 1
