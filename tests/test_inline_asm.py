"""Inline assembly in the kernels' sources: a register that a statement writes by name is in its list of clobbers, or the compiler may
keep a value there across it."""
import glob
import os
import re

import pytest

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nn-cpp_amd", "src")
# the operand that an instruction of these writes first
WRITES = re.compile(r"(?:^|[\"\s]|\\n\\t)(?:s_|v_readfirstlane|v_readlane)\w+\s+(m0|vcc|exec|scc)\b")


def statements():
    """(file, line, text) of each asm statement."""
    for path in sorted(glob.glob(os.path.join(KERNELS, "**", "*.h*"), recursive=True)):
        text = open(path).read()
        for m in re.finditer(r"\basm\s+volatile\s*\(|\basm\s*\(", text):
            depth, at, quoted = 0, m.end() - 1, False
            while True:
                c = text[at]
                if c == '"' and text[at - 1] != "\\":
                    quoted = not quoted
                depth += 0 if quoted else (c == "(") - (c == ")")
                at += 1
                if depth == 0:
                    break
            yield os.path.relpath(path, KERNELS), text.count("\n", 0, m.start()) + 1, text[m.start():at]


def test_there_are_statements_to_check():
    assert sum("m0" in text for _, _, text in statements()) >= 3


@pytest.mark.parametrize("where", [(f, line, text) for f, line, text in statements()], ids=lambda w: f"{w[0]}:{w[1]}")
def test_named_registers_are_clobbers(where):
    text = where[2]
    clobbers = re.findall(r'"([\w]+)"', text.rsplit(":", 1)[1]) if text.count(":") >= 3 else []
    for name in set(WRITES.findall(text)):
        assert name in clobbers, (name, text)
    if re.search(r"\bs_add_u32\b", text):
        assert "scc" in clobbers, text
