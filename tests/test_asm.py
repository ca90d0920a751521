"""Inline assembly in csrc names the registers that it writes by itself."""

import pathlib
import re

CSRC = pathlib.Path(__file__).resolve().parent.parent / "torchsplinekan_amd" / "csrc"


def _statements(text):
    """Every asm statement, from its keyword to the closing parenthesis."""
    for m in re.finditer(r"\basm\s+volatile\s*\(", text):
        depth, i = 1, m.end()
        while depth:
            if text[i] == '"':
                i = text.index('"', i + 1)
            else:
                depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        yield text[m.start():i]


def test_asm_that_writes_m0_says_so():
    seen = 0
    for path in sorted(CSRC.iterdir()):
        for s in _statements(path.read_text()):
            if re.search(r"s_mov_b32 m0\b", s):
                seen += 1
                assert re.search(r':\s*"m0"\s*\)$', s), f"{path.name}: {s}"
    assert seen == 1
