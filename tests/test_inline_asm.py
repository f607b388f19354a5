"""What the kernels' inline assembly writes is declared to the compiler."""

from __future__ import annotations

import pathlib
import re

CSRC = pathlib.Path(__file__).resolve().parents[1] / "blackwell-switchyard_amd" / "csrc"


def statements(text: str):
    """Every asm statement of a source, to the parenthesis that closes it."""
    for m in re.finditer(r"\basm\s*(?:volatile\s*)?\(", text):
        depth, at, quoted = 1, m.end(), False
        while depth:
            c = text[at]
            if c == '"' and text[at - 1] != "\\":
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            at += 1
        yield text[m.start():at]


def test_special_registers_that_are_written_are_declared():
    """m0, vcc and exec: the compiler uses them itself, wherever it sees fit."""
    seen = 0
    for path in sorted(p for p in CSRC.iterdir() if p.suffix in (".hip", ".hpp", ".cpp")):
        for s in statements(path.read_text()):
            seen += 1
            for reg in ("m0", "vcc", "exec"):
                if re.search(rf"\bs_\w+ {reg}\b|\bv_cmp\w* {reg}\b", s):
                    assert s.count(f'"{reg}"') == 1, f"{path.name}: {s} writes {reg}"
    assert seen > 5
