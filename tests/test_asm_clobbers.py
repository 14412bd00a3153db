"""Inline assembly names every register that it writes and is not an operand (sources only)."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "laprune_amd" / "csrc"
WRITTEN = ("m0", "vcc", "exec", "scc")


def _statements():
    for path in sorted(CSRC.iterdir()):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\((.*?)\)\s*;", text, re.S):
            yield path.name, m.group(1)


def test_written_registers_are_clobbered():
    seen = 0
    for name, body in _statements():
        strings = re.findall(r'"((?:[^"\\]|\\.)*)"', body)
        code = strings[0] if strings else ""
        for reg in WRITTEN:
            # the destination of an instruction: its first operand
            if re.search(rf"(?:^|\\n\\t|\\n)\s*[sv]_\w+\s+{reg}\b", code):
                seen += 1
                assert reg in strings[1:], f"{name}: asm writes {reg} and does not say so: {code}"
    assert seen >= 2
