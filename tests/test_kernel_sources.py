"""What the kernels' sources must say for the compiler to keep what they rely on."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "adambridge_amd" / "csrc"
FIXED = re.compile(r"\b(m0|vcc|exec|scc|s\d+|v\d+)\b")   # registers that an instruction names itself


def _assembly(text):
    """(template, clobbers) of each inline assembly."""
    for found in re.finditer(r"\basm\s*(?:volatile)?\s*\(", text):
        depth, end = 1, found.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[end], 0)
            end += 1
        body = text[found.end():end - 1]
        parts = re.split(r":(?=(?:[^\"]*\"[^\"]*\")*[^\"]*$)", body)   # colons outside strings
        yield parts[0], parts[3] if len(parts) > 3 else ""


@pytest.mark.parametrize("path", sorted(p for p in CSRC.iterdir() if p.suffix in (".hip", ".hpp", ".inc", ".cpp")), ids=lambda p: p.name)
def test_inline_assembly_names_the_registers_it_writes(path):
    """A first operand that is a register's own name is written: the compiler has to hear of it."""
    for template, clobbers in _assembly(path.read_text()):
        for line in re.sub(r'"\s*"', "", template).strip().strip('"').split("\\n"):
            operands = line.replace("\\t", " ").strip().split(None, 1)
            written = FIXED.match(operands[1].split(",")[0].strip()) if len(operands) == 2 else None
            if written and not operands[0].startswith(("s_nop", "s_waitcnt")):
                assert f'"{written[0]}"' in clobbers, (line, clobbers)
