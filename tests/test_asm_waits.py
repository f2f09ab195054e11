"""Wait states that inline assembly has to bring itself: on the CPU, from the sources.

A vector memory instruction that reads a scalar register needs five wait states after
a vector instruction that wrote it.  The compiler counts them for its own instructions,
not for those inside an asm statement, and may bring a base to its scalar registers by
v_readfirstlane (or v_readlane, from a spill) right before the statement.  A scalar
move may read it at once, and its result by a load too.  An m0 write needs one wait state
before a load into LDS."""
import glob
import os
import re

import pytest

from common import REPO

SOURCES = sorted(f for kind in ("*.hip", "*.h") for f in glob.glob(os.path.join(REPO, "llm.c_amd", "csrc", kind)))


def statements(text):
    """(instructions, the rest) of each asm statement."""
    text = re.sub(r"/\*.*?\*/|//[^\n]*", "", text, flags=re.S)
    for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
        depth, i = 1, m.end()
        while depth:
            if text[i] == '"':
                i = re.compile(r'"(?:\\.|[^"\\])*"').match(text, i).end()
                continue
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        body = text[m.end():i - 1]
        code = re.match(r'(?:\s*"(?:\\.|[^"\\])*")*', body).group(0)
        yield "".join(re.findall(r'"((?:\\.|[^"\\])*)"', code)), body[len(code):]


def test_statements_are_found():
    text = 'asm volatile("s_nop 4\\n\\t" "global_load_dword %0, %1" : : "v"(f(x)), "s"(b) : "memory"); asm("" : "+v"(x));'
    got = list(statements(text))
    assert [c for c, _ in got] == ["s_nop 4\\n\\tglobal_load_dword %0, %1", ""] and '"s"(b)' in got[0][1]


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_loads_from_scalar_bases_wait(path):
    for code, operands in statements(open(path).read()):
        parts = operands.split(":")  # "", outputs, inputs, ...
        outputs = re.findall(r'"([^"]*)"\s*\(', parts[1]) if len(parts) > 1 else []
        inputs = re.findall(r'"([^"]*)"\s*\(', ":".join(parts[2:]))
        waited = 0
        for line in re.split(r"\\n|;", code):
            line = line.replace("\\t", " ").strip()
            if re.match(r"(global|flat|buffer|scratch)_", line):
                read = [int(i) - len(outputs) for i in re.findall(r"%(\d+)", line)]
                if any(i >= 0 and "s" in inputs[i] for i in read):
                    assert waited >= 5, (os.path.basename(path), code)
                if "{m0}" in inputs:
                    assert waited >= 1, (os.path.basename(path), code)
            waited += int(line.split()[1]) + 1 if line.startswith("s_nop") else 1
