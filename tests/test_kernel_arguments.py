"""Tables that travel in kernel arguments hold whole words.

Scalar loads drop the two lowest bits of their base and of their offset apart.  Where a table
of bytes stands beside one of addresses under the same index, the compiler may form one
element's address from the other's by adding 7 t to either of the two, and an address that is
then read by a scalar load is a wrong one for most t."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "tgengine_amd" / "csrc"
TEXT = "\n".join(re.sub(r"//[^\n]*", "", p.read_text()) for p in sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.hip")))
SMALL = re.compile(r"\b(?:u?int8_t|u?int16_t|unsigned char|signed char|char|bool|short|bf16|__bf16|half|_Float16|fp8)\b")


def _structs():
    """{name: body} of every struct with braces matched."""
    out = {}
    for m in re.finditer(r"\bstruct\s+(?:__attribute__\(\(.*?\)\)\s*)?(?:alignas\([^)]*\)\s*)?(\w+)\s*(?::[^{;]*)?\{", TEXT):
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(TEXT[i], 0)
            i += 1
        out[m[1]] = TEXT[m.end():i - 1]
    return out


def _by_value():
    """Names of the structs that kernels take by value."""
    structs, out = _structs(), set()
    for m in re.finditer(r"__global__[^;{]*?\bvoid\s+\w+\s*\(", TEXT):
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(TEXT[i], 0)
            i += 1
        for arg in TEXT[m.end():i - 1].split(","):
            out |= {w for w in re.findall(r"\w+", arg) if w in structs and "*" not in arg and "&" not in arg}
    return structs, out


def _arrays(structs, name):
    """(type, declarator) of the arrays in a struct and in the structs that it holds."""
    flat = re.sub(r"\{[^{}]*\}", ";", structs[name])
    for line in flat.split(";"):
        m = re.match(r"\s*(?:const\s+)?([\w:]+)\s*([^()=]*)$", line.strip(), re.S)
        if m is None:
            continue
        if "[" in m[2]:
            yield m[1], " ".join(m[2].split())
        if m[1] in structs and m[1] != name and "*" not in m[2]:
            yield from _arrays(structs, m[1])


def test_the_kernels_are_found():
    structs, names = _by_value()
    assert {"ClipList", "AdamList", "StepList", "ScanArgs", "ResArgs"} <= names
    assert {d for _, d in _arrays(structs, "AdamList")} >= {"* p[kList]", "size[kList]", "kind[kList]"}


@pytest.mark.parametrize("name", sorted(_by_value()[1]))
def test_tables_are_of_words(name):
    structs, _ = _by_value()
    small = [f"{t} {d}" for t, d in _arrays(structs, name) if SMALL.search(t) and "*" not in d]
    assert not small, small
