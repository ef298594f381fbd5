"""Instructions written by hand say which registers they change beyond their operands: what the compiler does not know of, it may keep a value in."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "arboretum_amd", "csrc")
SCALAR_ARITHMETIC = re.compile(r"\bs_(add|sub|addc|subb|and|or|xor|andn2|orn2|lshl|lshr|ashr|bfe|min|max|not|abs|cmp)\w*_[iub]\d+")


def statements(text):
    """The operands of every asm statement: what stands between its parentheses."""
    for start in re.finditer(r"\basm(?:\s+volatile)?\s*\(", text):
        depth, quoted, at = 1, False, start.end()
        while depth:
            c = text[at]
            if c == "\\":
                at += 1
            elif c == '"':
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            at += 1
        yield text[start.end():at - 1]


def parts(statement):
    """(instructions, clobbers): the strings before the first colon, and those behind the third"""
    fields, quoted, now = [], False, ""
    for c in statement:
        quoted ^= c == '"'
        if c == ":" and not quoted:
            fields.append(now)
            now = ""
        else:
            now += c
    fields.append(now)
    strings = lambda s: re.findall(r'"((?:[^"\\]|\\.)*)"', s)  # noqa: E731
    return "\n".join(strings(fields[0])).replace("\\n", "\n").replace("\\t", " "), strings(fields[3]) if len(fields) > 3 else []


def test_the_reader_of_statements():
    one = r'asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" ::"s"(f(x)) : "m0", "memory");'
    assert [parts(s) for s in statements(one)] == [("s_mov_b32 m0, %0\n s_nop 0", ["m0", "memory"])]
    assert [parts(s) for s in statements('asm("" : "+v"(a)); asm volatile("s_nop 4" : "+s"(b));')] == [("", []), ("s_nop 4", [])]


@pytest.mark.parametrize("name", sorted(f for f in os.listdir(CSRC) if f.endswith((".h", ".hip", ".cpp"))))
def test_registers_that_statements_change_are_named(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    for statement in statements(text):
        instructions, clobbers = parts(statement)
        for line in instructions.splitlines():
            words = line.replace(",", " ").split()
            if len(words) > 1 and words[1] == "m0":
                assert "m0" in clobbers, line
            if SCALAR_ARITHMETIC.match(words[0] if words else ""):
                assert "scc" in clobbers, line
