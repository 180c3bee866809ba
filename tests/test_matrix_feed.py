"""Assembly written in the sources: m0, which copies to LDS go by, is an operand.  The
compiler sets it by itself at any place of its own and ignores it in a list of clobbered
registers, so no statement may write it, and those that read it have to say so."""

import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "ns_fps_amd", "csrc")


def statements(text):
    """(instructions, operands) of every asm statement."""
    out = []
    for m in re.finditer(r"\basm\s+volatile\s*\(", text):
        depth, k = 1, m.end()
        while depth:
            c = text[k]
            if c == '"':
                k = text.index('"', k + 1)
            depth += (c == "(") - (c == ")")
            k += 1
        body = text[m.end():k - 1]
        # the instructions are the literals ahead of the first colon between literals
        code, rest, at = "", [], 0
        for s in re.finditer(r'"([^"]*)"', body):
            if not rest and ":" not in body[at:s.start()]:
                code += s.group(1)
            else:
                rest.append(s.group(1))
            at = s.end()
        out.append((code, rest))
    return out


def wrong(text):
    return [code for code, operands in statements(text)
            if re.search(r"\bs_\w+ m0\b", code) or ("_lds_" in code and "{m0}" not in operands)]


def test_the_check_sees_both():
    writes = 'asm volatile("s_mov_b32 m0, %0\\n\\ts_nop 4" : : "s"(f(a, b)) : "memory", "m0");'
    reads = 'asm volatile("s_nop 4\\n\\tglobal_load_lds_dwordx4 %0, %1" :: "v"(a), "s"(b) : "memory");'
    assert len(wrong(writes)) == len(wrong(reads)) == 1
    assert wrong(reads.replace('"s"(b)', '"s"(b), "{m0}"(c)')) == []
    assert wrong('asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");') == []


@pytest.mark.parametrize("name", sorted(os.listdir(CSRC)))
def test_copies_to_lds_name_the_register_that_they_go_by(name):
    with open(os.path.join(CSRC, name)) as f:
        assert wrong(f.read()) == []
