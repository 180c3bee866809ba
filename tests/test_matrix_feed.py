"""Assembly written in the sources: registers that it sets by name are named as such,
so that the compiler keeps nothing of its own there across it."""

import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "ns_fps_amd", "csrc")


def statements(text):
    """(instructions, clobbers) of every asm statement."""
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
        strings = list(re.finditer(r'"([^"]*)"', body))
        # the instructions are the literals ahead of the first colon between literals
        parts, at = [[]], 0
        for s in strings:
            parts += [[] for _ in range(body[at:s.start()].count(":"))]
            parts[-1].append(s.group(1))
            at = s.end()
        out.append(("".join(parts[0]), parts[3] if len(parts) > 3 else []))
    return out


def unnamed(text):
    return [code for code, clobbers in statements(text)
            if re.search(r"\bs_mov_b32 m0\b", code) and "m0" not in clobbers]


def test_the_check_sees_both():
    bad = 'asm volatile("s_mov_b32 m0, %0\\n\\ts_nop 4" : : "s"(f(a, b)) : "memory");'
    assert len(unnamed(bad)) == 1 and unnamed(bad.replace('"memory"', '"memory", "m0"')) == []
    assert unnamed('asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");') == []


@pytest.mark.parametrize("name", sorted(os.listdir(CSRC)))
def test_registers_that_assembly_sets_are_named(name):
    with open(os.path.join(CSRC, name)) as f:
        assert unnamed(f.read()) == []
