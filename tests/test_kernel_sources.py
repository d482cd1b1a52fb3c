"""CPU: what the compiler cannot check in the kernels' inline assembly."""
import glob
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCES = sorted(p for folder in ("vectorsimilarity_amd/csrc", "tools") for kind in ("hip", "hpp", "h")
                 for p in glob.glob(os.path.join(ROOT, folder, "**", "*." + kind), recursive=True))


def statements(text):
    """every asm statement of a source, to the parenthesis that closes it (strings skipped)"""
    for m in re.finditer(r"\basm\s*(?:volatile)?\s*\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if quoted:
                if c == "\\":
                    i += 1
                elif c == '"':
                    quoted = False
            elif c == '"':
                quoted = True
            else:
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[m.start():i]


def test_the_scan_finds_statements():
    assert list(statements('asm volatile("s_mov_b32 m0, %0 ) \\" (" ::"s"(f(x)) : "memory"); asm("" : "+v"(a));')) == \
        ['asm volatile("s_mov_b32 m0, %0 ) \\" (" ::"s"(f(x)) : "memory")', 'asm("" : "+v"(a))']


@pytest.mark.parametrize("path", SOURCES, ids=[os.path.relpath(p, ROOT) for p in SOURCES])
def test_assembly_that_sets_m0_says_so(path):
    """m0 holds the LDS address of a direct load; the compiler may keep something of its own there"""
    with open(path) as f:
        text = f.read()
    for s in statements(text):
        if re.search(r"\bs_mov_b32\s+m0\b", s):
            assert re.search(r':[^:]*"m0"[^:]*\)$', s), s
