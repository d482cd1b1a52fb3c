"""CPU: what the compiler cannot check in the kernels' inline assembly, and what it made of kernels that must not spill."""
import glob
import os
import re
import struct

import msgpack
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


# ---- the built kernels --------------------------------------------------------------------------------------------------------------
def kernels(path):
    """{mangled name: its entry in the code object's metadata} of every gfx950 kernel in a library"""
    with open(path, "rb") as f:
        data = f.read()
    out = {}
    for m in re.finditer(b"\x7fELF\x02\x01", data):
        at = m.start()
        if struct.unpack_from("<H", data, at + 18)[0] != 224:   # EM_AMDGPU
            continue
        phoff, = struct.unpack_from("<Q", data, at + 32)
        size, count = struct.unpack_from("<HH", data, at + 54)
        for i in range(count):
            kind, _, offset, _, _, length = struct.unpack_from("<IIQQQQ", data, at + phoff + i * size)
            if kind != 4:   # PT_NOTE
                continue
            p, end = at + offset, at + offset + length
            while p < end:
                name, desc, what = struct.unpack_from("<III", data, p)
                body = p + 12 + (name + 3) // 4 * 4
                if what == 32:   # NT_AMDGPU_METADATA
                    for k in msgpack.unpackb(data[body:body + desc])["amdhsa.kernels"]:
                        out[k[".name"]] = k
                p = body + (desc + 3) // 4 * 4
    return out


def test_sq8_filters_keep_their_registers():
    """a scan's loop that goes through scratch memory is a third slower; two registers outside of it are not felt"""
    found = {n: k for n, k in kernels(os.path.join(ROOT, "vectorsimilarity_amd", "libvsgpu.so")).items() if "k_mfma_filter_lowpILi4E" in n}
    assert len(found) >= 10
    assert {n: k[".vgpr_spill_count"] for n, k in found.items() if k[".vgpr_spill_count"] > 2} == {}
