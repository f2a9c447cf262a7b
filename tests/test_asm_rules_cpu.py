"""What inline assembly in the kernels may do.  The compiler takes an asm statement's outputs as written once it has been issued and does not see what it reads later:
a load whose wait stands in another statement leaves a register that may be copied, spilled or given away while the load is in flight; a store written in asm may
read a register after it has been overwritten, or a matrix product before it is there.  So: no loads into registers without their wait in the same statement, no
stores, no matrix instructions, and M0 named as clobbered where it is written."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alphazero-connect6_amd", "csrc")
SOURCES = sorted(f for e in ("*.hip", "*.h", "*.inc", "*.cpp") for f in glob.glob(os.path.join(CSRC, e)))
LOAD = re.compile(r"\b(global|flat|buffer|scratch)_load_\w+|\bds_read\w*|\bds_load\w*|\bs_load_\w+|\bs_buffer_load_\w+")
STORE = re.compile(r"\b(global|flat|buffer|scratch)_(store|atomic)_\w+|\bds_write\w*|\bds_store\w*")


def statements(path):
    """(line, text of the instructions, the whole statement) of every asm statement outside comments"""
    src = re.sub(r"/\*.*?\*/", lambda m: re.sub(r"[^\n]", " ", m.group()), open(path).read(), flags=re.S)
    src = re.sub(r'("(?:\\.|[^"\\])*")|//[^\n]*', lambda m: m.group(1) or "", src)
    for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", src):
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(src[i], 0) if not in_string(src, m.end(), i) else 0
            i += 1
        whole = src[m.end():i - 1]
        code = "".join(re.findall(r'"((?:\\.|[^"\\])*)"', re.split(r'(?<=")\s*:', whole)[0])).replace("\\n", "\n").replace("\\t", " ")
        yield src.count("\n", 0, m.start()) + 1, code, whole


def in_string(src, start, i):
    return len(re.findall(r'(?<!\\)"', src[start:i])) % 2 == 1


def faults(code, whole):
    out = []
    lines = [x for x in code.split("\n") if x.strip()]
    for k, x in enumerate(lines):
        m = LOAD.search(x)
        if m and "_lds" not in m.group():
            counter = "lgkmcnt(0)" if m.group().startswith(("ds_", "s_")) else "vmcnt(0)"
            if not any(counter in y for y in lines[k + 1:]):
                out.append("a load whose wait is not in the statement: " + x.strip())
        if STORE.search(x):
            out.append("a store: " + x.strip())
        if "mfma" in x:
            out.append("a matrix instruction, whose wait states nobody counts: " + x.strip())
    if re.search(r"\bs_mov_b32 m0\b", code) and '"m0"' not in whole:
        out.append("M0 is written and not named as clobbered")
    return out


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_inline_assembly(path):
    bad = [(line, f) for line, code, whole in statements(path) for f in faults(code, whole)]
    assert not bad, bad


def test_the_rules_see_what_they_are_for():
    bad = ['asm volatile("global_load_dwordx4 %0, %1, %2" : "=v"(d) : "v"(o), "s"(b) : "memory")',
           'asm volatile("global_store_dwordx4 %0, %1, %2 offset:" #imm "\\n\\ts_nop 1" ::"v"(o), "v"(d), "s"(b) : "memory")',
           'asm volatile("s_mov_b32 m0, %2\\n\\ts_nop 0\\n\\tglobal_load_lds_dwordx4 %0, %1" ::"v"(l), "s"(g), "s"(o) : "memory")',
           'asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+v"(ACC) : "v"(A), "v"(B))']
    good = ['asm volatile("global_load_dwordx4 %0, %1, %2\\n\\ts_waitcnt vmcnt(0)" : "=&v"(d) : "v"(o), "s"(b) : "memory")',
            'asm volatile("s_mov_b32 m0, %2\\n\\ts_nop 0\\n\\tglobal_load_lds_dwordx4 %0, %1" ::"v"(l), "s"(g), "s"(o) : "memory", "m0")',
            'asm volatile("" : "+v"(d))']
    for text, want in [(t, 1) for t in bad] + [(t, 0) for t in good]:
        whole = text[text.index("(") + 1:-1]
        code = "".join(re.findall(r'"((?:\\.|[^"\\])*)"', re.split(r'(?<=")\s*:', whole)[0])).replace("\\n", "\n").replace("\\t", " ")
        assert len(faults(code, whole)) == want, (text, faults(code, whole))


def test_statements_are_found():
    assert sum(1 for p in SOURCES for _ in statements(p)) > 15
