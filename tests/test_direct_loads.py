"""Loads from memory into LDS that are written as inline assembly: the hardware wants an instruction between the one that writes M0 (the LDS address) and the load that
reads it, and the compiler, which inserts it behind its own builtins, does not look into an assembly string.  The address is an operand in M0 itself, so that the compiler
knows what the register holds, and the string begins with the instruction between."""
import os
import re

from tilelang_ascend_amd import build

LOAD = re.compile(r"(global|buffer|scratch)_load_(lds_|.* lds\b)")


def too_near(text):
    """The statements of inline assembly in which a load into LDS follows a write of M0 at once, and how many such loads there are."""
    bad, loads = [], 0
    for literals in re.findall(r'asm(?:\s+volatile)?\s*\(\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', text):
        code = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', literals)).replace("\\t", "").replace("\\n", "\n")
        lines = [line.strip() for line in re.split(r"[\n;]", code) if line.strip()]
        for before, line in zip([""] + lines, lines):
            if LOAD.match(line):
                loads += 1
                # (the first of its string: the write may be the instruction ahead)
                if not before or re.match(r"s_\w+ m0\b", before):
                    bad.append(code)
    return bad, loads


def test_an_instruction_between_the_lds_address_and_its_load():
    loads = 0
    for name in sorted(os.listdir(build.CSRC_DIR)):
        if name.endswith((".hip", ".h", ".cpp")):
            with open(os.path.join(build.CSRC_DIR, name)) as f:
                bad, n = too_near(f.read())
            assert not bad, f"{name}: {bad}"
            loads += n
    assert loads >= 20, loads


def test_the_search_finds_them():
    assert too_near('asm volatile("s_mov_b32 m0, %0\\n\\tglobal_load_lds_dwordx4 %1, off" ::"s"(a));') == (["s_mov_b32 m0, %0\nglobal_load_lds_dwordx4 %1, off"], 1)
    assert too_near('asm volatile("s_mov_b32 m0, %0\\n\\ts_nop 0\\n\\t"\n "global_load_lds_dword %1, %2" ::"s"(a));') == ([], 1)
    assert too_near('asm volatile("s_nop 0\\n\\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(a), "v"(b));') == ([], 1)
    assert too_near('asm("global_load_lds_dword %0, off" ::"v"(a))')[0] and too_near('asm volatile("s_waitcnt vmcnt(0)" ::: "memory");') == ([], 0)
