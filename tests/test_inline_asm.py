"""Inline assembly of the kernels, read from their sources: copies from memory into LDS take their place from m0. An
instruction of its own must lie between the write of m0 and the copy (a required wait state of gfx9: without it the copy may
still take the old place), and the compiler puts none into inline assembly, nor does it know of a write of m0 in there."""
import pathlib
import re

import pytest

KERNELS = pathlib.Path(__file__).resolve().parent.parent / "inference_engine_rust_amd" / "csrc" / "kernels"
SOURCES = sorted(p for p in KERNELS.iterdir() if p.suffix in (".hip", ".cuh", ".h"))


def assemblies(path):
    """The inline assembly statements of a file, from asm to the semicolon behind its closing parenthesis."""
    return re.findall(r"\basm\b[^;]*?\((?:[^;\"]|\"[^\"]*\")*\);", path.read_text())


def faults(statement):
    text = "".join(re.findall(r'"([^"]*)"', statement.split(":")[0]))
    lines = [x.strip() for x in re.split(r"\\n(?:\\t)?", text) if x.strip()]
    bad = []
    for i, line in enumerate(lines):
        if re.match(r"s_\w+ m0\b", line):
            bad.append("writes m0 behind the compiler's back: " + line)
        if re.match(r"(global|buffer|scratch)_load_lds_", line):
            if '"{m0}"' not in statement:
                bad.append("m0 is not an operand: " + line)
            if i == 0 or not lines[i - 1].startswith("s_nop"):
                bad.append("no wait state before " + line)
    return bad


def test_the_check_finds_what_it_is_for():
    good = r'asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, off" ::"{m0}"(x), "v"(g));'
    old = r'asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" ::"s"(x), "v"(g));'
    assert faults(good) == [] and len(faults(old)) == 3
    assert len(faults(good.replace(r"s_nop 0\n\t", ""))) == 1


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_copies_into_lds(path):
    bad = [f for s in assemblies(path) for f in faults(s)]
    assert not bad, bad


def test_every_copy_is_seen():
    seen = sum(s.count("load_lds_dword") for p in SOURCES for s in assemblies(p))
    assert seen == sum(len(re.findall(r"^(?!\s*//).*_load_lds_dword", p.read_text(), re.M)) for p in SOURCES) > 0
