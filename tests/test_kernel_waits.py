"""Waits that the hardware does not make by itself, along every way through the built kernels of every source (isa_waits.py holds the rules for
matrix instructions).  An object file that is not there or not up to date is compiled for the test."""
import functools
import os
import re
import shutil
import subprocess
import tempfile

import pytest

from isa_waits import LLVM, functions, short_waits


@functools.lru_cache(None)
def _code(source):
    from sqd import lib
    src, obj = os.path.join(lib.CSRC, source + ".hip"), os.path.join(lib.OBJ_DIR, source + ".o")
    if not os.path.exists(LLVM):
        pytest.skip("no disassembler")
    with tempfile.TemporaryDirectory() as folder:
        if lib._stale(src, max(os.path.getmtime(h) for h in lib._headers())):
            hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
            if not os.path.exists(hipcc):
                pytest.skip("no object file of this source, and no compiler")
            obj = os.path.join(folder, source + ".o")
            subprocess.check_call([hipcc] + lib.compile_flags() + ["-c", src, "-o", obj])
        out = os.path.join(folder, "parts")
        os.makedirs(out)
        return functions(obj, out)


# sources with matrix instructions; a new one is noticed by the last test
MATRIX = ["attention", "attention_bwd", "bins", "conv", "sql", "vit"]


@pytest.mark.parametrize("source", MATRIX)
def test_results_of_matrix_instructions_are_waited_for(source):
    code = _code(source)
    assert any(line.lstrip().startswith("v_mfma") for c in code.values() for line in c)
    bad = {name: short_waits(c) for name, c in code.items()}
    assert not any(bad.values()), {name: b[:2] for name, b in bad.items() if b}


def test_the_token_kernel_waits_by_itself():
    """few rows: the product of the scores is followed by a wait of its own, as long as the product's type needs (the compiler's count is not relied on)"""
    code = {n: c for n, c in _code("attention").items() if "attn_token_kernel" in n}
    assert len(code) > 20
    for name, c in code.items():
        nops = [sum(int(x, 0) + 1 for x in m) for m in (re.findall(r"s_nop (\d+)", "\n".join(c[i:i + 2])) for i in range(len(c)))]
        assert max(nops) >= (18 if "_kernelIf" in name else 12), (name, max(nops))


_SCALAR = re.compile(r"\bs(?:\[(\d+):(\d+)\]|(\d+)\b)")


def _scalars(text):
    out = set()
    for m in _SCALAR.finditer(text):
        first, last = (m.group(1), m.group(2)) if m.group(1) else (m.group(3), m.group(3))
        out.update(range(int(first), int(last) + 1))
    return out | ({"vcc"} if "vcc" in text else set())


def _instructions(code):
    ins, label = [], {}
    for line in code:
        line = line.strip()
        if line.endswith(":"):
            label[line[:-1]] = len(ins)
        elif line:
            op, _, rest = line.partition(" ")
            ins.append((op, rest.strip()))
    return ins, label


def short_bases(code):
    """a scalar register written by a vector instruction and read as the address of a memory access within five states, on any way"""
    (ins, label), found = _instructions(code), []
    for i, (op, rest) in enumerate(ins):
        dst = _scalars(rest.split(",")[0]) if op.startswith("v_") else set()
        ways, seen = [(i + 1, 0)] if dst else [], set()
        while ways:
            j, n = ways.pop()
            while j < len(ins) and n < 5 and (j, n) not in seen:
                seen.add((j, n))
                o, r = ins[j]
                if o.startswith(("global_", "buffer_", "flat_")) and _scalars(r) & dst:
                    found.append((n, op + " " + rest, o + " " + r))
                    break
                n += int(r, 0) + 1 if o == "s_nop" else 1
                if o in ("s_endpgm", "s_setpc_b64"):
                    break
                if o == "s_branch":
                    j = label[r]
                    continue
                if o.startswith("s_cbranch"):
                    ways.append((label[r], n))
                j += 1
    return found


def test_base_counter():
    write, load = "v_readfirstlane_b32 s4, v1", "global_load_lds_dwordx4 v2, s[4:5]"
    assert short_bases([write, "s_mov_b32 m0, s9", "s_nop 0", load]) and not short_bases([write, "s_nop 3", "s_mov_b32 m0, s9", load])
    assert short_bases([write, "s_cbranch_scc1 L1", "s_nop 4", "L1:", load]) and not short_bases([write, "s_nop 0", "global_load_dword v2, v3, s[6:7]"])


@pytest.mark.parametrize("source", ["attention", "attention_bwd"])
def test_bases_of_loads_in_assembly_are_waited_for(source):
    bad = {name: short_bases(c) for name, c in _code(source).items()}
    assert len(bad) > 50 and not any(bad.values()), {name: b[:2] for name, b in bad.items() if b}


@pytest.mark.parametrize("source", ["attention", "attention_bwd"])
def test_no_wave_meets_others_with_reads_under_way(source):
    """behind a barrier another wave overwrites what this one was reading: every read of LDS has come back before it, on every way"""
    for name, c in _code(source).items():
        ins, label = _instructions(c)
        seen, ways = set(), [i + 1 for i, (op, _) in enumerate(ins) if op.startswith("ds_read")]
        while ways:
            j = ways.pop()
            while j < len(ins) and j not in seen:
                seen.add(j)
                o, r = ins[j]
                assert o != "s_barrier", (name, j)
                if "lgkmcnt(0)" in r or o in ("s_endpgm", "s_setpc_b64"):
                    break
                if o.startswith("s_cbranch"):
                    ways.append(label[r])
                j = label[r] if o == "s_branch" else j + 1


def test_no_gradient_kernel_is_built_that_no_call_reaches():
    """16-bit types past 64 features: 128 keys by 64 rows in 8 waves, or 64 keys by 64 rows"""
    names = [n for n in _code("attention_bwd") if "attn_dkv_kernel" in n]
    assert any(re.search("bf16_tELi128ELi4ELi2", n) for n in names) and not any(re.search("f16_tELi128ELi4ELi1", n) for n in names)


def test_assembly_that_writes_m0_says_so():
    """the compiler keeps values of its own there"""
    from sqd import lib
    n = 0
    for src in lib.sources() + lib._headers():
        with open(src) as f:
            for block in re.findall(r"asm volatile\(.*?\);", f.read(), re.S):
                if re.search(r"\bm0,", block):
                    n += 1
                    assert '"m0")' in block, (src, block)
    assert n


def test_every_source_with_matrix_instructions_is_looked_at():
    from sqd import lib
    found = set()
    for src in lib.sources():
        with open(src) as f:
            text = f.read()
        if "mfma" in text or "Mma<" in text:
            found.add(os.path.basename(src)[:-4])
    assert found == set(MATRIX)
