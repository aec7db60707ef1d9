"""Waits that the hardware does not make by itself, along every way through the built kernels of every source (isa_waits.py holds the rules for
matrix instructions).  An object file that is not there or not up to date is compiled for the test."""
import os
import re
import shutil
import subprocess

import pytest

from isa_waits import LLVM, functions, short_waits


def _code(source, folder):
    from sqd import lib
    src, obj = os.path.join(lib.CSRC, source + ".hip"), os.path.join(lib.OBJ_DIR, source + ".o")
    if not os.path.exists(LLVM):
        pytest.skip("no disassembler")
    if lib._stale(src, max(os.path.getmtime(h) for h in lib._headers())):
        hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
        if not os.path.exists(hipcc):
            pytest.skip("no object file of this source, and no compiler")
        obj = os.path.join(str(folder), source + ".o")
        subprocess.check_call([hipcc] + lib.compile_flags() + ["-c", src, "-o", obj])
    out = os.path.join(str(folder), "parts")
    os.makedirs(out)
    return functions(obj, out)


# sources with matrix instructions; a new one is noticed by the last test
MATRIX = ["attention", "attention_bwd", "bins", "conv", "sql", "vit"]


@pytest.mark.parametrize("source", MATRIX)
def test_results_of_matrix_instructions_are_waited_for(source, tmp_path):
    code = _code(source, tmp_path)
    assert any(line.lstrip().startswith("v_mfma") for c in code.values() for line in c)
    bad = {name: short_waits(c) for name, c in code.items()}
    assert not any(bad.values()), {name: b[:2] for name, b in bad.items() if b}


def test_the_token_kernel_waits_by_itself(tmp_path):
    """few rows: the product of the scores is followed by a wait of its own, as long as the product's type needs (the compiler's count is not relied on)"""
    code = {n: c for n, c in _code("attention", tmp_path).items() if "attn_token_kernel" in n}
    assert len(code) > 20
    for name, c in code.items():
        nops = [sum(int(x, 0) + 1 for x in m) for m in (re.findall(r"s_nop (\d+)", "\n".join(c[i:i + 2])) for i in range(len(c)))]
        assert max(nops) >= (18 if "_kernelIf" in name else 12), (name, max(nops))


def test_every_source_with_matrix_instructions_is_looked_at():
    from sqd import lib
    found = set()
    for src in lib.sources():
        with open(src) as f:
            text = f.read()
        if "mfma" in text or "Mma<" in text:
            found.add(os.path.basename(src)[:-4])
    assert found == set(MATRIX)
