"""The wait from a matrix instruction to the first other use of its result, along the shortest way through the built kernels.

The hardware does not hold an instruction back that reads such a result early: the compiler has to keep 12 states (32x32x16, 8 passes) or 8 (16x16x32,
4 passes) between them in 16 bits, 18 and 10 in fp32 (32x32x2, 16x16x4).  Where two ways lead to the use it has been seen to count the longer one."""
import os
import re
import subprocess

LLVM = "/opt/rocm/llvm/bin/llvm-objdump"
STATES = {"32x32x2_f32": 18, "16x16x4_f32": 10, "32x32x16_bf16": 12, "32x32x16_f16": 12, "16x16x32_bf16": 8, "16x16x32_f16": 8}
_REG = re.compile(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(text):
    out = set()
    for m in _REG.finditer(text):
        first, last = (m.group(2), m.group(3)) if m.group(2) else (m.group(4), m.group(4))
        out.update((m.group(1), i) for i in range(int(first), int(last) + 1))
    return out


def states_of(op):
    for shape, n in STATES.items():
        if shape in op:
            return n
    return 20                                              # 16 passes in 16 bits, and any form not listed


def short_waits(code):
    """code: lines of one function ("label:" or an instruction) -> [(states, wanted, matrix instruction, use)]"""
    ins, label = [], {}
    for line in code:
        line = line.strip()
        if line.endswith(":"):
            label[line[:-1]] = len(ins)
        elif line:
            op, _, rest = line.partition(" ")
            ins.append((op, rest.strip()))
    found = []
    for i, (op, rest) in enumerate(ins):
        if not op.startswith("v_mfma"):
            continue
        dst, want, best, ways = registers(rest.split(",")[0]), states_of(op), {}, [(i + 1, 0)]
        while ways:
            j, n = ways.pop()
            while j < len(ins) and n < want and n < best.get(j, want):
                best[j] = n
                o, r = ins[j]
                if o.startswith("v_mfma"):
                    args = re.split(r",(?![^\[]*\])", r)
                    if registers(args[1] + " " + args[2]) & dst:
                        found.append((n, want, op + " " + rest, o + " " + r))
                        break
                    if registers(args[0]) & dst:           # a chain of products into one accumulator has no wait
                        break
                elif not o.startswith("s_") and registers(r) & dst:
                    found.append((n, want, op + " " + rest, o + " " + r))
                    break
                if o in ("s_endpgm", "s_setpc_b64"):
                    break
                n += int(r, 0) + 1 if o == "s_nop" else 1
                if o == "s_branch":
                    j = label[r]
                    continue
                if o.startswith("s_cbranch"):
                    ways.append((label[r], n))
                j += 1
    return found


def functions(obj, folder):
    """name -> lines of code of every gfx950 function in the object file `obj`; folder: for what is taken out of it"""
    name = os.path.join(folder, os.path.basename(obj))
    with open(obj, "rb") as a, open(name, "wb") as b:
        b.write(a.read())
    subprocess.run([LLVM, "--offloading", name], check=True, capture_output=True, cwd=folder)
    out, cur = {}, None
    for part in sorted(os.listdir(folder)):
        if part.startswith(os.path.basename(obj)) and "gfx950" in part:
            text = subprocess.run([LLVM, "-d", "--no-show-raw-insn", "--no-leading-addr", "--symbolize-operands", os.path.join(folder, part)], check=True,
                                  capture_output=True, text=True).stdout
            for line in text.splitlines():
                line = line.split("//")[0].rstrip()
                m = re.match(r"<(\w+)>:$", line)
                if m and not re.match(r"L\d+$", m.group(1)):
                    cur = out.setdefault(m.group(1), [])
                elif cur is not None and line:
                    cur.append(m.group(1) + ":" if m else line)
    return out
