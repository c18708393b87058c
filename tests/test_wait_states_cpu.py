"""The built code of the tree and prefix attention: a maximum taken in asm of an MFMA's results stands behind the wait that
such results need (settle in flexatt_device.h).  The compiler keeps none in front of asm, so without the wait it is up to
what instructions happen to be between."""
import glob
import os
import re
import shutil
import subprocess

import pytest

import flexatt_lib as L

ROCM = os.path.dirname(os.path.dirname(os.path.realpath(shutil.which("hipcc") or "/opt/rocm/bin/hipcc")))
OBJDUMP = os.path.join(ROCM, "llvm", "bin", "llvm-objdump")


def registers(operand):
    """v5, v[0:15] -> their numbers."""
    m = re.fullmatch(r"v(\d+)|v\[(\d+):(\d+)\]", operand.strip(" ,"))
    if not m:
        return set()
    return {int(m[1])} if m[1] else set(range(int(m[2]), int(m[3]) + 1))


def step(op, args, fresh):
    """What is fresh behind an instruction: written by an MFMA, and neither waited for nor read by the compiler's code."""
    if op == "s_nop" and args[0].strip() == "15":
        return frozenset()
    if op.startswith("v_mfma"):
        return fresh | registers(args[0])
    if op.startswith(("v_", "ds_", "global_")):
        return fresh.difference(*(registers(x) for x in args))
    return fresh


def unsettled(lines):
    """v_max3_f32 that, on some way through the code, read what an MFMA wrote without the longest s_nop between them."""
    code, at = [], {}
    for line in lines:
        text, _, where = line.partition("//")
        op = text.split(None, 1)
        if op and not op[0].endswith(":"):
            if where:
                at[int(where.split(":")[0], 16)] = len(code)
            code.append((op[0], op[1].split(",") if len(op) > 1 else [], int(where.split(":")[0], 16) if where else None))
    seen, bad, todo = [None] * len(code), set(), [(0, frozenset())]
    while todo:
        i, fresh = todo.pop()
        while i < len(code):
            if seen[i] is not None and fresh <= seen[i]:
                break
            fresh = seen[i] = fresh | (seen[i] or frozenset())
            op, args, where = code[i]
            if op == "v_max3_f32" and any(registers(x) & fresh for x in args[1:]):
                bad.add(f"{op} {','.join(args)}".strip())
            fresh = step(op, args, fresh)
            if op == "s_endpgm":
                break
            if op.startswith(("s_branch", "s_cbranch")):
                to = int(args[0].split()[0])
                todo.append((at[where + 4 + 4 * (to - 65536 if to > 32767 else to)], fresh))
                if op == "s_branch":
                    break
            i += 1
    return sorted(bad)


def test_what_counts_as_unsettled():
    mfma, top = "v_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], 0", "v_max3_f32 v30, v40, v1, v2"
    assert unsettled([mfma, "s_barrier", top]) == [top]
    assert unsettled([mfma, "s_nop 15", "s_nop 2", top]) == [] == unsettled([top, mfma])
    assert unsettled([mfma, "v_max3_f32 v30, v16, v17, s0"]) == []
    assert unsettled([mfma, "v_cndmask_b32_e32 v1, v5, v6, vcc", "v_max3_f32 v30, v40, v1, v1"]) == []


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="needs the ROCm toolchain")
def test_maxima_of_products_wait(tmp_path):
    """Kernels without a soft-cap; with one the scores pass through instructions of the compiler's own."""
    os.symlink(L.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    looked = 0
    for obj in glob.glob(str(tmp_path / "lib.so.*gfx950")):
        with open(obj, "rb") as f:
            if b"tree_attn_kernel" not in f.read():
                continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", obj], check=True,
                              capture_output=True, text=True).stdout
        for block in text.split("\n\n"):
            name = block.strip().split("\n")[0]
            # <T, D, waves, sharing, CAP, PRE> and <T, D, CAP>
            if ("tree_attn_kernel" in name and "ELb0ELb" in name) or ("prefix_wide_kernel" in name and "ELb0E" in name):
                assert "v_mfma" in block, name
                assert unsettled(block.split("\n")[1:]) == [], name
                looked += 1
    assert looked > 20
