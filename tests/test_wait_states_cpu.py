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


NEEDED = 11  # issue slots from an MFMA of eight passes (32x32x16 of 16 bits) to a read of what it wrote
FAR = 40


def slots(lines):
    """The fewest issue slots, on any way through the code, from an MFMA to a v_max3_f32 that reads what it wrote, of those
    that no instruction of the compiler's own has read or written in between; and whether settle's wait is in each."""
    code, at = [], {}
    for line in lines:
        text, _, where = line.partition("//")
        op = text.split(None, 1)
        if op and not op[0].endswith(":"):
            if where:
                at[int(where.split(":")[0], 16)] = len(code)
            code.append((op[0], op[1].split(",") if len(op) > 1 else [], int(where.split(":")[0], 16) if where else None))
    seen, fewest, settled, todo = [None] * len(code), FAR, True, [(0, {})]
    while todo:
        i, fresh = todo.pop()
        while i < len(code):
            if seen[i] is not None and all(seen[i].get(r, FAR) <= n for r, n in fresh.items()):
                break
            old = seen[i] or {}
            fresh = {r: min(old.get(r, FAR), fresh.get(r, FAR)) for r in old.keys() | fresh.keys()}
            seen[i] = dict(fresh)
            op, args, where = code[i]
            if op == "v_max3_f32":
                near = [fresh[r] for x in args[1:] for r in registers(x) if r in fresh]
                fewest = min([fewest] + near)
                settled = settled and not near
            if op == "s_nop" and args[0].strip() == "15":
                fresh = {}
            elif op.startswith(("v_", "ds_", "global_")) and not op.startswith("v_mfma"):
                for x in args:
                    for r in registers(x):
                        fresh.pop(r, None)
            more = int(args[0]) + 1 if op == "s_nop" else 1
            fresh = {r: min(n + more, FAR) for r, n in fresh.items()}
            if op.startswith("v_mfma"):
                fresh.update((r, 0) for r in registers(args[0]))
            if op == "s_endpgm":
                break
            if op.startswith(("s_branch", "s_cbranch")):
                to = int(args[0].split()[0])
                todo.append((at[where + 4 + 4 * (to - 65536 if to > 32767 else to)], dict(fresh)))
                if op == "s_branch":
                    break
            i += 1
    return fewest, settled


def test_what_counts():
    mfma, top = "v_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], 0", "v_max3_f32 v30, v40, v1, v2"
    assert slots([mfma, "s_barrier", top]) == (1, False)
    assert slots([mfma, "s_nop 3", "s_barrier", top]) == (5, False)
    assert slots([mfma, "s_nop 15", "s_nop 2", top]) == slots([top, mfma]) == (FAR, True)
    assert slots([mfma, "v_max3_f32 v30, v16, v17, s0"]) == (FAR, True)
    assert slots([mfma, "v_cndmask_b32_e32 v1, v2, v6, vcc", "v_max3_f32 v30, v40, v1, v2"]) == (FAR, True)
    loop = [f"v_max3_f32 v30, v40, v1, v2 // {0:012X}: 0", f"{mfma} // {8:012X}: 0", f"s_cbranch_scc1 65531 // {16:012X}: 0"]
    assert slots(loop + ["s_endpgm"]) == (1, False)


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="needs the ROCm toolchain")
def test_maxima_of_products_wait(tmp_path):
    """Kernels whose scores reach a maximum in asm without an instruction of the compiler's own on the way: the tree's and
    the prefix's have settle's wait; the forward's, which work a phase apart, slots enough between the phases."""
    os.symlink(L.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    tree = forward = 0
    for obj in glob.glob(str(tmp_path / "lib.so.*gfx950")):
        with open(obj, "rb") as f:
            held = f.read()
            if not any(name in held for name in (b"tree_attn_kernel", b"fwd_mfma_kernel", b"fwd_ws_kernel")):
                continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", obj], check=True,
                              capture_output=True, text=True).stdout
        for block in text.split("\n\n"):
            name = block.strip().split("\n")[0]
            # <T, D, waves, sharing, CAP, PRE> and <T, D, CAP>
            if ("tree_attn_kernel" in name and "ELb0ELb" in name) or ("prefix_wide_kernel" in name and "ELb0E" in name):
                assert "v_mfma" in block and slots(block.split("\n")[1:])[1], name
                tree += 1
            elif "fwd_mfma_kernel" in name or "fwd_ws_kernel" in name:
                assert "v_mfma" in block and slots(block.split("\n")[1:])[0] >= NEEDED, name
                forward += 1
    assert tree > 20 and forward > 20
