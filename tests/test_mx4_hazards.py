"""CPU check of the MXFP4 product's assembly, as this compiler makes it.

csrc/mx4_gemm.hip writes its matrix instructions and its loads to LDS as inline
assembly, of which the compiler knows no latency, so two distances rest on its
schedule: two wait states between a vector instruction that writes an operand of a
matrix instruction and the latter, and five between a vector instruction that
writes a scalar register and a load that takes its descriptor or offset from it.
Both are measured here over the instructions in order."""
import os
import re
import shutil
import subprocess

import pytest

DIR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sushiblas_amd")
WINDOW = 8


def _registers(arg):
    m = re.fullmatch(r"([vas])\[(\d+):(\d+)\]", arg)
    if m:
        return {m[1] + str(i) for i in range(int(m[2]), int(m[3]) + 1)}
    return {arg} if re.fullmatch(r"[vas]\d+", arg) else {"vcc"} if arg.startswith("vcc") else set()


def near(assembly):
    """(matrix instructions, loads to LDS, descriptions of distances that are too short)."""
    products = loads = 0
    bad, past = [], []  # past: (what a vector instruction wrote, wait states it takes, text)
    for line in assembly.split("\n"):
        line = line.split(";")[0].strip()
        if not line or line[0] in ".#" or line.endswith(":"):
            continue
        op, _, rest = line.partition(" ")
        args = [a.strip().split(" ")[0] for a in rest.split(",")]
        product, load = op.startswith("v_mfma"), op.startswith("buffer_load") and " lds" in line
        products, loads = products + product, loads + load
        if product or load:
            uses, need = set().union(*[_registers(a) for a in args[1:]]), 2 if product else 5
            if load:
                uses = {r for r in uses if r[0] == "s"}
            between = 0
            for wrote, takes, text in reversed(past):
                if wrote & uses and between < need:
                    bad.append(f"{between} between: {text} -> {line}")
                between += takes
        vector = op.startswith("v_") and not product
        # (a swap writes both of its registers)
        wrote = set().union(*[_registers(a) for a in args[:2 if "swap" in op else 1]]) if vector else set()
        past = (past + [(wrote, int(args[0], 0) + 1 if op == "s_nop" else 1, line)])[-WINDOW:]
    return products, loads, bad


def test_the_check_itself():
    mma = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[4:7], v[8:11], a[0:3], v12, v13"
    assert near(f"v_mov_b32_e32 v9, v1\n{mma}")[2]
    assert near(f"v_accvgpr_write_b32 a2, 0\ns_nop 0\n{mma}")[2]
    assert near(f"v_mov_b32_e32 v12, v1\nds_read_b128 v[20:23], v1\ns_mov_b32 s0, s1\n{mma}") == (1, 0, [])
    assert near(f"v_mov_b32_e32 v9, v1\ns_nop 1\n{mma}") == (1, 0, [])
    load = "buffer_load_dwordx4 v1, s[4:7], s8 offen lds"
    assert near(f"v_readfirstlane_b32 s6, v1\ns_mov_b32 m0, s1\ns_nop 0\n{load}")[2]
    assert near(f"v_readfirstlane_b32 s6, v1\ns_nop 4\n{load}") == (0, 1, [])
    assert near(f"v_mov_b32_e32 v1, v2\n{load}") == (0, 1, [])  # (vector registers need no wait)


def test_product_kernels(tmp_path):
    if shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("no ROCm compiler")
    plan = subprocess.run(["make", "-n", "-B", "-C", DIR, "_build/mx4_gemm.o"], stdout=subprocess.PIPE, text=True,
                          check=True).stdout
    (command,) = [c for c in plan.split("\n") if "hipcc" in c and "csrc/mx4_gemm.hip" in c]
    out = tmp_path / "mx4_gemm.s"
    command = command.replace("-o _build/mx4_gemm.o", f"-S --cuda-device-only -o {out}")
    subprocess.run(command.split(), cwd=DIR, check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL,
                   timeout=300)
    products, loads, bad = near(out.read_text())
    assert products > 700 and loads > 400
    assert not bad, bad[:5]
