"""What the matrix kernels' inline assembly relies on and no compiler checks, looked up in
the assembly that hipcc writes for ragged_gemm.hip: nothing is spilled; a vector
instruction's scalar result is five instructions old when a vector memory instruction reads
it; a matrix product's result is left alone for 20 instruction slots by all but further
products into it, and its operands are not written by the two vector instructions before."""
import os
import re
import shutil
import subprocess

import pytest

SOURCE = os.path.join(os.path.dirname(__file__), "..", "learning_at_home_amd", "ops", "hip", "ragged_gemm.hip")
FLAGS = "-O3 -std=c++17 --offload-arch=gfx950 -Xclang -target-feature -Xclang -packed-fp32-ops -S --offload-device-only"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    out = tmp_path_factory.mktemp("code") / "ragged_gemm.s"
    subprocess.run([hipcc, *FLAGS.split(), SOURCE, "-o", str(out)], check=True, capture_output=True)
    text = out.read_text()
    found = {}
    for m in re.finditer(r"^(_Z\S*ragged_(?:big|rows)_kernel\S*):.*?\.Lfunc_end", text, re.M | re.S):
        lines = (line.split(";")[0].strip() for line in m.group(0).split("\n")[1:])
        found[m.group(1)] = [line for line in lines if line and not line.startswith(".") and not line.endswith(":")]
    assert len(found) == 15
    return text, found


def registers(text, kinds):
    out = set()
    for kind, first, last, k, one in re.findall(r"\b([%s])\[(\d+):(\d+)\]|\b([%s])(\d+)\b" % (kinds, kinds), text):
        out |= {k + one} if k else {kind + str(i) for i in range(int(first), int(last) + 1)}
    return out


def slots(lines):
    """(slot, operation, operands) of each instruction; s_nop n takes n + 1."""
    slot = 0
    for line in lines:
        op, _, rest = line.partition(" ")
        yield slot, op, rest.split(",")
        slot += int(rest) + 1 if op == "s_nop" else 1


def test_nothing_is_spilled(kernels):
    text, _ = kernels
    spills = re.findall(r"\.name:\s+(_Z\S*ragged_(?:big|rows)\S*).*?\.vgpr_spill_count:\s+(\d+)", text, re.S)
    assert len(spills) == 15
    assert {n for _, n in spills} == {"0"}
    assert not any(line.startswith("scratch_") for lines in kernels[1].values() for line in lines)


def test_descriptors_have_settled(kernels):
    for name, lines in kernels[1].items():
        written = {}
        for slot, op, args in slots(lines):
            if op.startswith("buffer_"):
                for r in registers(",".join(args), "s"):
                    assert slot - written.get(r, -9) > 5, (name, op, args)
            elif op.startswith("v_"):
                written.update((r, slot) for r in registers(args[0], "s"))
            elif op.startswith("s_"):
                for r in registers(args[0], "s"):
                    written.pop(r, None)


def test_products_have_settled(kernels):
    for name, lines in kernels[1].items():
        if "big" not in name:
            continue
        product, vector = {}, {}
        for slot, op, args in slots(lines):
            every = registers(",".join(args), "va")
            if op.startswith("v_mfma"):
                for r in registers(",".join(args[1:]), "va"):
                    assert slot - vector.get(r, -9) > 2, (name, op, args)
                for r in registers(",".join(args[1:3]), "va"):
                    assert slot - product.get(r, -99) >= 20, (name, op, args)
                product.update((r, slot) for r in registers(args[0], "va"))
            elif op.startswith(("v_", "ds_", "buffer_", "global_")):
                for r in every:
                    assert slot - product.get(r, -99) >= 20, (name, op, args)
                if op.startswith("v_"):
                    vector.update((r, slot) for r in registers(args[0], "va"))
