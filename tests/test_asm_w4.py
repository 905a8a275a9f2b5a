"""The 4-bit products' kernels as compiled for gfx950.

* The result of an MFMA is there some cycles after the instruction, and the compiler keeps a reader
  behind it by wait states. Where it had moved the reader past a conditional branch, it left them out on
  the taken side (the sums of three activation rows in four were wrong there). So no branch may stand
  between an MFMA and the reader of its result: within 12 wait states of the last MFMA of a chain, none.
* No kernel spills vector registers.
"""
import importlib.util
import os
import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "kt-prefill-lend_amd" / "csrc"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

pytestmark = pytest.mark.skipif(not shutil.which(HIPCC) and not Path(HIPCC).exists(), reason="hipcc not available")

STATES = 12
MFMA = re.compile(r"v_mfma\S+ ([av])\[(\d+):(\d+)\]")


def _registers(text):
    """Vector registers that an instruction names."""
    out = set()
    for kind, lo, hi in re.findall(r"\b([av])\[(\d+):(\d+)\]", text):
        out |= {(kind, i) for i in range(int(lo), int(hi) + 1)}
    return out | {(kind, int(i)) for kind, i in re.findall(r"\b([av])(\d+)\b", text)}


def branches_after_mfma(lines):
    """(MFMAs, those with a branch before the first instruction that names their result)."""
    total, found = 0, []
    code = [t for t in (l.strip() for l in lines) if t and not t.startswith((";", "."))]
    for n, t in enumerate(code):
        m = MFMA.match(t)
        if not m:
            continue
        total += 1
        result = _registers(m.group(0))
        states = 0
        for u in code[n + 1:n + 40]:
            if _registers(u) & result:
                break  # in the same block, where the compiler counts right
            if re.match(r"s_(c?branch|endpgm|setpc)", u):
                found.append(f"{t} -> {u}")
                break
            states += int(u.split()[1]) + 1 if u.startswith("s_nop") else 1
            if states > STATES:
                break
    return total, found


def test_the_scan_finds_a_branch():
    lines = ["v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], 0", "s_cbranch_vccnz .L1", "v_fmac_f32 v20, v21, v0"]
    assert branches_after_mfma(lines)[1]
    lines[1:1] = ["s_nop 7", "v_fmac_f32 v20, v21, v0"]
    assert branches_after_mfma(lines) == (1, [])


def test_mfma_results_are_read_before_a_branch(tmp_path):
    out = tmp_path / "w4_bf16.s"
    cmd = [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-mllvm", "-amdgpu-kernarg-preload-count=16", "--cuda-device-only", "-S",
           str(CSRC / "w4_bf16.hip"), "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=900)
    lines = out.read_text().split("\n")
    total, found = branches_after_mfma(lines)
    assert total > 1000
    assert not found, found[:5]
    spills = [int(l.split(":")[1]) for l in lines if ".vgpr_spill_count:" in l]
    assert len(spills) > 40 and not any(spills)


def _build_flags():
    """The flags that the library is built with."""
    spec = importlib.util.spec_from_file_location("ktmi_build", CSRC.parent / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    return build.HIP_FLAGS


# fp32 rows take three products an operand, but have no passes of 32 rows: fewer kernels
@pytest.mark.parametrize("name,mfmas,kernels", [("w4_f16", 5000, 60), ("w4_f32", 4000, 24)])
def test_mfma_results_are_read_before_a_branch_in_the_other_types(tmp_path, name, mfmas, kernels):
    out = tmp_path / (name + ".s")
    cmd = [HIPCC, *_build_flags(), "--cuda-device-only", "-S", str(CSRC / (name + ".hip")), "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=900)
    lines = out.read_text().split("\n")
    total, found = branches_after_mfma(lines)
    assert total > mfmas
    assert not found, found[:5]
    spills = [int(l.split(":")[1]) for l in lines if ".vgpr_spill_count:" in l]
    assert len(spills) > kernels and not any(spills)
