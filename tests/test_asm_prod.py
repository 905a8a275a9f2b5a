"""The products' kernels as compiled for gfx950.

* The result of an MFMA is there some cycles after the instruction, and the compiler keeps a reader behind it by
  wait states, but not past a conditional branch. The kernels put settle()'s waits where their loops end and keep the other
  readers in the products' own block: on every path from an MFMA, past branches too, no instruction other than an MFMA that adds to
  it names the result within the wait states that it needs.
* No kernel of 16-bit rows spills vector registers.
"""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from test_asm_w4 import CSRC, HIPCC, _build_flags, _registers

pytestmark = pytest.mark.skipif(not shutil.which(HIPCC) and not Path(HIPCC).exists(), reason="hipcc not available")

MFMA = re.compile(r"(v_mfma\S+) ([av]\[\d+:\d+\])")


def states_of(op):
    """Wait states between an MFMA and a vector instruction that reads its result: its passes and three more."""
    passes = 16 if "32x32x2_f32" in op else 8 if re.search("32x32x16|16x16x4_f32|f8f6f4", op) else 4
    return passes + 3


def early_readers(lines):
    """(MFMAs, those whose result another instruction names too early on a path past a branch)."""
    code, labels = [], {}
    for t in (l.strip() for l in lines):
        if re.match(r"\.LBB\d+_\d+:", t):
            labels[t.split(":")[0]] = len(code)
        elif t and not t.startswith((";", ".")) and not t.endswith(":"):
            code.append(t.split(";")[0].strip())
    total, found = 0, []
    for n, t in enumerate(code):
        m = MFMA.match(t)
        if not m:
            continue
        total += 1
        result, need = _registers(m.group(2)), states_of(m.group(1))
        todo, seen = [(n + 1, 0, False)], set()
        while todo:
            at, states, past = todo.pop()
            while at < len(code) and states < need:
                if (at, past) in seen:
                    break
                seen.add((at, past))
                u = code[at]
                if _registers(u) & result:
                    if past and not u.startswith("v_mfma"):
                        found.append(f"{t} -> {u} after {states}")
                    break
                b = re.match(r"s_(c?branch)\S* (\.LBB\d+_\d+)", u)
                if u.startswith("s_endpgm"):
                    break
                if b:
                    todo.append((labels[b.group(2)], states + 1, True))
                    if b.group(1) == "branch":
                        break
                    past = True
                # an MFMA behind this one waits for the pipe: it is issued at the earliest when this one's passes are half through
                states += int(u.split()[1], 0) + 1 if u.startswith("s_nop") else 4 if u.startswith("v_mfma") else 1
                at += 1
    return total, found


def test_the_scan_finds_an_early_reader():
    lines = ["v_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], v[24:27], v[0:15]", "s_cbranch_scc1 .LBB0_2", "s_nop 15", "s_endpgm",
             ".LBB0_2:", "v_add_f32_e32 v30, v3, v4"]
    assert early_readers(lines)[1]
    lines[5:5] = ["s_nop 15", "s_nop 7"]
    assert early_readers(lines) == (1, [])


@pytest.mark.parametrize("name,mfmas", [("prod_bf16", 700), ("prod_f32", 1500)])
def test_results_of_mfmas_are_read_late_enough(tmp_path, name, mfmas):
    out = tmp_path / (name + ".s")
    cmd = [HIPCC, *_build_flags(), "--cuda-device-only", "-S", str(CSRC / (name + ".hip")), "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=900)
    text = out.read_text()
    total = 0
    for kernel in re.split(r"\n(?=_ZN\S+:)", text)[1:]:
        n, found = early_readers(kernel.split("\n"))
        total += n
        assert not found, (kernel.split(":")[0], found[:5])
    assert total > mfmas
    spills = [int(s) for s in re.findall(r"\.vgpr_spill_count:\s+(\d+)", text)]
    assert len(spills) > 40 and (name == "prod_f32" or not any(spills))
