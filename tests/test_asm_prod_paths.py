"""The products' kernels as compiled for gfx950, on every path: the scan of test_asm_prod ends a path where another one came by
before, also if that one had more wait states behind it. Here a path goes on where it comes with fewer; an MFMA counts as
one state, as the compiler counts it, and one that takes another's result as a factor counts as a reader. Of all element types.

No instruction names an MFMA's result within the wait states that it needs, on any path past a branch; before one, the
compiler keeps them. No kernel of 16-bit rows spills vector registers."""
import heapq
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

from test_asm_prod import early_readers as pruned_scan
from test_asm_w4 import CSRC, HIPCC, _build_flags, _registers

pytestmark = pytest.mark.skipif(not shutil.which(HIPCC) and not Path(HIPCC).exists(), reason="hipcc not available")

MFMA = re.compile(r"(v_mfma\S+) (.*)")


def states_of(op):
    """Wait states between an MFMA and a reader of its result, as the compiler puts them on gfx950 in straight code: the passes
    and four more, of fp32 operands two more."""
    if re.search(r"x[24]_f32", op):
        return 18 if "32x32" in op else 10
    return 12 if re.search("32x32x16|f8f6f4", op) else 8


def reads(u, result):
    """Whether instruction u has to wait for an MFMA's result: an MFMA that adds to the whole of it does not, nor does one that
    writes there, which ends behind it."""
    m = MFMA.match(u)
    if not m:
        return bool(_registers(u) & result)
    a, b, c = (_registers(t) for t in m.group(2).split(", ")[1:4])
    return bool((a | b) & result) or bool(c & result and c != result)


def early_readers(lines):
    """(MFMAs, those whose result is named too early on a path past a branch)."""
    code, labels = [], {}
    for t in (l.split(";")[0].strip() for l in lines):
        if re.match(r"\.LBB\d+_\d+:", t):
            labels[t.split(":")[0]] = len(code)
        elif t and not t.startswith(".") and not t.endswith(":"):
            code.append(t)
    total, found = 0, []
    for n, t in enumerate(code):
        m = MFMA.match(t)
        if not m:
            continue
        total += 1
        result, need = _registers(m.group(2).split(", ")[0]), states_of(m.group(1))
        todo, least = [(0, n + 1, False)], {}
        while todo:
            states, at, past = heapq.heappop(todo)  # the path with the fewest states first
            if at >= len(code) or states >= need or (at, past) in least:
                continue
            least[at, past] = states
            u = code[at]
            if past and reads(u, result):
                found.append(f"{t} -> {u} after {states} of {need}")
                continue
            if _registers(u) & result or u.startswith(("s_endpgm", "s_setpc", "s_swappc")):
                continue
            states += int(u.split()[1], 0) + 1 if u.startswith("s_nop") else 1
            b = re.match(r"s_(c?branch)\S* (\.LBB\d+_\d+)", u)
            if b:
                heapq.heappush(todo, (states, labels[b.group(2)], True))
            if not b or b.group(1) == "cbranch":
                heapq.heappush(todo, (states, at + 1, past or bool(b)))
    return total, found


def test_a_shorter_path_that_joins_later_is_followed():
    """The branch's path comes to the last wait with less behind it than the path that goes straight on, which is scanned first."""
    head = ["v_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], v[24:27], v[0:15]", "s_cbranch_scc1 .LBB0_2", "s_nop 3", ".LBB0_2:"]
    lines = head + ["s_nop 6", "v_add_f32_e32 v30, v3, v4"]
    assert pruned_scan(lines) == (1, [])  # 12 states by the straight path, 8 by the branch
    assert early_readers(lines)[1]
    assert early_readers(head + ["s_nop 10", "v_add_f32_e32 v30, v3, v4"]) == (1, [])


def test_readers():
    branch = ["v_mfma_f32_16x16x32_f16 v[0:3], v[20:23], v[24:27], 0", "s_cbranch_scc1 .LBB0_2", ".LBB0_2:"]
    for reader, early in [("v_mfma_f32_16x16x32_f16 v[0:3], v[20:23], v[24:27], v[0:3]", False),
                          ("v_mfma_f32_16x16x32_f16 v[2:5], v[20:23], v[24:27], v[0:3]", False),
                          ("v_mfma_f32_16x16x32_f16 v[4:7], v[0:3], v[24:27], v[4:7]", True),
                          ("v_mfma_f32_16x16x32_f16 v[2:5], v[20:23], v[24:27], v[2:5]", True),
                          ("ds_write_b128 v9, v[0:3]", True), ("v_mov_b32_e32 v2, 0", True), ("v_mov_b32_e32 v4, 0", False)]:
        assert bool(early_readers(branch + [reader, "s_nop 15"])[1]) == early, reader


def test_results_of_mfmas_are_read_late_enough(tmp_path):
    def compiled(name):
        out = tmp_path / (name + ".s")
        cmd = [HIPCC, *_build_flags(), "--cuda-device-only", "-S", str(CSRC / (name + ".hip")), "-o", str(out)]
        subprocess.run(cmd, check=True, capture_output=True, timeout=900)
        return out.read_text()

    names = ["prod_bf16", "prod_f16", "prod_f32"]
    with ThreadPoolExecutor(3) as pool:
        texts = list(pool.map(compiled, names))
    for name, text in zip(names, texts):
        total = 0
        for kernel in re.split(r"\n(?=_ZN\S+:)", text)[1:]:
            n, found = early_readers(kernel.split("\n"))
            total += n
            assert not found, (kernel.split(":")[0], found[:5])
        assert total > (1500 if name == "prod_f32" else 700)
        spills = [int(s) for s in re.findall(r"\.vgpr_spill_count:\s+(\d+)", text)]
        assert len(spills) > 40 and (name == "prod_f32" or not any(spills))
