"""The products' stores from fragments to rows (store_rows in prod_tile.h), compiled for the CPU with a wave's 64 lanes one
after the other: every value comes to its place, no place outside the rows and columns that are there is written, and the
rows that are not there are not asked for: a routed call reads a row's place from the routes' order, which ends with
the last row."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from test_asm_w4 import CSRC, HIPCC

CLANG = Path(shutil.which(HIPCC) or HIPCC).resolve().parent.parent / "llvm" / "bin" / "clang++"
pytestmark = pytest.mark.skipif(not CLANG.exists(), reason="clang++ not available")

HEAD = r"""
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>
#define __device__
#define __forceinline__ inline
#define __builtin_amdgcn_fence(...)
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
template <typename S> struct vec4_of { typedef S type __attribute__((ext_vector_type(4))); };
template <bool STREAM> void gstore(void* p, u32x4_t v) { __builtin_memcpy(p, &v, 16); }
"""

MAIN = r"""
template <typename O, int FR, int NO>
void check() {
  constexpr int W = FR * NO, STRIDE = W + 3;
  alignas(16) static uint8_t stage[STAGE_BYTES];
  for (int rows = 1; rows <= FR; ++rows)
    for (int cols = 1; cols <= W + 1; ++cols) {
      std::vector<O> out(FR * STRIDE, (O)-1);
      for (int twice = 0; twice < 2; ++twice)  // the second time every lane's part of the area is there
        for (int lane = 0; lane < 64; ++lane) {
          auto v = [&](int i, int r) {  // fragment i: row lane % FR, column 4 (lane / FR) + r % 4 of every group of 256 / FR
            return (float)(lane % FR * W + FR * i + 256 / FR * (r / 4) + 4 * (lane / FR) + r % 4);
          };
          auto at = [&](int i) {
            if (i < 0 || i >= rows) printf("row %d of %d (values of %zu bytes, %d x %d)\n", i, rows, sizeof(O), FR, NO), exit(1);
            return (int64_t)i * STRIDE;
          };
          store_rows<O, FR, NO, false>(stage, v, out.data(), at, rows, cols, lane);
        }
      for (int r = 0; r < FR; ++r)
        for (int c = 0; c < STRIDE; ++c) {
          const bool there = r < rows && c < cols && c < W;
          if (out[r * STRIDE + c] != (O)(there ? r * W + c : -1)) printf("place %d %d of %d %d\n", r, c, rows, cols), exit(1);
        }
    }
}
int main() {
  check<float, 32, 1>(), check<float, 32, 2>(), check<float, 16, 4>();
  check<_Float16, 32, 1>(), check<_Float16, 32, 2>(), check<_Float16, 16, 4>();
}
"""


def test_store_rows(tmp_path):
    text = (CSRC / "prod_tile.h").read_text()
    body = re.search(r"constexpr int STAGE_BYTES.*?\n}\n", text, re.S).group(0)
    assert "void store_rows" in body
    source, program = tmp_path / "store.cpp", tmp_path / "store"
    source.write_text(HEAD + body + MAIN)
    subprocess.run([CLANG, "-std=c++17", "-O1", str(source), "-o", str(program)], check=True, timeout=300)
    run = subprocess.run([program], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout
