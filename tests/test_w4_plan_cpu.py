"""The 4-bit product's shared memory on the host: every byte that an MMA column may read lies in what the launch
asks for, for every row count, type and length.  (A read past it is an invalid access: it is shown here,
never by running it.)"""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
PROGRAM = r"""
#include <cstdio>
#include "w4.cuh"
using namespace llmp_b200::w4;
int main() {
  int bad = 0;
  for (int type : {kF32, kF16, kBF16}) {
    const int pieces = HalfPieces(type);
    for (int rows = 1; rows <= 16; ++rows) {
      const int tokens = ColumnTiles(rows, pieces) * TokensATile(pieces);
      if (rows > tokens) std::printf("type %d, %d rows: %d tokens in the column tiles\n", type, rows, tokens), ++bad;
      for (int token = 0; token < tokens; ++token) {
        for (int piece = 0; piece < pieces; ++piece) {
          const int column = StagedColumn(token, piece, rows, pieces);
          const bool zeros = column >= rows * pieces;
          if (zeros != (token >= rows) || (zeros && !ZeroColumn(rows, pieces))) {
            std::printf("type %d, %d rows: token %d, piece %d reads column %d\n", type, rows, token, piece, column), ++bad;
          }
          for (int wide = 0; wide < 2; ++wide) {
            for (int group : {32, 64, 128}) {
              for (int ranks = 1; ranks <= 8; ranks *= 2) {
                for (int steps : {8, 9, 24, 63, 128, 1024}) {
                  const int most = (steps + ranks - 1) / ranks;      // steps of the longest rank
                  const long long end = StagedAt(wide != 0, rows, BlockBytes(group)) + (column * static_cast<long long>(Pitch(most))) + (256 * most);
                  const long long bytes = SmemBytes(wide != 0, ranks, rows, steps, pieces, BlockBytes(group));
                  if (end > bytes) {
                    std::printf("type %d, %d rows, %d steps over %d: token %d reads to %lld of %lld bytes\n", type, rows, steps, ranks, token, end, bytes);
                    ++bad;
                  }
                }
              }
            }
          }
        }
      }
    }
  }
  return bad != 0;
}
"""


@pytest.mark.skipif(not os.path.exists(os.path.join(CUDA, "include", "cuda_fp16.h")), reason="needs the CUDA headers")
def test_every_column_that_is_read_is_staged(tmp_path):
    source, program = tmp_path / "plan.cc", tmp_path / "plan"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "llmp_b200", "csrc"),
                    "-I", os.path.join(CUDA, "include"), str(source), "-o", str(program)], check=True)
    ran = subprocess.run([str(program)], capture_output=True, text=True)
    assert ran.returncode == 0, ran.stdout[:2000]
