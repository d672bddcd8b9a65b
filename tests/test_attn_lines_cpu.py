"""The attention kernels' lines by distance in LDS: every index that any tile of any accepted bucketing touches, on the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# R, the first distance of the last bucket, lies in [1, VDB_OP_MAX_DISTANCE]; a tile's e0 is a multiple of 32
PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "attn_lines.h"
using namespace vdbk;
int main() {
  int bad = 0;
  for (int reach = 1; reach <= 512; ++reach)
    for (int e0 = -1024; e0 <= 1024; e0 += 32) {
      if (tile_is_far(e0, reach)) continue;
      for (int half = 0; half < 2; ++half)
        for (int l = 0; l < 32; ++l) {
          // sums: the two places a lane adds to stay inside its half's own line
          const int at = sums_at(reach, e0, half, l);
          if (at < 0 || at + 32 >= sums_span(reach)) { if (!bad++) printf("sums: reach %d e0 %d half %d lane %d: %d, %d of %d\n", reach, e0, half, l, at, at + 32, sums_span(reach)); }
          for (int r = 0; r < 16; ++r) {
            const int row = (r & 3) + 8 * (r >> 2) + 4 * half;
            // what the 32 x 32 distances of the tile belong to is one of the two
            const int e = sums_zero(reach) + e0 + row - l;
            if (e < 0 || e >= sums_span(reach)) bad++;
            // start values, keys in the rows and queries in the rows
            for (int s : {start_at(reach, e0 + row - l), start_at(reach, e0 + l - row)})
              if (s < 0 || s >= start_span(reach)) { if (!bad++) printf("start: reach %d e0 %d\n", reach, e0); }
          }
        }
    }
  printf("%d\n", bad);
  return bad != 0;
}
"""


def test_every_tile_stays_inside_its_line(tmp_path):
    source = tmp_path / "lines.cpp"
    source.write_text(PROGRAM)
    exe = str(tmp_path / "lines")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "vectordb_amd", "csrc"), "-o", exe, str(source)])
    done = subprocess.run([exe], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
