"""Where packed attention's copies of keys and values read: every lane of every
copy of a step, for every number of rows left, computed by a host program from the
kernel's own header. A read of a row that is there lies in that row; one past the
last is dropped by what the hardware compares, an address's vector offset and the
buffer's bytes."""

import shutil
import subprocess

import pytest

from conftest import PACKAGE

PROGRAM = r"""
#include "packed_copies.hpp"
#include <cstdio>
#include <set>
using namespace mi::packed_copies;

int main()
{
  struct Form { int hd, waves, keys; };
  const Form forms[] = {{64, 4, 128}, {128, 4, 128}, {64, 8, 128}, {128, 4, 64}};
  const unsigned strides[] = {0, 8, 1024, (1u << 20) + 8, (1u << 24) - 8}; // halves past a row's own
  for (const Form &f : forms)
  {
    const int at_once = rows_at_once(f.hd, f.waves), count = copies(f.hd, f.waves, f.keys);
    if (at_once * count != f.keys) { std::printf("rows\n"); return 1; }
    for (const unsigned more : strides)
    {
      const unsigned elements = f.hd + more < (1u << 24) ? f.hd + more : (1u << 24) - 8;
      const unsigned step = 2 * elements;
      for (int left = 0; left < f.keys + 2; ++left) // rows behind the step's first
      {
        const unsigned bytes = rows_bytes(left, step, f.hd);
        std::set<unsigned long long> seen;
        for (int t = 0; t < 64 * f.waves; ++t)
        {
          for (int i = 0; i < count; ++i)
          {
            const int row = t / pieces(f.hd) + i * at_once, piece = t % pieces(f.hd);
            const unsigned at = copy_at(lane_at(t / pieces(f.hd), piece, step), i, at_once, step);
            const unsigned long long whole = static_cast<unsigned long long>(row) * step + 16ull * piece;
            const bool dropped = at >= bytes;
            if (at != whole || dropped != (row > left) || (!dropped && at + 16ull > bytes))
            {
              std::printf("hd %d step %u left %d row %d piece %d: %u of %u\n", f.hd, step, left, row, piece, at, bytes);
              return 1;
            }
            seen.insert(whole);
          }
        }
        if (seen.size() != static_cast<std::size_t>(f.keys) * pieces(f.hd)) { std::printf("pieces\n"); return 1; }
      }
    }
  }
  return 0;
}
"""


def test_every_lane_reads_its_row_or_nothing(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    source, program = tmp_path / "copies.cpp", tmp_path / "copies"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", f"-I{PACKAGE / 'csrc'}", str(source), "-o", str(program)],
                   check=True)
    result = subprocess.run([str(program)], capture_output=True, text=True)
    assert result.returncode == 0, result.stdout
