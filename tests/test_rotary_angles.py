"""The angle arithmetic of the rotary kernels, compiled for the host: no step of it is undefined in C++."""

import math
import pathlib
import shutil
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent

MAIN = r"""
#include <cmath>
#include <cstdio>
#include <initializer_list>
#define __device__
#define __forceinline__ inline
%s
int main() {
  // fractions of a turn all around, and next to the borders of every eighth
  for (unsigned long long i = 0; i < 4096; ++i)
    for (long long off : {0ll, -1ll, 1ll, -0x80000000ll, 0x80000000ll, 0x10000000000ll}) {
      const unsigned long long turn = (i << 52) + (unsigned long long)off;
      float c, s;
      cos_sin(1, turn, &c, &s);
      std::printf("%%llu %%.9g %%.9g\n", turn, c, s);
      cos_sin(-3, turn, &c, &s);  // (and what is a multiple of it)
    }
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_angles_all_around(tmp_path):
    text = (ROOT / "attnax_b200" / "csrc" / "rotary.cu").read_text()
    start = text.index("__device__ __forceinline__ void cos_sin(")
    (tmp_path / "angles.cc").write_text(MAIN % text[start:text.index("\n}\n", start) + 3])
    # (an overflow of a signed integer ends the program)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=signed-integer-overflow", "-fsanitize-undefined-trap-on-error",
                    "-o", tmp_path / "angles", tmp_path / "angles.cc"], check=True)
    out = subprocess.run([tmp_path / "angles"], capture_output=True, text=True)
    assert out.returncode == 0, f"undefined arithmetic (status {out.returncode})"
    lines = out.stdout.splitlines()
    assert len(lines) == 4096 * 6
    for line in lines:
        turn, c, s = line.split()
        a = 2 * math.pi * (int(turn) / 2**64)
        # 6 half steps of 2^-24 of the value at most, and 2^-33 turns of the angle that its 32 bits leave out
        for got, want in ((c, math.cos(a)), (s, math.sin(a))):
            assert abs(float(got) - want) <= 6 * 2.0 ** -24 * abs(want) + 2 * math.pi * 2.0 ** -33 + 1e-15
