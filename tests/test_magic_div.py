"""csrc/magic_div.h compiled for the host: the quotients by which kernels find heads, pages and tokens."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "magic_div.h"
using namespace pa;
static int wrong(uint32_t x, const MagicDiv& v) {
  if (div_by(x, v) == x / v.d) return 0;
  std::printf("%u / %u gave %u\n", x, v.d, div_by(x, v));
  return 1;
}
// Around every multiple of d is where a quotient goes wrong first, and the larger the worse.
static int check(uint32_t d) {
  const MagicDiv v = magic_div(d);
  int bad = wrong(0, v) + wrong(1, v) + wrong(0x7fffffffu, v);
  for (uint32_t top : {1u << 24, 0x7fffffffu}) {
    uint32_t q = top / d;
    for (int i = 0; i < 64 && q > 0; ++i, q = i < 32 ? q - 1 : q / 2 + (q & 1 ? 0 : 1)) {
      const uint64_t x = (uint64_t)q * d;
      if (x > 0x7fffffffu) continue;
      bad += wrong((uint32_t)x, v) + wrong((uint32_t)x - 1, v);
      if (x + d - 1 <= 0x7fffffffu) bad += wrong((uint32_t)(x + d - 1), v);
      if (q == 1) break;
    }
  }
  return bad;
}
int main() {
  int bad = 0;
  for (uint32_t d = 1; d <= 1u << 17 && bad < 5; ++d) bad += check(d);
  for (uint32_t s = 17; s < 31 && bad < 5; ++s)
    for (uint32_t e = 0; e < 200; ++e) bad += check((1u << s) + e) + check((1u << s) - e) + check((1u << s) + e * 40503u % (1u << s));
  bad += check(0x7fffffffu);
  // the rotation's pieces: every size of a head, with as many heads as its limit of 2^24 elements leaves
  for (uint32_t units = 1; units <= 1u << 20 && bad < 5; ++units) {
    const MagicDiv v = magic_div(units);
    const uint32_t heads = (1u << 24) / units;
    for (uint32_t h = heads; h > 0 && h + 2 > heads; --h) bad += wrong(h * units - 1, v) + wrong(h * units - units, v);
  }
  return bad != 0;
}
"""


def test_quotients(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    # in place of the device's runtime header
    (tmp_path / "hip").mkdir()
    (tmp_path / "hip" / "hip_runtime.h").write_text("#define __host__\n#define __device__\n"
                                                    "#define __forceinline__ inline\n")
    (tmp_path / "m.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-O2", "-std=c++17", "-I", ".", "-I", os.path.join(ROOT, "vllm-jax_amd", "csrc"), "m.cpp", "-o", "m"],
                   cwd=tmp_path, check=True)
    res = subprocess.run([str(tmp_path / "m")], capture_output=True, text=True, timeout=100)
    assert res.returncode == 0, res.stdout
