"""Which bytes of a cached head the attention kernels load, and where these lie in LDS: the kernels' own
header, built for the host (CPU only)."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "qwen-ascend_amd" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include "attention_layout.h"

template <int NK, bool FULL, bool KEYS>
int check(int D) {
  using L = Layout<NK>;
  int bad = 0;
  for (int row = 0; row < 64; ++row) {
    bool there[32] = {};
    for (int place = 0; place < L::PIECES; ++place) {
      const int lane = row % L::RPI * L::PIECES + place, piece = L::template piece_of<FULL, KEYS>(lane, row, D);
      // within the head
      bad += !(piece >= 0 && 16 * piece + 16 <= 2 * D);
      // a piece of the head lies where it is read from
      const int want = place ^ (KEYS ? L::k_swizzle(row) : L::v_swizzle(row));
      if (want < D / 8) bad += piece != want, there[want] = true;
    }
    for (int piece = 0; piece < D / 8; ++piece) bad += !there[piece];
  }
  return bad;
}
template <int NK>
int heads(int D) {
  if (D > 32 * NK || D < Layout<NK>::D_LEAST) return 1;
  return D == 32 * NK ? check<NK, true, true>(D) + check<NK, true, false>(D) : check<NK, false, true>(D) + check<NK, false, false>(D);
}

int main() {
  int wrong = 0;
  for (int D = 8; D <= 256; D += 8) {
    const int nk = blocks_of(D);
    const int bad = nk == 2 ? heads<2>(D) : nk == 3 ? heads<3>(D) : nk == 4 ? heads<4>(D) : nk == 6 ? heads<6>(D) : nk == 8 ? heads<8>(D) : 1;
    if (bad) std::printf("heads of %d: %d loads\n", D, bad);
    wrong += bad != 0;
  }
  return wrong != 0;
}
"""


def test_loads_stay_within_a_head(tmp_path):
    """For every head size: no lane's 16 bytes pass the head's end, which may be the cache's, and each piece of the
    head comes to its place."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    source, exe = tmp_path / "layout.cpp", tmp_path / "layout"
    source.write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-O1", "-I", str(CSRC), str(source), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
