"""The tree's list of work on the host: places of sequences whose boundaries fall."""
import subprocess

import pytest

from vla_abft_estimate_b200 import _build

from .test_paged_host import _have_nvcc

PLACES_PROGRAM = r"""
#include <cstdio>
#include "paged_tree.cuh"
using namespace abft;
int main() {
  // As the lanes of a warp count them: each adds its sequences, then the lanes' sums are scanned.
  const long long each[] = {0, 1, 7, 4099, 262144LL * 3, 1LL << 26, (1LL << 31) - 2};
  for (int batch = 1; batch <= 600; batch = batch * 2 + 1)
    for (long long places : each) {
      int sums[32];
      long long whole[32];
      for (int lane = 0; lane < 32; ++lane) {
        sums[lane] = 0, whole[lane] = 0;
        const int part = (batch + 31) / 32;
        for (int b = lane * part; b < batch && b < (lane + 1) * part; ++b) {
          sums[lane] = add_places(sums[lane], b % 2 ? 0 : static_cast<int>(places));
          whole[lane] += b % 2 ? 0 : places;
        }
      }
      for (int o = 1; o < 32; o <<= 1)
        for (int lane = 31; lane >= o; --lane) {
          sums[lane] = add_places(sums[lane], sums[lane - o]);
          whole[lane] += whole[lane - o];
        }
      for (int lane = 0; lane < 32; ++lane) {
        const long long want = whole[lane] < kNoMore ? whole[lane] : kNoMore;
        if (sums[lane] != want) {
          std::printf("batch %d places %lld lane %d: %d, not %lld\n", batch, places, lane, sums[lane], want);
          return 1;
        }
      }
    }
  return 0;
}
"""


@pytest.mark.skipif(not _have_nvcc(), reason="needs nvcc")
def test_places_that_pass_31_bits(tmp_path):
    src, exe = tmp_path / "places.cu", tmp_path / "places"
    src.write_text(PLACES_PROGRAM)
    subprocess.check_call([_build._nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2",
                           f"-I{_build.CSRC_DIR}", f"-I{_build.INCLUDE_DIR}", str(src), "-o", str(exe)])
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
