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


DOWN_PROGRAM = r"""
#include <cstdio>
#include <cstring>
#include "paged_tree.cuh"
using namespace abft;
int main() {
  long checks = 0;
  unsigned seed = 1;
  auto rnd = [&]() { return (seed = seed * 1664525u + 1013904223u) >> 8; };
  const int sizes[] = {1, 64, 65, 128, 200, 600};
  for (int n : sizes)
    for (int kind = 0; kind < 4; ++kind) {
      int up[600];
      for (int i = 0; i < n; ++i) {
        up[i] = kind == 0 ? i - 1 : kind == 1 ? (i ? 0 : -1) : i ? i - 1 - static_cast<int>(rnd() % (i < 9 ? i + 1 : 9)) : -1;
        if (kind == 3 && rnd() % 8 == 0) up[i] = static_cast<int>(rnd()) - (1 << 23);  // bad ones among them
        if (kind == 3 && rnd() % 8 == 0) up[i] = i;
      }
      for (int before = -n; before < 200; before += 7)  // slots before the drafted ones (below 0: more rows than tokens)
        for (int own = before < 0 ? -before : 0; own < n; ++own) {
          unsigned char see[1024] = {0};
          for (int i = 0; i < before; ++i) see[i] = 1;
          for (int i = own; i >= 0;) {
            if (before + i >= 0) see[before + i] = 1;
            i = up[i] < i ? up[i] : -1;
          }
          // From the last step to the first, by windows of 64 parents and nothing else.
          int at = own;
          for (int step = (before + n - 1) / 64; step >= 0; --step) {
            const int first = step * 64 - before;
            int held[64];
            memset(held, 0x7F, sizeof held);
            for (int c = 0; c < 64; ++c)
              if (first + c >= 0 && first + c < n) held[c] = up[first + c];
            uint32_t w[2];
            at = tree_words(TreeParents{held, first}, at, -first, w);
            if (at >= first && at >= 0) return 2;
            for (int k = 0; k < 64; ++k, ++checks)
              if ((w[k / 32] >> (k % 32) & 1u) != see[step * 64 + k]) {
                std::printf("n %d kind %d before %d step %d own %d key %d\n", n, kind, before, step, own, k);
                return 1;
              }
          }
        }
    }
  std::printf("%ld\n", checks);
  return 0;
}
"""


@pytest.mark.skipif(not _have_nvcc(), reason="needs nvcc")
def test_the_walk_goes_on_from_step_to_step(tmp_path):
    """Each step's words from where the walk has come to, with the parents of that step's rows alone."""
    src, exe = tmp_path / "down.cu", tmp_path / "down"
    src.write_text(DOWN_PROGRAM)
    subprocess.check_call([_build._nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2",
                           f"-I{_build.CSRC_DIR}", f"-I{_build.INCLUDE_DIR}", str(src), "-o", str(exe)])
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, (out.returncode, out.stdout)
    assert int(out.stdout) > 10_000_000
