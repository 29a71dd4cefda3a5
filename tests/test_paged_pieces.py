"""Paged prefill's list of work on the host: the rows of a sequence lie within
the call's whatever the boundaries say, and the pieces chosen for a batch fit
the grid and the scratch, whatever its lengths."""
import ctypes
import subprocess

import pytest

from vla_abft_estimate_b200 import _build
from vla_abft_estimate_b200 import _native as N

from .test_paged_host import _have_nvcc, _kv

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "paged_prefill.cuh"
using namespace abft;
static uint64_t state = 88172645463325252ull;
static int below(int n) {
  state ^= state << 13, state ^= state >> 7, state ^= state << 17;
  return static_cast<int>((state >> 11) % n);
}
int main() {
  static int blocks[256], steps[256];
  for (int piece : {1, 4, 100})
    for (int s = 0; s < 1000; ++s) {
      const int n = pieces_of(s, piece);
      if (n < 1 || (s > 0 && ((n - 1) * piece >= s || n * piece < s))) return std::printf("pieces_of %d %d\n", s, piece), 1;
    }
  const int edge[] = {-2147483647 - 1, -5, -1, 0, 1, 3, 7, 59, 60, 61, 900, 2147483647};
  for (int lo : edge)
    for (int hi : edge) {
      const int cu[2] = {lo, hi};
      int begin, end;
      packed_range(cu, 0, 60, &begin, &end);
      const bool ok = 0 <= lo && lo <= hi && hi <= 60;
      if (ok ? begin != lo || end != hi : begin != 0 || end != 0) return std::printf("packed_range %d %d\n", lo, hi), 1;
    }
  long cut = 0, tight = 0;
  for (int round = 0; round < 300000; ++round) {
    const int batch = 1 + below(1 << below(8)), room = 1 + below(200), splits = 1 + below(200);
    const int top = 1 + below(1 << (1 + below(round % 50 == 0 ? 22 : 12))), idle = below(4);
    WorkSums all = {0, 0, 0, 0};
    for (int b = 0; b < batch; ++b) {
      blocks[b] = below(4) == 0 ? 0 : 1 + below(3);
      steps[b] = below(4) < idle ? 0 : 1 + below(top);
      all.add(blocks[b], steps[b]);
    }
    const int piece = fitting_piece(all, room, splits);
    auto places = [&](int of) {
      long sum = 0;
      for (int b = 0; b < batch; ++b) sum += static_cast<long>(blocks[b]) * pieces_of(steps[b], of);
      return sum;
    };
    const long limit = all.blocks < room ? room : all.blocks;
    if (places(piece) > limit) return std::printf("%ld places for %ld\n", places(piece), limit), 1;
    for (int b = 0; b < batch; ++b)
      if (blocks[b] > 0 && pieces_of(steps[b], piece) > splits) return std::printf("more pieces than scratch\n"), 1;
    cut += places(piece) > all.blocks;
    tight += places(piece) > all.blocks && places(piece) == room - 1;  // (weight - blocks) / piece < room - blocks
  }
  std::printf("%ld %ld\n", cut, tight);
  return 0;
}
"""


@pytest.mark.skipif(not _have_nvcc(), reason="needs nvcc")
def test_chosen_pieces_fit_the_grid(tmp_path):
    """Random batches, sequences without keys and without new rows among them:
    no more places than items that run at once (or than blocks, when those alone
    are more), no sequence in more pieces than the scratch holds. Boundaries that fall or lie
    outside the rows give a sequence none."""
    src = tmp_path / "pieces.cu"
    src.write_text(PROGRAM)
    exe = tmp_path / "pieces"
    subprocess.check_call([_build._nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2",
                           f"-I{_build.CSRC_DIR}", f"-I{_build.INCLUDE_DIR}", str(src), "-o", str(exe)])
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    cut, tight = (int(x) for x in out.stdout.split())
    assert cut > 10_000 and tight > 100  # batches that are cut, and lists that reach the bound


def test_decode_list_is_counted_in_32_bits():
    """2^31 places in the list of tiles are refused, the batch below is not (the
    table, 2^30 - 16 slots, is the widest that any call takes)."""
    L = N.lib()

    def scratch(batch):
        a = N.PagedAttnArgs()
        a.kv, a.q, a.out, a.tokens, a.heads, a.scale, a.num_sms = _kv(), 0x50000, 0x60000, batch, 28, 0.1, 148
        a.kv.max_pages = a.kv.table_stride = (1 << 26) - 1
        a.kv.batch = batch
        return L.abft_paged_decode_workspace_bytes(ctypes.byref(a))  # 0 for a call that is refused

    assert scratch(16) == 0  # 64 segments of 2^25 tiles
    assert scratch(15) > 0
