"""Paged cache on the host: index arithmetic, struct layouts, refusals."""
import ctypes
import shutil
import subprocess

import pytest
import torch

from vla_abft_estimate_b200 import _build
from vla_abft_estimate_b200 import _native as N
from vla_abft_estimate_b200.paged import PagedKVCache, rope_table

INDEX_PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "paged_prefill.cuh"
using namespace abft;
static void need(bool ok, const char* what) {
  if (!ok) { std::printf("FAILED %s\n", what); std::exit(1); }
}
int main() {
  long checks = 0;
  // pieces cover the tiles once, in order, and split_count counts the non-empty ones
  const int sizes[] = {0, 1, 2, 3, 4, 5, 31, 32, 33, 1000, 4096, 1 << 25};
  const int pieces[] = {1, 2, 3, 7, 37, 148, 1000, 1 << 20};
  for (int tiles : sizes)
    for (int splits : pieces) {
      int at = 0, filled = 0;
      for (int s = 0; s < splits; ++s) {
        int b, e;
        split_tiles(tiles, splits, s, &b, &e);
        need(b <= e && e <= tiles, "range");
        if (b < e) {
          need(b == at, "gap");
          need(s == filled, "an empty piece before a filled one");
          at = e;
          ++filled;
        }
        ++checks;
      }
      need(at == tiles, "cover");
      need(filled == split_count(tiles, splits), "count");
    }
  // shares cover the tiles in order, differ by one at most, and share_of inverts them
  for (int total : {0, 1, 3, 4, 591, 592, 5000})
    for (int shares : {1, 2, 4, 12, 592}) {
      need(share_start(total, shares, 0) == 0 && share_start(total, shares, shares) == total, "share ends");
      for (int w = 0; w < shares; ++w) {
        const int a = share_start(total, shares, w), e = share_start(total, shares, w + 1);
        need(a <= e && e - a >= total / shares && e - a <= total / shares + 1, "share size");
        for (int u = a; u < e; ++u) need(share_of(total, shares, u) == w, "share_of");
      }
    }
  const int huge = 0x7FFFFFF0;
  need(share_of(huge, 592, share_start(huge, 592, 300)) == 300, "large shares");
  need(share_start(huge, 592, 592) == huge && share_of(huge, 592, huge - 1) == 591, "large share ends");
  // lengths are cut to the table
  bool bad;
  need(paged_clamp_len(0, 3, 4, &bad) == 0 && !bad, "0");
  need(paged_clamp_len(48, 3, 4, &bad) == 48 && !bad, "48");
  need(paged_clamp_len(49, 3, 4, &bad) == 48 && bad, "49");
  need(paged_clamp_len(-1, 3, 4, &bad) == 0 && bad, "-1");
  need(paged_clamp_len(0x7FFFFFFF, 3, 4, &bad) == 48 && bad, "max");
  need(paged_clamp_len(static_cast<int>(0x80000000u), 3, 4, &bad) == 0 && bad, "min");
  // offsets pass 32 bits
  const int64_t page = int64_t{32} * 128 * 128;
  need(paged_offset(1 << 20, page, 31, 127, 7, 7) == (int64_t{1} << 20) * page + (int64_t{31} * 128 + 127) * 128, "offset");
  need(paged_offset(3, 1000000, 2, 5, 4, 6) == 3000000 + (2 * 16 + 5) * 64, "small offset");
  // packed rows of a sequence stay within the tensor whatever the boundaries say
  const int cu[] = {-5, 3, 2, 900, 50, 50, 0x7FFFFFFF, static_cast<int>(0x80000000u), 7};
  for (int b = 0; b < 8; ++b) {
    int lo, hi;
    packed_range(cu, b, 60, &lo, &hi);
    need(0 <= lo && lo <= hi && hi <= 60, "packed range");
  }
  int lo, hi;
  const int good[] = {0, 4, 4, 60};
  packed_range(good, 0, 60, &lo, &hi);
  need(lo == 0 && hi == 4, "packed 0");
  packed_range(good, 1, 60, &lo, &hi);
  need(lo == 4 && hi == 4, "packed 1");
  packed_range(good, 2, 60, &lo, &hi);
  need(lo == 4 && hi == 60, "packed 2");
  need(visible_keys(10, 3, 0) == 8 && visible_keys(10, 3, 2) == 10, "visible");
  need(visible_keys(1, 3, 0) == 0 && visible_keys(1, 3, 1) == 0 && visible_keys(1, 3, 2) == 1, "none visible");
  for (int group = 1; group <= 64; ++group)
    for (int row = 0; row < 128; ++row)
      need(row_token(row, (65536u + group - 1) / group) == row / group, "row token");
  std::printf("%ld\n", checks);
  return 0;
}
"""


def _have_nvcc() -> bool:
    try:
        _build._nvcc()
        return True
    except RuntimeError:
        return False


@pytest.mark.skipif(not _have_nvcc(), reason="needs nvcc")
def test_index_arithmetic(tmp_path):
    src = tmp_path / "ix.cu"
    src.write_text(INDEX_PROGRAM)
    exe = tmp_path / "ix"
    subprocess.check_call([_build._nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2",
                           f"-I{_build.CSRC_DIR}", f"-I{_build.INCLUDE_DIR}", str(src), "-o", str(exe)])
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert int(out.stdout) > 10_000_000


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layouts_match_c(tmp_path):
    src = tmp_path / "sz.c"
    src.write_text(
        '#include <stdio.h>\n#include <stddef.h>\n#include "abft_b200.h"\n'
        "int main(void){printf(\"%zu %zu %zu %zu %zu %zu %zu %zu\\n\", sizeof(abft_paged_kv), "
        "offsetof(abft_paged_kv, dtype), sizeof(abft_kv_append_args), offsetof(abft_kv_append_args, rope), "
        "offsetof(abft_kv_append_args, heads), sizeof(abft_paged_attn_args), "
        "offsetof(abft_paged_attn_args, scale), offsetof(abft_paged_attn_args, num_splits));return 0;}\n")
    exe = tmp_path / "sz"
    subprocess.check_call(["gcc", f"-I{_build.INCLUDE_DIR}", str(src), "-o", str(exe)])
    vals = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    assert vals == [ctypes.sizeof(N.PagedKv), N.PagedKv.dtype.offset, ctypes.sizeof(N.KvAppendArgs),
                    N.KvAppendArgs.rope.offset, N.KvAppendArgs.heads.offset, ctypes.sizeof(N.PagedAttnArgs),
                    N.PagedAttnArgs.scale.offset, N.PagedAttnArgs.num_splits.offset]


def _kv():
    kv = N.PagedKv()
    kv.k_pages, kv.v_pages, kv.page_table, kv.seq_lens = 0x10000, 0x20000, 0x30000, 0x40000
    kv.num_pages, kv.page_size, kv.kv_heads, kv.head_dim = 8, 16, 4, 128
    kv.k_page_stride = kv.v_page_stride = 4 * 16 * 128
    kv.batch, kv.max_pages, kv.table_stride = 2, 3, 3
    return kv


BAD_KV = [
    ("batch", -1, -1), ("num_pages", -1, -1), ("max_pages", -1, -1), ("kv_heads", 0, -1), ("dtype", 2, -3),
    ("dtype", 9, -1), ("head_dim", 96, -3), ("page_size", 8, -3), ("page_size", 48, -3), ("k_pages", None, -1),
    ("v_pages", None, -1), ("page_table", None, -1), ("seq_lens", None, -1), ("max_pages", 0, -1), ("num_pages", 0, -1),
    ("batch", 70000, -3), ("table_stride", 2, -1), ("max_pages", 1 << 27, -3), ("k_page_stride", 4 * 16 * 128 - 8, -1),
    ("v_page_stride", 0, -1), ("k_page_stride", 4 * 16 * 128 + 4, -2), ("k_pages", 0x10008, -2), ("v_pages", 0x20002, -2),
]


@pytest.mark.parametrize("field,value,code", BAD_KV)
def test_cache_refusals(field, value, code):
    """The same cache checks stand before each operator."""
    L = N.lib()
    kv = _kv()
    setattr(kv, field, value)
    a = N.KvAppendArgs()
    a.kv, a.k, a.v, a.tokens = kv, 0x50000, 0x60000, kv.batch
    assert L.abft_kv_append(ctypes.byref(a), None) == code
    d = N.PagedAttnArgs()
    d.kv, d.q, d.out, d.heads, d.tokens, d.scale = kv, 0x50000, 0x60000, 28, kv.batch, 1.0
    assert L.abft_paged_decode(ctypes.byref(d), None) == code
    assert L.abft_paged_decode_workspace_bytes(ctypes.byref(d)) == 0
    d.cu_seqlens = 0x70000
    assert L.abft_paged_prefill(ctypes.byref(d), None) == code
    assert L.abft_paged_prefill_workspace_bytes(ctypes.byref(d)) == 0


def test_append_refusals():
    L = N.lib()

    def call(**over):
        a = N.KvAppendArgs()
        a.kv, a.q, a.k, a.v, a.q_out, a.tokens, a.heads = _kv(), 0x50000, 0x60000, 0x70000, 0x80000, 2, 28
        for k, v in over.items():
            setattr(a, k, v)
        return L.abft_kv_append(ctypes.byref(a), None)

    assert L.abft_kv_append(None, None) == -1
    for over, code in [({"tokens": -1}, -1), ({"heads": -4}, -1), ({"heads": 27}, -1), ({"heads": 4 * 65}, -3),
                       ({"tokens": 3}, -1), ({"tokens": 1 << 31, "cu_seqlens": 0x90000}, -3), ({"k": None}, -1),
                       ({"v": None}, -1), ({"q": None}, -1), ({"q_out": None}, -1), ({"max_positions": -1}, -1),
                       ({"k": 0x60004}, -2), ({"v": 0x70008}, -2), ({"q": 0x50002}, -2), ({"q_out": 0x80008}, -2),
                       ({"rope": 0x90008}, -2), ({"k_token_stride": 4}, -2), ({"v_head_stride": 9}, -2),
                       ({"q_head_stride": 1}, -2), ({"o_token_stride": 12}, -2)]:
        assert call(**over) == code, over
    assert call(tokens=0, cu_seqlens=0x90000) == 0  # nothing to do
    if not torch.cuda.is_available():
        assert call() == -6


def test_attention_refusals():
    L = N.lib()

    def call(fn, **over):
        a = N.PagedAttnArgs()
        a.kv, a.q, a.out, a.tokens, a.heads, a.scale, a.cu_seqlens = _kv(), 0x50000, 0x60000, 2, 28, 0.1, 0x70000
        a.num_sms = 148
        for k, v in over.items():
            setattr(a, k, v)
        return fn(ctypes.byref(a), None)

    for fn in (L.abft_paged_decode, L.abft_paged_prefill):
        assert fn(None, None) == -1
        for over, code in [({"tokens": -1}, -1), ({"num_splits": -1}, -1), ({"num_sms": -1}, -1), ({"num_sms": 5000}, -3),
                           ({"scale": float("inf")}, -1), ({"scale": float("nan")}, -1), ({"heads": 0}, -1),
                           ({"heads": 27}, -1), ({"heads": 4 * 65}, -3), ({"q": None}, -1), ({"out": None}, -1),
                           ({"q": 0x50008}, -2), ({"out": 0x60004}, -2), ({"q_token_stride": 4}, -2),
                           ({"o_head_stride": 2}, -2)]:
            assert call(fn, **over) == code, over
        if not torch.cuda.is_available():
            assert call(fn) == -6
    assert call(L.abft_paged_decode, tokens=1) == -1  # one row per sequence
    kv = _kv()
    kv.max_pages = kv.table_stride = 1 << 26
    kv.batch = 16
    assert call(L.abft_paged_decode, kv=kv, tokens=16) == -3  # 2^31 tiles
    assert call(L.abft_paged_prefill, cu_seqlens=None) == -1
    assert call(L.abft_paged_prefill, tokens=0) == 0
    assert call(L.abft_paged_prefill, tokens=1 << 30) == -3


def test_workspace_sizes():
    a = N.PagedAttnArgs()
    a.kv, a.q, a.out, a.tokens, a.heads, a.scale, a.num_sms = _kv(), 0x50000, 0x60000, 2, 28, 0.1, 148
    a.cu_seqlens = 0x70000
    # decode: 2 sequences x 4 kv heads, 8 segments of 2 tiles of 32 slots: a CTA each and no scratch
    assert N.lib().abft_paged_decode_workspace_bytes(ctypes.byref(a)) == 0
    cta = 2 * 8 * (128 * 4 + 8) + 16  # two pieces of 8 heads and a record
    a.num_sms = 3
    assert N.lib().abft_paged_decode_workspace_bytes(ctypes.byref(a)) == 3 * cta
    a.num_sms = 148
    a.kv.max_pages = a.kv.table_stride = 64  # 1,024 slots: a cluster of 8 CTAs each and no scratch
    assert N.lib().abft_paged_decode_workspace_bytes(ctypes.byref(a)) == 0
    a.kv.max_pages = a.kv.table_stride = 130  # 65 tiles each, shared out: 520 tiles for 130 CTAs' warps
    assert N.lib().abft_paged_decode_workspace_bytes(ctypes.byref(a)) == 130 * cta
    a.kv.max_pages = a.kv.table_stride = 640  # 144 SMs, 18 for each segment
    assert N.lib().abft_paged_decode_workspace_bytes(ctypes.byref(a)) == 144 * cta
    a.kv.max_pages = a.kv.table_stride = 3
    a.num_splits = 1
    assert N.lib().abft_paged_prefill_workspace_bytes(ctypes.byref(a)) == 0
    a.kv.max_pages = a.kv.table_stride = 64  # 8 steps of 128 slots
    a.num_splits = 2
    assert N.lib().abft_paged_prefill_workspace_bytes(ctypes.byref(a)) == 2 * 28 * 2 * (128 * 4 + 8)


def test_python_refusals_without_gpu():
    ok = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError):
        PagedKVCache(None, ok, table, lens)
    for k, v in [(ok[0], ok[0]), (ok.float(), ok.float()), (ok, ok[:3]), (ok, ok.half()),
                 (ok[:, :, :8], ok[:, :, :8]), (ok[..., :32], ok[..., :32]), (ok[:, :0], ok[:, :0])]:
        with pytest.raises(ValueError):
            PagedKVCache(k, v, table, lens)
    with pytest.raises(ValueError, match="no CPU path"):
        PagedKVCache(ok, ok.clone(), table, lens)


def test_rope_table_is_exact_far_out():
    t = rope_table(1 << 18, 64, theta=1e4)
    assert t.shape == (1 << 18, 32, 2) and t.dtype == torch.float32
    p = (1 << 18) - 1
    ang = p * 1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert torch.equal(t[p, :, 0], ang.cos().float()) and torch.equal(t[p, :, 1], ang.sin().float())
    with pytest.raises(ValueError):
        rope_table(4, 7)
    with pytest.raises(ValueError):
        rope_table(-1, 8)


def test_host_extension_takes_only_its_struct_and_passes_on_the_rest():
    from vla_abft_estimate_b200.paged import _host

    Calls = _host().Calls
    with pytest.raises(ValueError):
        Calls(bytes(ctypes.sizeof(N.PagedKv) - 8), 0, 0, 0, 0, 0, 0)
    with pytest.raises(TypeError):
        Calls(bytes(ctypes.sizeof(N.PagedKv)), 0)
    c = Calls(bytes(_kv()), 0, 0, 0, 0, 0, 0)
    t = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    assert c.append(t, t, t, None, None, None) is None
    assert c.append(t) is None
    assert c.attend(False, t, None, None, None, 0, 0) is None
    assert c.attend(True, 3, None, "x", None, 0, 0) is None
