"""Drafted trees on the host: struct layouts, refusals of the C entries, the extension."""
import ctypes
import shutil
import subprocess

import pytest
import torch

from vla_abft_estimate_b200 import _build
from vla_abft_estimate_b200 import _native as N

from .test_paged_host import BAD_KV, _have_nvcc, _kv

STRUCTS = {"abft_kv_append_at_args": (N.KvAppendAtArgs, ("positions", "axes", "sections")),
           "abft_paged_tree_args": (N.PagedTreeArgs, ("parents",)),
           "abft_draft_accept_args": (N.DraftAcceptArgs, ("next", "tokens", "id_bytes")),
           "abft_kv_keep_args": (N.KvKeepArgs, ("pools", "lens_out", "layers")),
           "abft_kv_fork_args": (N.KvForkArgs, ("pools", "pages", "layers"))}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layouts_match_c(tmp_path):
    src, exe = tmp_path / "sz.c", tmp_path / "sz"
    lines = [f'printf("%zu ", sizeof({c}));' + "".join(f'printf("%zu ", offsetof({c}, {f}));' for f in fields)
             for c, (_, fields) in STRUCTS.items()]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "abft_b200.h"\nint main(void){' + "\n".join(lines)
                   + 'printf("%d %u %u", ABFT_MOST_AXES, ABFT_PAGED_BAD_DRAFT, ABFT_PAGED_BAD_FORK);return 0;}\n')
    subprocess.check_call(["gcc", f"-I{_build.INCLUDE_DIR}", str(src), "-o", str(exe)])
    want = []
    for t, fields in STRUCTS.values():
        want += [ctypes.sizeof(t)] + [getattr(t, f).offset for f in fields]
    want += [N.MOST_AXES, N.PAGED_BAD_DRAFT, N.PAGED_BAD_FORK]
    assert [int(x) for x in subprocess.check_output([str(exe)]).split()] == want


WORDS_PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "paged_tree.cuh"
using namespace abft;
int main() {
  long checks = 0;
  unsigned seed = 1;
  auto rnd = [&]() { return (seed = seed * 1664525u + 1013904223u) >> 8; };
  const int sizes[] = {1, 2, 31, 32, 33, 63, 64, 65, 150, 400};
  for (int n : sizes)
    for (int kind = 0; kind < 4; ++kind) {
      int up[400];
      for (int i = 0; i < n; ++i) {
        up[i] = kind == 0 ? i - 1 : kind == 1 ? (i ? 0 : -1) : i ? static_cast<int>(rnd() % (i + 1)) - 1 : -1;
        if (kind == 3 && rnd() % 8 == 0) up[i] = static_cast<int>(rnd()) - (1 << 23);  // bad ones among them
        if (kind == 3 && rnd() % 8 == 0) up[i] = i;
      }
      for (int before = -n; before < 200; before += 7)  // slots before the drafted ones (below 0: more rows than tokens)
        for (int step = 0; step * 64 < before + n; ++step)
          for (int own = before < 0 ? -before : 0; own < n; ++own) {
            uint32_t w[2];
            tree_words(up, own, before - step * 64, w);
            unsigned char see[700] = {0};
            for (int i = 0; i < before; ++i) see[i] = 1;
            for (int i = own; i >= 0;) {
              if (before + i >= 0) see[before + i] = 1;
              i = up[i] < i ? up[i] : -1;
            }
            for (int k = 0; k < 64; ++k) {
              if ((w[k / 32] >> (k % 32) & 1u) != see[step * 64 + k]) {
                std::printf("n %d kind %d before %d step %d own %d key %d\n", n, kind, before, step, own, k);
                return 1;
              }
              ++checks;
            }
          }
    }
  std::printf("%ld\n", checks);
  return 0;
}
"""


@pytest.mark.skipif(not _have_nvcc(), reason="needs nvcc")
def test_what_a_row_of_a_tree_sees(tmp_path):
    """The mask words on the host, against the way up row by row."""
    src, exe = tmp_path / "words.cu", tmp_path / "words"
    src.write_text(WORDS_PROGRAM)
    subprocess.check_call([_build._nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2",
                           f"-I{_build.CSRC_DIR}", f"-I{_build.INCLUDE_DIR}", str(src), "-o", str(exe)])
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert int(out.stdout) > 10_000_000


def _append(kv):
    a = N.KvAppendAtArgs()
    x = a.append
    x.kv, x.q, x.k, x.v, x.q_out, x.tokens, x.heads, x.rope, x.max_positions = \
        kv, 0x50000, 0x60000, 0x70000, 0x80000, 2, 28, 0x90000, 100
    a.positions, a.axes, a.sections[0] = 0xA0000, 1, 64
    return a


def _tree(kv):
    a = N.PagedTreeArgs()
    x = a.attn
    x.kv, x.q, x.out, x.tokens, x.heads, x.scale, x.cu_seqlens, x.num_sms = kv, 0x50000, 0x60000, 2, 28, 0.1, 0x70000, 148
    x.q_token_stride, x.q_head_stride, x.o_token_stride, x.o_head_stride = 28 * 128, 128, 28 * 128, 128
    a.parents = 0x80000
    return a


POOLS = (ctypes.c_void_p * 1024)(*range(0x100000, 0x100000 + 1024 * 64, 64))  # addresses that nobody follows


def _keep(kv):
    a = N.KvKeepArgs()
    a.kv, a.pools, a.cu_seqlens, a.kept, a.counts, a.lens_out, a.tokens, a.layers = \
        kv, ctypes.addressof(POOLS), 0x60000, 0x70000, 0x80000, kv.seq_lens, 8, 28
    return a


def _fork(kv):
    a = N.KvForkArgs()
    a.kv, a.pools, a.src, a.dst, a.pages, a.pairs, a.layers = \
        kv, ctypes.addressof(POOLS), 0x60000, 0x70000, 0x80000, 3, 28
    return a


def _accept():
    a = N.DraftAcceptArgs()
    a.cu_seqlens, a.parents, a.ids, a.answers, a.kept, a.counts, a.next = \
        0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0x60000, 0x70000
    a.tokens, a.batch, a.id_bytes = 8, 2, 8
    return a


def _call(name, a):
    return getattr(N.lib(), name)(ctypes.byref(a), None)


MAKE = {"abft_kv_append_at": _append, "abft_paged_tree": _tree, "abft_kv_keep": _keep, "abft_kv_fork": _fork}


@pytest.mark.parametrize("name", MAKE)
@pytest.mark.parametrize("field,value,code", BAD_KV)
def test_cache_refusals(name, field, value, code):
    kv = _kv()
    setattr(kv, field, value)
    a = MAKE[name](kv)
    if field == "batch" and value > 0 and name in ("abft_kv_append_at", "abft_paged_tree"):
        (a.append if name == "abft_kv_append_at" else a.attn).tokens = value
    assert _call(name, a) == code
    if name == "abft_paged_tree":
        assert N.lib().abft_paged_tree_workspace_bytes(ctypes.byref(a)) == 0


@pytest.mark.parametrize("name", [*MAKE, "abft_draft_accept"])
def test_no_arguments_and_no_device(name):
    assert getattr(N.lib(), name)(None, None) == -1
    if not torch.cuda.is_available():
        assert _call(name, _accept() if name == "abft_draft_accept" else MAKE[name](_kv())) == -6


def _set(a, over):
    for k, v in over.items():
        x = a
        *path, last = k.split(".")
        for p in path:
            x = getattr(x, p)
        if isinstance(v, tuple):
            for i, y in enumerate(v):
                getattr(x, last)[i] = y
        else:
            setattr(x, last, v)
    return a


def test_append_refusals():
    for over, code in [({"axes": 0}, -1), ({"axes": -3}, -1), ({"axes": 5}, -3), ({"sections": (63,)}, -1),
                       ({"sections": (65, -1), "axes": 2}, -1), ({"axes": 2}, 0), ({"sections": (32, 32), "axes": 2}, 0),
                       ({"sections": (2 ** 31 - 1, 2 ** 31 - 1, 66), "axes": 3}, -1), ({"append.rope": None}, -1),
                       ({"positions": None}, -1), ({"positions": 0xA0002}, -2), ({"append.max_positions": 0}, -1),
                       ({"position_stride": -2}, -1), ({"append.k": 0x60004}, -2), ({"append.heads": 27}, -1),
                       ({"append.tokens": 3}, -1)]:
        if code == 0 and torch.cuda.is_available():
            continue  # would be launched
        assert _call("abft_kv_append_at", _set(_append(_kv()), over)) == (code or -6), over
    assert _call("abft_kv_append_at", _set(_append(_kv()), {"append.tokens": 0, "append.cu_seqlens": 0x90000})) == 0


def test_tree_refusals():
    for over, code in [({"parents": None}, -1), ({"attn.cu_seqlens": None}, -1), ({"attn.tokens": -1}, -1),
                       ({"attn.num_splits": -1}, -1), ({"attn.num_sms": 5000}, -3), ({"attn.scale": float("nan")}, -1),
                       ({"attn.heads": 4 * 65}, -3), ({"attn.q": 0x50008}, -2), ({"attn.q_head_stride": 0}, -1),
                       ({"attn.q_token_stride": 0}, -1), ({"attn.q_token_stride": -8}, -1), ({"attn.o_head_stride": 2}, -2),
                       ({"attn.tokens": 1 << 30}, -3)]:
        assert _call("abft_paged_tree", _set(_tree(_kv()), over)) == code, over
    assert _call("abft_paged_tree", _set(_tree(_kv()), {"attn.tokens": 0})) == 0
    assert N.lib().abft_paged_tree_workspace_bytes(None) == 0


def test_accept_refusals():
    for over, code in [({"batch": -1}, -1), ({"tokens": -1}, -1), ({"id_bytes": 2}, -1), ({"batch": 70000}, -3),
                       ({"tokens": 1 << 30}, -3), ({"cu_seqlens": None}, -1), ({"counts": None}, -1), ({"next": None}, -1),
                       ({"parents": None}, -1), ({"ids": None}, -1), ({"answers": None}, -1), ({"kept": None}, -1),
                       ({"ids": 0x30004}, -2), ({"next": 0x70004}, -2), ({"answers": 0x40002, "id_bytes": 4}, -2)]:
        assert _call("abft_draft_accept", _set(_accept(), over)) == code, over
    assert _call("abft_draft_accept", _set(_accept(), {"batch": 0, "tokens": 0})) == 0


OFF, NONE = (ctypes.c_void_p * 56)(*POOLS[:56]), (ctypes.c_void_p * 56)(*POOLS[:56])
OFF[55], NONE[55] = 0x100008, None


def test_keep_refusals():
    lens = _kv().seq_lens
    for over, code in [({"layers": 0}, -1), ({"layers": 513}, -3), ({"pools": None}, -1), ({"pools": ctypes.addressof(OFF)}, -2),
                       ({"pools": ctypes.addressof(NONE)}, -1),
                       ({"tokens": -1}, -1), ({"tokens": 1 << 30}, -3), ({"cu_seqlens": None}, -1), ({"counts": None}, -1),
                       ({"lens_out": None}, -1), ({"kept": None}, -1), ({"lens_out": lens + 4}, -1), ({"lens_out": lens - 4}, -1)]:
        assert _call("abft_kv_keep", _set(_keep(_kv()), over)) == code, over


def test_fork_refusals():
    for over, code in [({"layers": 0}, -1), ({"layers": 513}, -3), ({"pools": None}, -1), ({"pools": ctypes.addressof(OFF)}, -2),
                       ({"pools": ctypes.addressof(NONE)}, -1),
                       ({"pairs": -1}, -1), ({"pairs": 70000}, -3), ({"src": None}, -1), ({"dst": None}, -1),
                       ({"pages": None}, -1)]:
        assert _call("abft_kv_fork", _set(_fork(_kv()), over)) == code, over
    assert _call("abft_kv_fork", _set(_fork(_kv()), {"pairs": 0})) == 0


def test_the_extension_takes_only_its_structs_and_passes_on_the_rest():
    from vla_abft_estimate_b200.paged import _host

    host = _host()
    c = host.Calls(bytes(_kv()), 0, 0, 0, 0, 0, 0)
    with pytest.raises(TypeError):
        c.drafts(1)
    with pytest.raises(TypeError):
        c.drafts("a", 1, 2)
    c.drafts(0, 0, 0)
    t, cu, up = torch.zeros(2, 4, 128, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    assert c.append(t, t, t, None, None, None, up[None], (64,)) is None
    assert c.tree(t, cu, up, None, None, 0, 0) is None
    assert c.tree(t) is None
    x = torch.zeros(3)
    with pytest.raises(ValueError):
        host.Layers(b"short", 0, bytes(16), 0, 0, 0, (x, x), x, x)
    with pytest.raises(ValueError):
        host.Layers(bytes(_kv()), 0, bytes(16), 0, 0, 0, (x, 3), x, x)
    with pytest.raises(ValueError):
        host.Layers(bytes(_kv()), 0, bytes(24), 0, 0, 0, (x, x), x, x)
    with pytest.raises(TypeError):
        host.Layers(bytes(_kv()), 0, 1)
    many = host.Layers(bytes(_kv()), 0, bytes(16), 0, 0, 0, (x, x), x, x)
    assert many.accept(cu, up, up, up) is None and many.keep(cu, up, up, up) is None and many.fork(up, up, up) is None
    assert many.accept() is None and many.keep(1) is None and many.fork(1, 2, 3, 4) is None
