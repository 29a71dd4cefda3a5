"""Arrays that a call writes and reads: refusals on the host."""

import pytest
import torch

from .test_draft_host import _accept, _call, _fork, _keep, _set
from .test_paged_host import _kv

HERE = -6  # in order, as far as the host can tell: what a host without a GPU answers


@pytest.mark.parametrize("field", ["cu_seqlens", "kept", "page_table"])
def test_keep_refuses_lengths_over_what_others_read(field):
    a = _keep(_kv())
    at = a.kv.page_table if field == "page_table" else getattr(a, field)
    size = 4 * {"cu_seqlens": a.kv.batch + 1, "kept": a.tokens,
                "page_table": (a.kv.batch - 1) * a.kv.table_stride + a.kv.max_pages}[field]
    for over in (at, at + 4, at - 4, at + size - 4, at - 4 * a.kv.batch + 4):
        assert _call("abft_kv_keep", _set(_keep(_kv()), {"lens_out": over})) == -1, over
    if not torch.cuda.is_available():
        for beside in (at + size, at - 4 * a.kv.batch):
            assert _call("abft_kv_keep", _set(_keep(_kv()), {"lens_out": beside})) == HERE


def test_keep_takes_the_counts_or_refuses_a_part_of_them():
    counts = _keep(_kv()).counts
    for over in (counts + 4, counts - 4):
        assert _call("abft_kv_keep", _set(_keep(_kv()), {"lens_out": over})) == -1
    if not torch.cuda.is_available():
        assert _call("abft_kv_keep", _set(_keep(_kv()), {"lens_out": counts})) == HERE


@pytest.mark.parametrize("field", ["src", "dst", "pages"])
def test_fork_refuses_lists_within_what_it_writes(field):
    kv = _kv()
    table = 4 * ((kv.batch - 1) * kv.table_stride + kv.max_pages)
    for over in (kv.page_table, kv.page_table + table - 4, kv.page_table - 8, kv.seq_lens, kv.seq_lens + 4 * kv.batch - 4,
                 kv.seq_lens - 8):
        assert _call("abft_kv_fork", _set(_fork(_kv()), {field: over})) == -1, over
    if not torch.cuda.is_available():
        for beside in (kv.page_table + table, kv.page_table - 12, kv.seq_lens + 4 * kv.batch, kv.seq_lens - 12):
            assert _call("abft_kv_fork", _set(_fork(_kv()), {field: beside})) == HERE, beside
        assert _call("abft_kv_fork", _set(_fork(_kv()), {"src": 0x60000, "dst": 0x60000, "pages": 0x60000})) == HERE


def test_accept_refuses_results_over_what_is_read():
    a = _accept()
    read = {"cu_seqlens": 4 * (a.batch + 1), "parents": 4 * a.tokens, "ids": 8 * a.tokens, "answers": 8 * a.tokens}
    written = {"kept": 4 * a.tokens, "counts": 4 * a.batch, "next": 8 * a.batch}
    for result, bytes_ in written.items():
        for field, size in {**read, **written}.items():
            if field == result:
                continue
            at = getattr(a, field)
            for over in (at, at + (size - 1) // 8 * 8, at - (bytes_ - 1) // 8 * 8):  # multiples of 8, as next has to be
                assert _call("abft_draft_accept", _set(_accept(), {result: over})) == -1, (result, field)
            if not torch.cuda.is_available():
                for beside in (at + (size + 7) // 8 * 8, at - bytes_):
                    assert _call("abft_draft_accept", _set(_accept(), {result: beside})) == HERE, (result, field)


@pytest.mark.parametrize("entries", [1, 2, 3, 7])
def test_what_lies_between_a_tables_rows_is_not_the_tables(entries):
    """Rows of 3 entries, 8 apart: every place of a list of some entries, against the sets of entries."""
    kv = _kv()
    kv.batch, kv.max_pages, kv.table_stride = 5, 3, 8
    rows = {r * 8 + c for r in range(kv.batch) for c in range(kv.max_pages)}
    for first in range(-9, 45):
        a = _set(_fork(kv), {"pages": kv.page_table + 4 * first, "pairs": entries})
        want = -1 if rows & set(range(first, first + entries)) else HERE
        if want == -1 or not torch.cuda.is_available():
            assert _call("abft_kv_fork", a) == want, first
    kv.batch, kv.table_stride = 1, 0
    for first, want in ((-1 - entries, HERE), (-entries, HERE), (1 - entries, -1), (0, -1), (2, -1), (3, HERE)):
        if want == -1 or not torch.cuda.is_available():
            assert _call("abft_kv_fork", _set(_fork(kv), {"pages": kv.page_table + 4 * first, "pairs": entries})) == want, first
