"""Packed boundaries that do not start at 0, fall, or pass the rows: append and
prefill skip what they do not describe, and the status tells."""
import pytest
import torch

from vla_abft_estimate_b200.paged import PagedKVCache, rope_table

from .paged_reference import Pool, attention, rotated
from .test_gpu_paged import BF16, bits, close

pytestmark = pytest.mark.gpu

TOTAL = (40, 90, 30)
ROWS = 12
# boundaries, and the (sequence, position) of each of the 12 rows: None where
# the row is left as it was, "unclear" where falling boundaries give it to more
# than one sequence (not appended, its attention not defined)
CASES = {
    "from 5": ((5, 8, 10, 12), [None] * 5 + [(0, 37), (0, 38), (0, 39), (1, 88), (1, 89), (2, 28), (2, 29)]),
    "slice of a longer list": ((9, 12, 16, 20), [None] * 9 + [(0, 37), (0, 38), (0, 39)]),
    "passes the rows": ((0, 4, 10, 20), [(0, 36 + i) for i in range(4)] + [(1, 84 + i) for i in range(6)] + [None] * 2),
    "starts behind the rows": ((0, 12, 13, 14), [(0, 28 + i) for i in range(12)]),
    "below 0": ((-3, 4, 10, 12), [None] * 4 + [(1, 84 + i) for i in range(6)] + [(2, 28), (2, 29)]),
    "falls": ((0, 6, 3, 12), [(0, 34), (0, 35), (0, 36)] + ["unclear"] * 3 + [(2, 24 + i) for i in range(6)]),
    "far outside": ((0, 3, -2147483648, 2147483647), ["unclear"] * 3 + [None] * 9),
    "all outside": ((-2147483648, -1, 13, 2147483647), [None] * 12),
}


def _setup(dev, case):
    bounds, rows = CASES[case]
    pool = Pool(TOTAL, 2, 16, 64, BF16, seed=31)
    cache = pool.device_cache(dev, PagedKVCache)
    return pool, cache, torch.tensor(bounds, dtype=torch.int32, device=dev), rows


@pytest.mark.parametrize("case", CASES)
def test_append_skips_rows_of_no_sequence(cuda_device, case):
    dev = cuda_device
    pool, cache, cu, rows = _setup(dev, case)
    want_k, want_v = bits(cache.k_pages).clone(), bits(cache.v_pages).clone()
    g = torch.Generator().manual_seed(32)
    q, k, v = (torch.randn(ROWS, h, 64, generator=g).to(BF16) for h in (4, 2, 2))
    out = torch.full((ROWS, 4, 64), 7.0, dtype=BF16, device=dev)
    cache.append(q.to(dev), k.to(dev), v.to(dev), rope_table(100, 64, device=dev), cu_seqlens=cu, q_out=out)
    kept = [i for i, r in enumerate(rows) if r is None or r == "unclear"]
    assert (out[kept] == 7.0).all()
    live = [i for i in range(ROWS) if i not in kept]
    at = torch.tensor([rows[i] for i in live], dtype=torch.int64).view(-1, 2)
    page, slot = pool.table[at[:, 0], at[:, 1] // 16].long(), at[:, 1] % 16
    if live:
        close(out[live], *rotated(q[live], at[:, 1]))
        close(cache.k_pages.cpu()[page, :, slot], *rotated(k[live], at[:, 1]))
    have_k, have_v = bits(cache.k_pages).clone(), bits(cache.v_pages).clone()
    assert torch.equal(have_v[page, :, slot], bits(v[live]))
    for x in (want_k, want_v, have_k, have_v):
        x[page, :, slot] = 0
    assert torch.equal(have_k, want_k) and torch.equal(have_v, want_v), "a slot of no appended row changed"
    with pytest.raises(ValueError, match="cu_seqlens"):
        cache.check_status()
    cache.check_status()


@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("case", CASES)
def test_prefill_leaves_rows_of_no_sequence(cuda_device, case, splits):
    dev = cuda_device
    pool, cache, cu, rows = _setup(dev, case)
    q = torch.randn(ROWS, 4, 64, generator=torch.Generator().manual_seed(33)).to(BF16)
    out = torch.full((ROWS, 4, 64), 7.0, dtype=BF16, device=dev)
    cache.prefill(q.to(dev), cu, out=out, num_splits=splits)
    left = [i for i, r in enumerate(rows) if r is None]
    assert (out[left] == 7.0).all()
    live = [i for i, r in enumerate(rows) if r is not None and r != "unclear"]
    if live:
        close(out[live], *attention(pool, q[live], [(rows[i][0], rows[i][1] + 1) for i in live]))
    with pytest.raises(ValueError, match="cu_seqlens"):
        cache.check_status()
    cache.check_status()


@pytest.mark.parametrize("batch", [1, 31, 33, 200])
def test_boundaries_of_any_batch_are_looked_at(cuda_device, batch):
    """The last sequence's end alone is wrong; then all are right again."""
    dev = cuda_device
    cache = Pool([3] * batch, 1, 16, 64, BF16).device_cache(dev, PagedKVCache)
    cu = torch.arange(batch + 1, dtype=torch.int32, device=dev)
    x = torch.zeros(batch, 1, 64, dtype=BF16, device=dev)
    for call in (lambda: cache.append(None, x, x, cu_seqlens=cu), lambda: cache.prefill(x, cu)):
        call()
        cache.check_status()
        cu[batch] += 1
        call()
        with pytest.raises(ValueError, match="cu_seqlens"):
            cache.check_status()
        cu[batch] -= 1
