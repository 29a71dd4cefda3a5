"""Small weights of long caches: many keys far below one that has nearly all the
weight, whose value is 0, so that the result is what the small ones carry."""
import pytest
import torch

from vla_abft_estimate_b200.paged import PagedKVCache

from .paged_reference import Pool, attention
from .test_gpu_paged import BF16, F16, close

pytestmark = pytest.mark.gpu


def sink(lens, at, d, dtype, gap, kv_heads=1):
    """Key `at` scores `gap` (scale 1, q all 0.5) and has value 0, all others
    score 0 and have value 64."""
    pool = Pool(lens, kv_heads, 64, d, dtype)
    for b, n in enumerate(lens):
        key, value = torch.zeros(n, d), torch.full((n, d), 64.0)
        if at < n:
            key[at], value[at] = gap / (0.5 * d), 0.0
        held = pool.table[b, : -(-n // 64)].long()
        for pages, rows in ((pool.k, key), (pool.v, value)):
            padded = torch.full((len(held) * 64, d), float("nan"))
            padded[:n] = rows
            pages[held] = padded.view(len(held), 1, 64, d).to(dtype).expand(-1, kv_heads, -1, -1)
    return pool


# 2^-25.3 of the greatest weight, times 60,000 keys: 1.4e-3 of the sum, and all of
# the result. 2^-20 for fewer.
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,at,gap", [(60_000, 0, 17.54), (60_000, 59_990, 17.54), (400, 100, 13.9)])
def test_small_weights_are_kept(cuda_device, n, at, gap, d, dtype):
    dev = cuda_device
    pool = sink([n, 70], at, d, dtype, gap)
    cache = pool.device_cache(dev, PagedKVCache)
    q = torch.full((2, 7, d), 0.5, dtype=dtype)
    want, tol = attention(pool, q, [(0, n), (1, 70)], 1.0)
    assert want[0].abs().min() > 0.02
    for sms in (0, 3):
        close(cache.decode(q.to(dev), scale=1.0, num_sms=sms), want, tol)
    new = (5, 1)
    q = torch.full((6, 7, d), 0.5, dtype=dtype)
    cu = torch.tensor([0, 5, 6], dtype=torch.int32, device=dev)
    want, tol = attention(pool, q, [(0, n - 4 + i) for i in range(5)] + [(1, 70)], 1.0)
    for splits in (0, 1, 3):
        close(cache.prefill(q.to(dev), cu, scale=1.0, num_splits=splits), want, tol)
    q = torch.full((300, 40, d), 0.5, dtype=dtype)  # more rows than SMs have tiles: two tiles an item
    cu = torch.tensor([0, 299, 300], dtype=torch.int32, device=dev)
    got = cache.prefill(q.to(dev), cu, scale=1.0)
    rows = [0, 100, 298, 299]
    want, tol = attention(pool, q[rows], [(0, n - 298), (0, n - 198), (0, n), (1, 70)], 1.0)
    close(got[rows], want, tol)
    cache.check_status()


@pytest.mark.parametrize("dtype,lag", [(BF16, 8), (F16, 5)])
@pytest.mark.parametrize("d", [64, 128])
def test_greatest_weight_above_a_lagging_maximum(cuda_device, d, dtype, lag):
    """One key has nearly all the weight, 128 slots behind the one the row's
    maximum still refers to, by less than the maximum may lag: its weight is then
    rounded like any other, where an exact maximum makes it 1. Two half steps in
    all: the weight's and the output's."""
    dev = cuda_device
    rows = 64
    pool = Pool([400], 1, 64, d, dtype)
    held = pool.table[0].long()
    key = torch.full((7 * 64, d), -16.0)  # the others: far below
    key[10], key[200] = 0.0, 1.0 / 16
    key[400:] = float("nan")
    pool.k[held] = key.view(7, 1, 64, d).to(dtype)
    cache = pool.device_cache(dev, PagedKVCache)
    # rows' scores of key 200 rise from 0 to `lag` powers of 2 above key 10's
    rise = torch.linspace(0.05, 0.95 * lag, rows) * 0.6931
    q = (rise * 16 / d)[:, None, None].expand(rows, 3, d).to(dtype).contiguous()
    want, tol = attention(pool, q, [(0, 337 + i) for i in range(rows)], 1.0)
    cu = torch.tensor([0, rows], dtype=torch.int32, device=dev)
    for splits in (0, 1):
        close(cache.prefill(q.to(dev), cu, scale=1.0, num_splits=splits), want, tol)
