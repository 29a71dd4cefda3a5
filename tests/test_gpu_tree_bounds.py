"""Tree attention where boundaries and depths are at their limits."""
import random

import pytest
import torch

from vla_abft_estimate_b200.paged import PagedKVCache

from .draft_reference import attention_over, chain, i32, packed, random_tree, visible_slots
from .paged_reference import Pool
from .test_gpu_paged import BF16, F16, close
from .test_gpu_tree import run_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [256, 512, 600])
def test_boundaries_that_give_every_other_sequence_all_rows(cuda_device, batch):
    """Of 64 query and 8 kv heads a tile holds 16 rows: batch / 2 sequences of 256 tiles, 8 heads and 8,195 places each,
    2,148,270,080 places for 256 sequences, which pass 31 bits, and 4,296,540,160 for 512, which pass 32. Nothing is
    answered, and the status tells."""
    dev = cuda_device
    pages = torch.zeros(2, 1, 8, 128, 64, dtype=BF16, device=dev)
    cache = PagedKVCache(pages[0], pages[1], torch.zeros(batch, 4096, dtype=torch.int32, device=dev),
                         torch.full((batch,), 4096 * 128, dtype=torch.int32, device=dev))
    q = torch.zeros(4096, 64, 64, dtype=BF16, device=dev)
    room = torch.full((4096 + 64, 64, 64), 7.0, dtype=BF16, device=dev)
    cu = i32([0, 4096] * (batch // 2) + [0], dev)
    cache.tree(q, cu, i32([-1] * 4096, dev), out=room[32:-32])
    with pytest.raises(ValueError, match="cu_seqlens"):
        cache.check_status()
    assert (room == 7.0).all()


@pytest.mark.parametrize("columns", [4, 400])
def test_boundaries_that_overlap(cuda_device, columns):
    """By cluster and by list: what several sequences claim is written within the rows, and the status tells."""
    dev = cuda_device
    pages = torch.randn(2, 9, 2, 16, 64, generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    table = torch.zeros(6, columns, dtype=torch.int32, device=dev)
    cache = PagedKVCache(pages[0], pages[1], table, i32([60] * 6, dev))
    q = torch.randn(40, 4, 64, generator=torch.Generator().manual_seed(2)).to(BF16).to(dev)
    room = torch.full((60, 4, 64), 7.0, dtype=BF16, device=dev)
    for bounds in ([0, 40, 0, 40, 0, 40, 0], [0, 40, 1, 39, 2, 38, 3], [0, 10, 5, 15, 10, 20, 15]):
        cache.tree(q, i32(bounds, dev), i32([-1] * 40, dev), out=room[10:50])
        with pytest.raises(ValueError, match="cu_seqlens"):
            cache.check_status()
        assert (room[:10] == 7.0).all() and (room[50:] == 7.0).all()


def deep_tree(n, seed):
    """A row's parent is one of the few before it: depths of about n / 3."""
    r = random.Random(seed)
    return [max(-1, i - r.choice([1, 1, 2, 3, 7])) for i in range(n)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("past", [0, 1, 63, 100, 1000])
@pytest.mark.parametrize("n", [64, 65, 127, 128, 129, 300])
def test_deep_trees(cuda_device, n, past, dtype):
    """Trees of one step, of two and of more, by cluster and by list."""
    for columns in (0, 800):
        run_tree(cuda_device, [deep_tree(n, 1), chain(n), random_tree(7, 2)], [n + past, n + past // 2, 90], 6, 2, 64, 16, dtype,
                 extra_columns=columns, seed=n)


@pytest.mark.parametrize("sms", [0, 1, 3, 11])
@pytest.mark.parametrize("n,past", [(500, 40), (513, 7), (900, 333), (1700, 0)])
def test_deep_trees_in_pieces(cuda_device, n, past, sms):
    """Pieces that begin and end among the drafted rows; parents of other rows are not held."""
    run_tree(cuda_device, [deep_tree(n, 3), random_tree(30, 2), chain(n // 2)], [n + past, 800, n // 2 + past], 2, 2, 128, 32, BF16,
             sms=sms)


@pytest.mark.parametrize("sms", [0, 2])
@pytest.mark.parametrize("n", [300, 1100])
def test_bad_parents_of_deep_trees(cuda_device, n, sms):
    dev = cuda_device
    pool = Pool([n + 70, 90], 1, 16, 64, BF16)
    cache = pool.device_cache(dev, PagedKVCache)
    q = torch.randn(n + 20, 2, 64, generator=torch.Generator().manual_seed(4)).to(BF16)
    good = [deep_tree(n, 2), random_tree(20, 5)]
    for at in (0, 1, 63, n // 2, n - 2, n - 1):
        for bad in (at, n + 5, -2, 2 ** 31 - 1, -2 ** 31):
            wrong = [list(good[0]), good[1]]
            wrong[0][at] = bad
            cu, parents = packed(wrong)
            got = cache.tree(q.to(dev), i32(cu, dev), i32(parents, dev), num_sms=sms)
            with pytest.raises(ValueError, match="parent"):
                cache.check_status()
            some = [i for i in range(0, n + 20, 17)] + [at, min(n - 1, at + 1), n - 1]
            rows = [(0, visible_slots(wrong[0], i, n + 70)) if i < n else (1, visible_slots(wrong[1], i - n, 90)) for i in some]
            close(got[some], *attention_over(pool, q[some], rows))
    cu, parents = packed(good)
    cache.tree(q.to(dev), i32(cu, dev), i32(parents, dev), num_sms=sms)
    cache.check_status()


def test_more_rows_than_tokens_in_deep_trees(cuda_device):
    """The first rows have no slots; later ones see themselves and the ancestors that have some."""
    dev = cuda_device
    for n, total in ((200, 130), (700, 90), (700, 699)):
        pool = Pool([total], 1, 16, 64, BF16)
        cache = pool.device_cache(dev, PagedKVCache)
        tree = deep_tree(n, 7)
        q = torch.randn(n, 2, 64, generator=torch.Generator().manual_seed(5)).to(BF16)
        got = cache.tree(q.to(dev), i32([0, n], dev), i32(tree, dev))
        close(got, *attention_over(pool, q, [(0, visible_slots(tree, i, total)) for i in range(n)]))
        with pytest.raises(ValueError, match="length"):
            cache.check_status()


def test_a_chain_of_many_rows(cuda_device):
    """60,000 rows, each seeing all before it: what prefill answers, and without a wait that gives up (a walk from each
    row in each of its steps would be 28 million hops a row, seconds)."""
    dev, n = cuda_device, 60000
    pool = Pool([n], 1, 64, 64, BF16)
    cache = pool.device_cache(dev, PagedKVCache)
    q = torch.randn(n, 1, 64, generator=torch.Generator().manual_seed(8)).to(BF16)
    cu = i32([0, n], dev)
    got = cache.tree(q.to(dev), cu, torch.arange(-1, n - 1, dtype=torch.int32, device=dev))
    cache.check_status()
    some = [0, 1, 63, 64, 127, 128, 129, 511, 512, 513, 4095, 4096, 30001, 59903, 59904, 59998, 59999]
    want, tol = attention_over(pool, q[some], [(0, list(range(i + 1))) for i in some])
    close(got[some], want, tol)
    close(cache.prefill(q.to(dev), cu)[some], want, tol)
