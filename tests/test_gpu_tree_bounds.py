"""Tree attention where boundaries, depths and results are at their limits."""
import pytest
import torch

from vla_abft_estimate_b200.paged import PagedKVCache

from .draft_reference import i32
from .test_gpu_paged import BF16

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
