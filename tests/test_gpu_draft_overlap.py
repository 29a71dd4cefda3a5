"""Arrays that a call writes and reads: from Python."""
import pytest
import torch

from vla_abft_estimate_b200 import _native as N
from vla_abft_estimate_b200 import paged

from .draft_reference import i32
from .test_gpu_draft_layers import contents, layers_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("long_way", [False, True])
def test_what_is_written_is_not_what_others_read(cuda_device, long_way, monkeypatch):
    if long_way:
        monkeypatch.setattr(paged, "_HOST", paged._LongWay)
    dev = cuda_device
    layers = layers_of(dev, [30, 30, 0])
    cu, kept, counts = i32([0, 4, 8, 8], dev), i32([0, 2, 3, -1, 1, -1, -1, -1], dev), i32([3, 1, 0], dev)
    before, table = contents(layers), layers.page_table.tolist()
    for out in (cu[:3], cu[1:], kept[:3], kept[5:]):
        with pytest.raises(N.AbftError, match="abft_kv_keep"):
            layers.keep(cu, kept, counts, lens_out=out)
    one = i32([0], dev)
    for lists in ((one, i32([2], dev), layers.page_table[2, 1:2]), (layers.seq_lens[2:], i32([2], dev), one),
                  (one, layers.seq_lens[1:2], one)):
        with pytest.raises(N.AbftError, match="abft_kv_fork"):
            layers.fork(*lists)
    assert torch.equal(contents(layers), before) and layers.page_table.tolist() == table
    assert layers.seq_lens.tolist() == [30, 30, 0] and cu.tolist() == [0, 4, 8, 8]
    # a count is read before its length is written
    assert layers.keep(cu, kept, counts, lens_out=counts) is counts and counts.tolist() == [29, 27, 0]
    layers.check_status()
