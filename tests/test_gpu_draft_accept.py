"""What accept gives, as tensors."""
import io

import pytest
import torch

from vla_abft_estimate_b200 import paged

from .draft_reference import chain, i32, packed
from .test_gpu_draft_layers import layers_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("long_way", [False, True])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_results_have_a_memory_of_their_own(cuda_device, dtype, long_way, monkeypatch):
    """Growing, shrinking, saving or freeing one leaves the others; by either way to the library."""
    if long_way:
        monkeypatch.setattr(paged, "_HOST", paged._LongWay)
    dev, n, batch = cuda_device, 5, 3
    layers = layers_of(dev, [1] * batch, layers=1)
    cu, parents = packed([chain(n)] * batch)
    ids = torch.ones(batch * n, dtype=dtype, device=dev)
    want = [list(range(n)) * batch, [n] * batch, [1] * batch]
    for which in range(3):
        for change in (lambda x: x.resize_(4000).fill_(-9), lambda x: x.resize_(1), lambda x: x.untyped_storage().resize_(0)):
            got = list(layers.accept(i32(cu, dev), i32(parents, dev), ids, ids))
            assert [x.tolist() for x in got] == want
            assert len({x.untyped_storage().data_ptr() for x in got}) == 3
            change(got[which])
            for k in range(3):
                assert k == which or got[k].tolist() == want[k]
    got = layers.accept(i32(cu, dev), i32(parents, dev), ids, ids)
    for x in got:
        assert x.storage_offset() == 0 and x.untyped_storage().nbytes() == x.numel() * x.element_size()
        file = io.BytesIO()
        torch.save(x, file)
        file.seek(0)
        assert torch.equal(torch.load(file), x)
