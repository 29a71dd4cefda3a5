"""Paged prefill of batches in which sequences without keys have new rows."""
import pytest
import torch

from vla_abft_estimate_b200.paged import PagedKVCache

from .paged_reference import Pool, attention
from .test_gpu_paged import BF16, close, owners_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_heads,group,lens,columns", [
    (4, 7, [0] * 8 + [8192] * 3, 512),
    (4, 7, [8192] * 3 + [0] * 8, 512),
    (8, 4, [0] * 7 + [2048] * 3, 128),
    (1, 7, [2560, 0] * 50, 4096),
    (1, 7, [0, 2560] * 50, 4096),
    (4, 7, [-5] * 8 + [8192] * 3, 512),
])
def test_empty_sequences_take_no_piece_of_the_others(cuda_device, kv_heads, group, lens, columns):
    """One new row for each sequence: the rows of empty ones are zeros, all
    others complete, and the status tells of the empty ones."""
    dev = cuda_device
    held = [max(n, 0) for n in lens]
    pool = Pool(held, kv_heads, 16, 64, BF16, extra_columns=columns - -(-max(held) // 16))
    cache = pool.device_cache(dev, PagedKVCache)
    cache.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    rows = len(lens)
    q = torch.randn(rows, kv_heads * group, 64, generator=torch.Generator().manual_seed(21)).to(BF16)
    cu = torch.arange(rows + 1, dtype=torch.int32, device=dev)
    want, tol = attention(pool, q, owners_of([1] * rows, held))
    x = q.to(dev)
    torch.full((1 << 26,), float("nan"), dtype=torch.float32, device=dev)  # freed: scratch that no kernel wrote is NaN
    out = torch.full_like(x, 7.0)
    cache.prefill(x, cu, out=out)
    close(out, want, tol)
    with pytest.raises(ValueError, match="length"):
        cache.check_status()
