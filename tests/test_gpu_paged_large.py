"""Rows far apart and many: offsets of q, k, v and results beyond 32 bits, the
largest batch."""
import pytest
import torch

from vla_abft_estimate_b200.paged import PagedKVCache, rope_table

from .paged_reference import Pool, attention
from .test_gpu_paged import BF16, F16, close

pytestmark = pytest.mark.gpu


def test_rows_beyond_32_bits(cuda_device):
    """Tokens 2^30 elements apart in a 4.3 GB buffer: the third starts at 2^31."""
    dev = cuda_device
    stride = (1 << 30) + 4096
    flat = torch.empty(2 * stride + 6 * 28 * 128, dtype=BF16, device=dev)  # only the rows are touched

    def rows(heads, at):
        return flat.as_strided((3, heads, 128), (stride, 128, 1), at * 28 * 128)

    pool = Pool([48, 300, 7], 4, 16, 128, BF16)
    cache = pool.device_cache(dev, PagedKVCache)
    g = torch.Generator().manual_seed(51)
    q, k, v = (torch.randn(3, h, 128, generator=g).to(BF16).to(dev) for h in (28, 4, 4))
    rope = rope_table(400, 128, device=dev)
    want_q = cache.append(q, k, v, rope)
    kept_k, kept_v = cache.k_pages.clone(), cache.v_pages.clone()
    want = cache.decode(want_q)
    cache.append(q, torch.zeros_like(k), torch.zeros_like(v), rope)
    for to, x in ((rows(28, 0), q), (rows(4, 1), k), (rows(4, 2), v)):
        to.copy_(x)
    far_q = cache.append(rows(28, 0), rows(4, 1), rows(4, 2), rope, q_out=rows(28, 3))
    assert torch.equal(far_q, want_q)
    # slots that no sequence uses hold NaN
    assert torch.equal(cache.k_pages.view(torch.int16), kept_k.view(torch.int16))
    assert torch.equal(cache.v_pages.view(torch.int16), kept_v.view(torch.int16))
    assert torch.equal(cache.decode(far_q, out=rows(28, 4)), want)
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev)
    near = cache.prefill(want_q, cu)
    for splits in (0, 2):
        got = cache.prefill(far_q, cu, out=rows(28, 5), num_splits=splits)
        assert splits or torch.equal(got, near)
        assert (got.float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max()
    cache.check_status()


def test_largest_batch(cuda_device):
    """65,535 sequences, most of them empty, and one more refused."""
    dev = cuda_device
    batch = 65535
    held = {0: 3, 1: 17, 30000: 40, 65533: 1, 65534: 33}
    pool = Pool(list(held.values()), 1, 16, 64, F16)
    table = torch.full((batch, pool.table.shape[1]), -1, dtype=torch.int32)
    lens = torch.zeros(batch, dtype=torch.int32)
    for i, (b, n) in enumerate(held.items()):
        table[b], lens[b] = pool.table[i], n
    cache = PagedKVCache(pool.k.to(dev), pool.v.to(dev), table.to(dev), lens.to(dev))
    at = list(held)
    g = torch.Generator().manual_seed(52)
    few = torch.randn(len(at), 2, 64, generator=g).to(F16)
    q = torch.zeros(batch, 2, 64, dtype=F16)
    q[at] = few
    want, tol = attention(pool, few, list(enumerate(held.values())))
    got = cache.decode(q.to(dev)).cpu()
    close(got[at], want, tol)
    got[at] = 0
    assert (got == 0).all()
    new = torch.zeros(batch, dtype=torch.int64)
    new[at] = 1
    cu = torch.cat((torch.zeros(1, dtype=torch.int64), new.cumsum(0))).int().to(dev)
    for splits in (0, 2):
        close(cache.prefill(few.to(dev), cu, num_splits=splits), want, tol)
    v = torch.randn(len(at), 1, 64, generator=g).to(F16)
    cache.append(None, v.to(dev), v.to(dev), cu_seqlens=cu)
    for i, (b, n) in enumerate(held.items()):
        assert torch.equal(cache.v_pages[pool.table[i, (n - 1) // 16].item(), 0, (n - 1) % 16].cpu(), v[i, 0])
    cache.check_status()
    more = PagedKVCache(cache.k_pages, cache.v_pages, torch.zeros(batch + 1, 1, dtype=torch.int32, device=dev),
                        torch.zeros(batch + 1, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError):
        more.decode(torch.zeros(batch + 1, 2, 64, dtype=F16, device=dev))
