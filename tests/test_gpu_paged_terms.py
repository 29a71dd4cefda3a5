"""Decode's weights have two 16-bit terms: the output's rounding is the only one
that counts."""
import pytest
import torch

from vla_abft_estimate_b200.paged import PagedKVCache

from .paged_reference import HALF_STEP, Pool
from .test_gpu_paged import BF16, F16

pytestmark = pytest.mark.gpu


def weights_and_values(pool, q, lens):
    """By row: (weights [kv_heads, group, n], values [kv_heads, n, d], size of the
    scores' terms) in 64 bits."""
    for b, n in enumerate(lens):
        k, v = pool.rows(pool.k, b, n), pool.rows(pool.v, b, n)
        x = q[b].double().view(pool.kv_heads, -1, pool.d)
        scale = pool.d ** -0.5
        size = (torch.matmul(x.abs(), k.abs().transpose(1, 2)) * scale).amax(-1, keepdim=True)
        yield torch.softmax(torch.matmul(x, k.transpose(1, 2)) * scale, -1), v, size


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,sms", [(7, 0), (7, 2), (12, 0)])
def test_only_the_output_is_rounded(cuda_device, heads, sms, d, dtype):
    """Tolerance by element, u half a step of the type and |o| the result:
      u |o|                the output's rounding
      u^2 sum p |v|        the second term's (fp16: below 2^-24 in steps of
                           2^-24 of a greatest weight of 2^15, less than u^2)
      2 e sum p |v|        e = (d + 4) 2^-24 times the scores' terms, and 2^-21
                           for the exponential
      n / 16 2^-22 sum p |v|   fp32 sums
    Scores are kept near 0, so that this is far below u sum p |v|: weights of one
    term fail it, which the test shows on the CPU."""
    dev, lens = cuda_device, [300, 77, 513]
    pool = Pool(lens, 1, 16, d, dtype, seed=41)
    cache = pool.device_cache(dev, PagedKVCache)
    q = (torch.randn(3, heads, d, generator=torch.Generator().manual_seed(42)) * 0.1).to(dtype)
    got = cache.decode(q.to(dev), num_sms=sms).double().cpu()
    cache.check_status()
    u = HALF_STEP[dtype]
    for b, (p, v, size) in enumerate(weights_and_values(pool, q, lens)):
        o, mass = torch.matmul(p, v), torch.matmul(p, v.abs())
        e = (d + 4) * 2.0 ** -24 * size + 2.0 ** -21
        tol = u * o.abs() + (u * u + 2 * e + max(lens[b] / 16, 8) * 2.0 ** -22) * mass
        assert ((got[b].view_as(o) - o).abs() <= tol).all()
        top = p / p.amax(-1, keepdim=True)
        one = torch.matmul(top.to(dtype).double(), v) / top.sum(-1, keepdim=True)
        assert ((one.to(dtype).double() - o).abs() > tol).any()
