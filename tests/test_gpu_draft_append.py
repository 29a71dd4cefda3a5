"""Append by given positions of one or several axes."""
import pytest
import torch

from vla_abft_estimate_b200.paged import PagedKVCache, rope_table

from .draft_reference import i32, rotated_by
from .paged_reference import Pool
from .test_gpu_paged import BF16, F16, bits, close

pytestmark = pytest.mark.gpu


def run_append(dev, new, total, heads, kv_heads, d, page, dtype, sections, *, cu=True, pad=0, joint=False, seed=0, most=5000,
               with_q=True):
    pool = Pool(total, kv_heads, page, d, dtype, seed=seed, joint=joint)
    cache = pool.device_cache(dev, PagedKVCache)
    before = bits(cache.k_pages), bits(cache.v_pages)
    tokens = (sum(new) if cu else len(total)) + pad
    g = torch.Generator().manual_seed(seed + 1)
    qkv = torch.randn(tokens, (heads + 2 * kv_heads) * d, generator=g).to(dtype)
    sizes = [heads * d, kv_heads * d, kv_heads * d]
    q, k, v = (x.view(tokens, -1, d) for x in qkv.split(sizes, -1))
    dq, dk, dv = (x.view(tokens, -1, d) for x in qkv.to(dev).split(sizes, -1))
    positions = torch.randint(0, most, (len(sections), tokens), generator=g, dtype=torch.int32)
    if pad:
        positions[:, tokens - pad:] = -1  # rows of no sequence: not looked at
    bounds = i32([0] + list(torch.tensor(new).cumsum(0)), dev) if cu else None
    q_out = torch.full((tokens, heads, d), 7.0, dtype=dtype, device=dev)
    got = cache.append(dq if with_q else None, dk, dv, rope_table(most, d, device=dev), cu_seqlens=bounds,
                       q_out=q_out if with_q else None, positions=positions.to(dev), sections=sections)
    assert got is (q_out if with_q else None)
    cache.check_status()
    owner, slot_of = [], []
    for b, (n, t) in enumerate(zip(new, total)):
        owner += [b] * n
        slot_of += range(t - n, t)
    rows = list(range(sum(new))) if cu else [b for b, n in enumerate(new) if n]
    at = torch.tensor(slot_of, dtype=torch.int64)
    if with_q:
        close(q_out[rows], *rotated_by(q[rows], positions[:, rows], sections))
        assert (q_out[[i for i in range(tokens) if i not in set(rows)]] == 7.0).all()
    page_of, slot = pool.table[torch.tensor(owner, dtype=torch.int64), at // page].long(), at % page
    close(cache.k_pages.cpu()[page_of, :, slot], *rotated_by(k[rows], positions[:, rows], sections))
    assert torch.equal(bits(cache.v_pages.cpu()[page_of, :, slot]), bits(v[rows]))
    for now, was in ((bits(cache.k_pages), before[0]), (bits(cache.v_pages), before[1])):
        now, was = now.clone(), was.clone()
        now[page_of, :, slot] = 0
        was[page_of, :, slot] = 0
        assert torch.equal(now, was), "a slot of no appended token changed"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,sections", [(64, (32,)), (64, (8, 12, 12)), (64, (1, 30, 1)), (128, (16, 24, 24)),
                                        (128, (7, 0, 50, 7)), (128, (63, 1)), (128, (64, 0))])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (28, 4), (64, 1)])
def test_layouts(cuda_device, heads, kv_heads, d, sections, dtype):
    run_append(cuda_device, [3, 1, 17], [20, 1, 33], heads, kv_heads, d, 16, dtype, sections)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("new,total", [([1], [1]), ([1], [513]), ([300], [300]), ([16, 16], [16, 32]),
                                       ([5, 0, 0, 40], [700, 3, 0, 40]), ([700, 900], [1000, 900])])
def test_lengths(cuda_device, new, total, page):
    run_append(cuda_device, new, total, 7, 1, 128, page, BF16, (16, 24, 24), pad=2)


def test_one_row_per_sequence_joint_pool_and_no_q(cuda_device):
    run_append(cuda_device, [1, 0, 1, 0], [9, 0, 100, 0], 8, 2, 64, 16, F16, (10, 10, 12), cu=False)
    run_append(cuda_device, [4, 30], [50, 30], 14, 2, 128, 16, BF16, (64,), joint=True, pad=3)
    run_append(cuda_device, [4, 30], [50, 30], 14, 2, 128, 16, BF16, (60, 4), with_q=False)
    run_append(cuda_device, [1] * 70, [i % 90 + 1 for i in range(70)], 8, 8, 128, 32, BF16, (16, 24, 24))


def test_far_positions(cuda_device):
    run_append(cuda_device, [2], [40], 2, 1, 64, 128, F16, (16, 16), most=1 << 20)


def test_the_slots_own_places_give_what_append_gives(cuda_device):
    """Positions that are the slots', on one axis or on all: the same bits."""
    dev = cuda_device
    pool = Pool([70, 300], 2, 16, 128, BF16)
    q, k, v = (torch.randn(40, h, 128, generator=torch.Generator().manual_seed(h)).to(BF16).to(dev) for h in (8, 2, 2))
    cu, rope = i32([0, 10, 40], dev), rope_table(300, 128, device=dev)
    place = i32(list(range(60, 70)) + list(range(270, 300)), dev)
    want_cache = pool.device_cache(dev, PagedKVCache)
    want = want_cache.append(q, k, v, rope, cu_seqlens=cu)
    for positions, sections in ((place, None), (place, (64,)), (place[None], (64,)), (place.expand(3, 40), (16, 24, 24)),
                                (place.repeat(4, 1), [1, 2, 3, 58]), (torch.stack((place, place), 1).T.contiguous(), (4, 60)),
                                (place.repeat(2, 2)[:, :40], (32, 32))):
        cache = pool.device_cache(dev, PagedKVCache)
        assert torch.equal(cache.append(q, k, v, rope, cu_seqlens=cu, positions=positions, sections=sections), want)
        assert torch.equal(bits(cache.k_pages), bits(want_cache.k_pages))
        assert torch.equal(bits(cache.v_pages), bits(want_cache.v_pages))
        again = q.clone()
        assert cache.append(again, k, v, rope, cu_seqlens=cu, positions=positions, sections=sections, q_out=again) is again
        assert torch.equal(again, want)


@pytest.mark.parametrize("bad", [-1, 64, -2 ** 31, 2 ** 31 - 1])
@pytest.mark.parametrize("axis", [0, 1, 2])
def test_positions_outside_the_table_skip_the_token(cuda_device, axis, bad):
    dev = cuda_device
    pool = Pool([40, 25], 2, 16, 64, BF16)
    cache = pool.device_cache(dev, PagedKVCache)
    q, k = torch.randn(5, 4, 64, device=dev).to(BF16), torch.randn(5, 2, 64, device=dev).to(BF16)
    positions = torch.full((3, 5), 63, dtype=torch.int32, device=dev)
    positions[axis, 3] = bad
    out = torch.full_like(q, 5.0)
    before = bits(cache.v_pages)
    cache.append(q, k, k, rope_table(64, 64, device=dev), cu_seqlens=i32([0, 2, 5], dev), q_out=out, positions=positions,
                 sections=(10, 11, 11))
    assert (out[3] == 5.0).all() and all((out[i] != 5.0).any() for i in (0, 1, 2, 4))
    page, slot = pool.table[1, 1].long(), 23 - 16
    assert torch.equal(bits(cache.v_pages)[page, :, slot], before[page, :, slot])
    with pytest.raises(ValueError, match="rotation table"):
        cache.check_status()
    cache.check_status()


def test_refusals(cuda_device):
    dev = cuda_device
    cache = Pool([40], 2, 16, 64, BF16).device_cache(dev, PagedKVCache)
    k, q = torch.zeros(6, 2, 64, dtype=BF16, device=dev), torch.zeros(6, 4, 64, dtype=BF16, device=dev)
    cu, rope, at = i32([0, 6], dev), rope_table(64, 64, device=dev), i32([1] * 6, dev)

    def call(positions=at, sections=None, table=rope):
        return cache.append(q, k, k, table, cu_seqlens=cu, positions=positions, sections=sections)

    before = bits(cache.k_pages).clone()
    for positions, sections in ((at[:5], None), (at.long(), None), (at.cpu(), None), (at[None, None], None),
                                (i32([1] * 12, dev)[::2], None), (at, (16, 16)), (at.repeat(2, 1), None),
                                (at.repeat(2, 1), (32,)), (at.repeat(2, 1), (16, 15)), (at.repeat(2, 1), (33, -1)),
                                (at.repeat(2, 1), (16.0, 16.0)), (at.repeat(2, 1), (2 ** 40, 32 - 2 ** 40)),
                                (at.repeat(5, 1), (8, 8, 8, 4, 4)), (at[:0][None], (32,))):
        with pytest.raises(ValueError):
            call(positions, sections)
    with pytest.raises(TypeError):
        call([1] * 6)
    with pytest.raises(ValueError, match="without rope"):
        call(table=None)
    with pytest.raises(ValueError, match="sections without"):
        cache.append(q, k, k, rope, cu_seqlens=cu, sections=(32,))
    with pytest.raises(ValueError, match="rope"):
        call(table=rope[:0])
    with pytest.raises(ValueError, match="gradient"):
        call(table=rope.clone().requires_grad_())
    assert torch.equal(bits(cache.k_pages), before)
    cache.check_status()
