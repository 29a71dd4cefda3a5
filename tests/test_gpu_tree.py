"""Tree attention over the paged cache against the plain 64-bit form."""
import math
import random

import pytest
import torch

from vla_abft_estimate_b200.paged import PagedKVCache

from .draft_reference import attention_over, chain, i32, packed, random_tree, visible_slots
from .paged_reference import Pool
from .test_gpu_paged import BF16, F16, bits, close

pytestmark = pytest.mark.gpu


def run_tree(dev, trees, total, heads, kv_heads, d, page, dtype, *, seed=0, pad=0, scale=None, sms=0, joint=False,
             strided=False, in_place=False, extra_columns=0):
    pool = Pool(total, kv_heads, page, d, dtype, seed=seed, joint=joint, extra_columns=extra_columns)
    cache = pool.device_cache(dev, PagedKVCache)
    cu, parents = packed(trees)
    tokens = cu[-1] + pad
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(tokens, heads, d, generator=g).to(dtype)
    dq = q.to(dev)
    if strided:  # a part of a wider projection
        wide = torch.zeros(tokens, heads + 3, d, dtype=dtype, device=dev)
        wide[:, 1:heads + 1] = dq
        dq = wide[:, 1:heads + 1]
    out = dq if in_place else torch.full((tokens, heads, d), 7.0, dtype=dtype, device=dev)
    before = bits(cache.k_pages), bits(cache.v_pages)
    got = cache.tree(dq, i32(cu, dev), i32(parents + [-1] * pad, dev), scale=scale, out=out, num_sms=sms)
    assert got is out
    cache.check_status()
    rows = [(b, visible_slots(tree, i, total[b])) for b, tree in enumerate(trees) for i in range(len(tree))]
    close(out[:cu[-1]], *attention_over(pool, q[:cu[-1]], rows, scale))
    assert torch.equal(out[cu[-1]:].cpu(), (q if in_place else torch.full_like(q, 7.0))[cu[-1]:])
    assert torch.equal(bits(cache.k_pages), before[0]) and torch.equal(bits(cache.v_pages), before[1])
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (28, 4), (6, 3), (16, 16), (64, 1), (24, 2)])
def test_head_layouts(cuda_device, heads, kv_heads, d, dtype):
    trees = [random_tree(13, 1), random_tree(1, 2), random_tree(29, 3)]
    run_tree(cuda_device, trees, [200, 1, 61], heads, kv_heads, d, 16, dtype)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n,total", [(1, 1), (1, 129), (16, 16), (17, 300), (64, 64), (64, 1000), (127, 255), (130, 130),
                                     (200, 456), (300, 301)])
def test_lengths(cuda_device, n, total, page):
    run_tree(cuda_device, [random_tree(n, n + total)], [total], 7, 1, 128, page, BF16)


@pytest.mark.parametrize("sms", [0, 1, 2, 5, 37, 600])
@pytest.mark.parametrize("d", [64, 128])
def test_long_caches_in_pieces(cuda_device, d, sms):
    trees = [random_tree(26, 5), random_tree(3, 6), [], random_tree(61, 7)]
    run_tree(cuda_device, trees, [3000, 700, 0, 1111], 14, 2, d, 32, BF16, sms=sms)


@pytest.mark.parametrize("shape", ["chain", "star", "many roots", "two deep", "roots only"])
def test_shapes_of_trees(cuda_device, shape):
    n = 150
    tree = {"chain": chain(n), "star": [-1] + [0] * (n - 1), "many roots": random_tree(n, 9, roots=40),
            "two deep": [-1, -1] + [i for i in range(n - 2)], "roots only": [-1] * n}[shape]
    run_tree(cuda_device, [tree, random_tree(5, 1)], [400, 50], 8, 4, 64, 16, BF16)


@pytest.mark.parametrize("offset", range(0, 33, 4))
def test_drafted_rows_across_steps(cuda_device, offset):
    """The drafted slots begin anywhere in a step of 128, and reach into the next ones."""
    for n, total in ((40, 100 + offset + 40), (140, 120 + offset + 140), (9, 119 + offset)):
        run_tree(cuda_device, [random_tree(n, offset)], [total], 2, 1, 64, 16, BF16, seed=offset)


def test_batches(cuda_device):
    for batch in (1, 31, 33, 150):
        trees = [random_tree(1 + (b * 7) % 12 if b % 5 != 4 else 0, b) for b in range(batch)]
        total = [len(t) + (b * 53) % 200 if t else 0 for b, t in enumerate(trees)]
        run_tree(cuda_device, trees, total, 4, 2, 64, 16, BF16, pad=3)


def test_strides_in_place_and_joint_pools(cuda_device):
    trees, total = [random_tree(20, 1), random_tree(7, 2)], [90, 40]
    run_tree(cuda_device, trees, total, 12, 4, 128, 16, F16, joint=True, strided=True, pad=4)
    run_tree(cuda_device, trees, total, 12, 4, 128, 16, BF16, in_place=True, pad=2)
    run_tree(cuda_device, trees, total, 12, 4, 128, 16, BF16, in_place=True, strided=True, extra_columns=900)


@pytest.mark.parametrize("scale", [0.0, -0.25, 1.0, 0.02])
def test_scales(cuda_device, scale):
    run_tree(cuda_device, [random_tree(20, 1), random_tree(7, 2)], [900, 40], 8, 2, 64, 32, BF16, scale=scale)


def test_a_chain_is_what_prefill_gives(cuda_device):
    pool = Pool([500, 90], 2, 16, 128, BF16)
    cache = pool.device_cache(cuda_device, PagedKVCache)
    cu, parents = packed([chain(30), chain(90)])
    q = torch.randn(120, 8, 128, generator=torch.Generator().manual_seed(1)).to(BF16).to(cuda_device)
    got = cache.tree(q, i32(cu, cuda_device), i32(parents, cuda_device))
    rows = [(b, list(range(t - n + i + 1))) for b, (n, t) in enumerate(((30, 500), (90, 90))) for i in range(n)]
    want, tol = attention_over(pool, q.cpu(), rows)
    close(got, want, tol)
    close(cache.prefill(q, i32(cu, cuda_device)), want, tol)


def test_hidden_rows_do_not_count_however_large(cuda_device):
    """Siblings' keys that would win every softmax, with large values: nothing of them is seen."""
    pool = Pool([300], 1, 16, 64, BF16)
    tree = [-1] + [0] * 20 + list(range(1, 21))  # twenty branches of two
    before = 300 - len(tree)
    for x, by in ((pool.k, 1e4), (pool.v, 1e30)):
        for row in range(2, len(tree), 2):
            at = before + row
            x[pool.table[0, at // 16].long(), :, at % 16] *= by
    cache = pool.device_cache(cuda_device, PagedKVCache)
    q = torch.randn(len(tree), 4, 64, generator=torch.Generator().manual_seed(2)).to(BF16)
    got = cache.tree(q.to(cuda_device), i32([0, len(tree)], cuda_device), i32(tree, cuda_device))
    odd = [i for i in range(len(tree)) if all(a % 2 or a == 0 for a in (i, max(tree[i], 0)))]
    want, tol = attention_over(pool, q, [(0, visible_slots(tree, i, 300)) for i in range(len(tree))])
    close(got[odd], want[odd], tol[odd])


@pytest.mark.parametrize("columns", [0, 1000])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_key_that_is_no_number_reaches_the_rows_that_see_it(cuda_device, value, columns):
    tree, total, at_row = [-1, 0, 0, 1, 2, 3, 4], 200, 2  # rows 2, 4 and 6 are one branch
    pool = Pool([total], 2, 16, 64, BF16, extra_columns=columns)
    q = torch.randn(len(tree), 4, 64, generator=torch.Generator().manual_seed(6)).to(BF16).to(cuda_device)
    cu, up = i32([0, len(tree)], cuda_device), i32(tree, cuda_device)
    want = pool.device_cache(cuda_device, PagedKVCache).tree(q, cu, up)
    at = total - len(tree) + at_row
    pool.k[pool.table[0, at // 16].long(), :, at % 16] = value
    got = pool.device_cache(cuda_device, PagedKVCache).tree(q, cu, up)
    others = [0, 1, 3, 5]
    assert torch.equal(bits(got[others]), bits(want[others]))
    assert got[[2, 4, 6]].isnan().all()


@pytest.mark.parametrize("sms", [0, 1, 3])
def test_bad_parents_end_the_way_up(cuda_device, sms):
    dev = cuda_device
    tree = random_tree(40, 3)
    tree[7], tree[11], tree[20], tree[39] = 7, 30, -9, 2 ** 31 - 1
    tree[25], tree[30] = 20, -2 ** 31
    tree[26] = 11
    pool = Pool([700], 2, 16, 64, BF16)
    cache = pool.device_cache(dev, PagedKVCache)
    q = torch.randn(40, 4, 64, generator=torch.Generator().manual_seed(4)).to(BF16)
    got = cache.tree(q.to(dev), i32([0, 40], dev), i32(tree, dev), num_sms=sms)
    close(got, *attention_over(pool, q, [(0, visible_slots(tree, i, 700)) for i in range(40)]))
    with pytest.raises(ValueError, match="parent"):
        cache.check_status()
    cache.check_status()


@pytest.mark.parametrize("bad", [-2, 2 ** 31 - 1])
def test_one_bad_parent_is_told(cuda_device, bad):
    """Of any row, in any step, and of none when all are right."""
    dev = cuda_device
    pool = Pool([333, 20], 1, 16, 64, BF16)
    cache = pool.device_cache(dev, PagedKVCache)
    cu, parents = packed([random_tree(200, 1), random_tree(20, 2)])
    q = torch.zeros(220, 2, 64, dtype=BF16, device=dev)
    for at in (0, 63, 127, 199, 200, 219):
        wrong = list(parents)
        wrong[at] = bad
        cache.tree(q, i32(cu, dev), i32(wrong, dev))
        with pytest.raises(ValueError, match="parent"):
            cache.check_status()
    cache.tree(q, i32(cu, dev), i32(parents, dev))
    cache.check_status()


def test_lengths_below_the_rows(cuda_device):
    """More rows than tokens: the first rows have no slots and see nothing; later ones see themselves."""
    dev = cuda_device
    pool = Pool([5, 40], 2, 16, 64, BF16)
    cache = pool.device_cache(dev, PagedKVCache)
    trees = [[-1, 0, 1, 2, 1, 4, 3, 5], random_tree(6, 1)]
    cu, parents = packed(trees)
    q = torch.randn(14, 4, 64, generator=torch.Generator().manual_seed(5)).to(BF16)
    got = cache.tree(q.to(dev), i32(cu, dev), i32(parents, dev))
    rows = [(b, visible_slots(t, i, (5, 40)[b])) for b, t in enumerate(trees) for i in range(len(t))]
    assert rows[0][1] == [] and rows[4][1] == [1]
    close(got, *attention_over(pool, q, rows))
    with pytest.raises(ValueError, match="length"):
        cache.check_status()


def test_bad_pages_read_as_zeros(cuda_device):
    dev = cuda_device
    pool = Pool([200], 1, 16, 64, BF16)
    cache = pool.device_cache(dev, PagedKVCache)
    tree = random_tree(20, 1)
    q = torch.randn(20, 2, 64, generator=torch.Generator().manual_seed(6)).to(BF16)
    cache.page_table[0, 3] = 10 ** 6
    got = cache.tree(q.to(dev), i32([0, 20], dev), i32(tree, dev))
    for x in (pool.k, pool.v):
        x[pool.table[0, 3].long()] = 0
    close(got, *attention_over(pool, q, [(0, visible_slots(tree, i, 200)) for i in range(20)]))
    with pytest.raises(ValueError, match="page_table"):
        cache.check_status()


@pytest.mark.parametrize("bounds", [(0, 4, 10, 20), (5, 8, 10, 12), (-3, 4, 10, 12), (0, 3, -2 ** 31, 2 ** 31 - 1)])
def test_bad_boundaries(cuda_device, bounds):
    """Sequences whose boundaries lie outside the rows are not answered, the others are."""
    dev = cuda_device
    total = (40, 90, 30)
    pool = Pool(total, 2, 16, 64, BF16, seed=3)
    cache = pool.device_cache(dev, PagedKVCache)
    q = torch.randn(12, 4, 64, generator=torch.Generator().manual_seed(7)).to(BF16)
    out = torch.full((12, 4, 64), 7.0, dtype=BF16, device=dev)
    parents = [-1] * 12
    cache.tree(q.to(dev), i32(bounds, dev), i32(parents, dev), out=out)
    rows = [None] * 12
    for b in range(3):
        lo, hi = bounds[b], bounds[b + 1]
        if 0 <= lo <= hi <= 12:
            for i in range(hi - lo):
                rows[lo + i] = (b, visible_slots([-1] * (hi - lo), i, total[b]))
    live = [i for i, r in enumerate(rows) if r]
    close(out[live], *attention_over(pool, q[live], [rows[i] for i in live]))
    assert (out[[i for i, r in enumerate(rows) if r is None]] == 7.0).all()
    with pytest.raises(ValueError, match="cu_seqlens"):
        cache.check_status()


def test_large_pools_and_rows(cuda_device):
    """Offsets beyond 2^31 elements in the pool."""
    dev = cuda_device
    pages = (1 << 31) // (2 * 16 * 128) + 9
    k = torch.zeros(pages, 2, 16, 128, dtype=BF16, device=dev)
    v = torch.zeros_like(k)
    pool = Pool([50], 2, 16, 128, BF16, seed=8)
    held = torch.tensor([pages - 1, 0, pages - 3, 5])
    k[held.to(dev)] = pool.k[pool.table[0, :4].long()].to(dev)
    v[held.to(dev)] = pool.v[pool.table[0, :4].long()].to(dev)
    cache = PagedKVCache(k, v, held.int()[None].to(dev), i32([50], dev))
    tree = random_tree(21, 4)
    q = torch.randn(21, 6, 128, generator=torch.Generator().manual_seed(9)).to(BF16)
    got = cache.tree(q.to(dev), i32([0, 21], dev), i32(tree, dev))
    cache.check_status()
    close(got, *attention_over(pool, q, [(0, visible_slots(tree, i, 50)) for i in range(21)]))


def test_repeated_and_transposed_query_rows(cuda_device):
    """One row for all heads or tokens, heads before tokens: the same as their dense copies."""
    dev = cuda_device
    cache = Pool([90, 40], 2, 16, 64, BF16).device_cache(dev, PagedKVCache)
    cu, parents = packed([random_tree(20, 1), random_tree(7, 2)])
    g = torch.Generator().manual_seed(3)
    x = torch.randn(27, 6, 64, generator=g).to(BF16).to(dev)
    for q in (x[:, :1].expand(27, 6, 64), x[:1].expand(27, 6, 64), x.transpose(0, 1).contiguous().transpose(0, 1),
              torch.nn.functional.pad(x, (0, 8))[..., :64], x.flip(0), x.new_zeros(27 * 6 * 64 + 1)[1:].view(27, 6, 64).copy_(x)):
        got = cache.tree(q, i32(cu, dev), i32(parents, dev))
        assert torch.equal(got, cache.tree(q.clone(memory_format=torch.contiguous_format), i32(cu, dev), i32(parents, dev)))
    cache.check_status()


@pytest.mark.parametrize("n", [511, 512, 513, 700])
def test_trees_around_the_parents_that_are_held(cuda_device, n):
    run_tree(cuda_device, [random_tree(n, 1), chain(n), random_tree(3, 2)], [n + 130, n, 70], 2, 1, 64, 16, BF16)


def test_refusals(cuda_device):
    dev = cuda_device
    cache = Pool([40], 2, 16, 64, BF16).device_cache(dev, PagedKVCache)
    q, cu, up = torch.zeros(6, 4, 64, dtype=BF16, device=dev), i32([0, 6], dev), i32([-1] * 6, dev)
    for parents in (up[:5], up.long(), up.cpu(), up[None], i32([-1] * 12, dev)[::2], None, [-1] * 6):
        with pytest.raises(ValueError, match="parents"):
            cache.tree(q, cu, parents)
    with pytest.raises(ValueError, match="cu_seqlens"):
        cache.tree(q, i32([0, 3, 6], dev), up)
    with pytest.raises(ValueError):
        cache.tree(q, cu, up, scale=math.inf)
    with pytest.raises(ValueError):
        cache.tree(q, cu, up, num_sms=-1)
    with pytest.raises(ValueError, match="q must be"):
        cache.tree(q.half(), cu, up)
    with pytest.raises(ValueError, match="heads"):
        cache.tree(q[:, :3], cu, up)
    with pytest.raises(ValueError, match="repeat"):
        cache.tree(q, cu, up, out=q[:1].expand(6, 4, 64))
    with pytest.raises(ValueError, match="gradient"):
        cache.tree(q.clone().requires_grad_(), cu, up)
    assert cache.tree(q[:0], i32([0, 0], dev), up[:0]).shape == (0, 4, 64)


# The table's width decides whether a segment has a cluster of CTAs or a part of the
# list, the number of rows how many segments there are.
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("columns", [0, 2000])
@pytest.mark.parametrize("heads,kv_heads,n", [(4, 4, 5), (8, 2, 4), (14, 2, 4), (16, 2, 8), (7, 1, 16), (64, 1, 3)])
def test_small_trees(cuda_device, heads, kv_heads, n, columns, d, dtype):
    for sizes, total in (([n], [600]), ([n], [n]), ([n], [64 + n]), ([n, n, 1, 0, n], [129, 64, 1, 0, 2000]),
                         ([n] * 9, [n + 61 * b for b in range(9)])):
        run_tree(cuda_device, [random_tree(x, 3 + i) for i, x in enumerate(sizes)], total, heads, kv_heads, d, 16, dtype,
                 extra_columns=columns)


@pytest.mark.parametrize("columns", [0, 1000])
def test_uneven_small_trees(cuda_device, columns):
    """Trees of several times the average's rows: more segments than one, and idle sequences."""
    for seed in range(4):
        sizes = [1, 60, 0, 2, 0, 33, 1, 1, 0, 5, 1, 2]
        total = [1, 900, 0, 40, 0, 33, 700, 64, 0, 300, 2, 129]
        run_tree(cuda_device, [random_tree(n, seed + n) for n in sizes], total, 12, 2, 128, 16, BF16, seed=seed, pad=5,
                 extra_columns=columns)


# By the number of segments and the table's width one to eight CTAs share a segment,
# with tiles of 128 rows or less.
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("batch,n,slots,d", [(1, 16, 1000, 128), (1, 5, 1000, 64), (1, 64, 1000, 128), (4, 16, 1000, 128),
                                             (4, 16, 3900, 128), (8, 16, 500, 64), (8, 16, 1000, 64), (8, 16, 2000, 64),
                                             (16, 16, 500, 128), (16, 16, 1000, 128), (32, 8, 1200, 128), (9, 30, 700, 128)])
def test_segments_shared_by_some_ctas(cuda_device, batch, n, slots, d, ragged):
    r = random.Random(batch * slots)
    sizes = [r.choice([0, 1, n // 2, n, n]) if ragged else n for _ in range(batch - 1)] + [n]
    total = [r.randrange(x, slots) if ragged else slots - b for b, x in enumerate(sizes)]
    run_tree(cuda_device, [random_tree(x, 5 + i) for i, x in enumerate(sizes)], total, 28, 4, d, 16, F16 if ragged else BF16,
             seed=batch, pad=3 * ragged)


def test_long_caches_of_small_trees(cuda_device):
    """Segments that cross many CTAs, whole ones inside one, and many sequences."""
    run_tree(cuda_device, [random_tree(6, 1)], [20000], 8, 1, 128, 64, BF16)
    run_tree(cuda_device, [random_tree(6, 1), random_tree(3, 2)], [9000, 30], 20, 2, 64, 32, F16)
    run_tree(cuda_device, [random_tree(4, b) for b in range(40)], [30 + 97 * (b * b % 41) for b in range(40)], 8, 4, 64, 16, BF16)
    run_tree(cuda_device, [random_tree(1 + b % 3, b) for b in range(1100)], [3 + b % 70 for b in range(1100)], 2, 1, 64, 16, BF16)


def test_small_trees_say_what_is_wrong(cuda_device):
    """Bad lengths, pages, parents and boundaries, by cluster and by list."""
    dev = cuda_device
    for columns in (0, 1000):
        trees, total = [random_tree(6, 1), random_tree(5, 2), random_tree(4, 3)], [40, 100, 3]
        cu, parents = packed(trees)
        q = torch.randn(cu[-1], 4, 64, generator=torch.Generator().manual_seed(4)).to(BF16)

        def answer(change, match, want=None, total=total, cu=cu, parents=parents):
            pool = Pool([40, 100, 10], 2, 16, 64, BF16, extra_columns=columns)
            cache = pool.device_cache(dev, PagedKVCache)
            cache.seq_lens.copy_(i32(total))
            change(cache)
            out = torch.full((len(q), 4, 64), 7.0, dtype=BF16, device=dev)
            cache.tree(q.to(dev), i32(cu, dev), i32(parents, dev), out=out)
            with pytest.raises(ValueError, match=match):
                cache.check_status()
            cache.check_status()
            return pool, out

        pool, out = answer(lambda c: None, "length")  # sequence 2 has more rows than tokens
        close(out, *attention_over(pool, q, [(b, visible_slots(t, i, total[b])) for b, t in enumerate(trees)
                                             for i in range(len(t))]))
        for lens in ([40, 100, 0], [40, 100, -5]):
            pool, out = answer(lambda c: None, "length", total=lens)
            assert (out[cu[2]:] == 0).all()
            close(out[:cu[2]], *attention_over(pool, q[:cu[2]], [(b, visible_slots(trees[b], i, total[b])) for b in (0, 1)
                                                                 for i in range(len(trees[b]))]))

        def spoil(c):
            c.page_table[1, 2] = -7

        pool, out = answer(spoil, "page_table")
        for x in (pool.k, pool.v):
            x[pool.table[1, 2].long()] = 0
        rows = [(b, visible_slots(t, i, total[b])) for b, t in enumerate(trees) for i in range(len(t))]
        close(out, *attention_over(pool, q, rows))
        wrong = list(parents)
        wrong[8], wrong[14] = 4, -3
        pool, out = answer(lambda c: None, "parent", parents=wrong, total=[40, 100, 10])
        bad = [wrong[a:b] for a, b in zip(cu, cu[1:])]
        close(out, *attention_over(pool, q, [(b, visible_slots(t, i, (40, 100, 10)[b])) for b, t in enumerate(bad)
                                             for i in range(len(t))]))
        pool, out = answer(lambda c: None, "cu_seqlens", cu=[0, 6, 40, 50], total=[40, 100, 10])
        close(out[:6], *attention_over(pool, q[:6], rows[:6]))
        assert (out[6:] == 7.0).all()
        answer(lambda c: None, "cu_seqlens", cu=[-1, -1, -1, -1], total=[40, 100, 10])
