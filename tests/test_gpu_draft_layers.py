"""Accept, keep and fork against plain forms, row by row."""
import random

import pytest
import torch

from vla_abft_estimate_b200.paged import PagedKVCache, PagedLayers

from .draft_reference import accepted, chain, i32, packed, path_to, random_tree
from .paged_reference import Pool
from .test_gpu_paged import BF16, F16, bits

pytestmark = pytest.mark.gpu


def layers_of(dev, lens, *, kv_heads=2, page=16, d=64, dtype=BF16, layers=3, joint=True, spare=2, extra_columns=0):
    """Pools of random bits (every slot differs), one table, one array of lengths."""
    pool = Pool(lens, kv_heads, page, d, dtype, spare=spare, extra_columns=extra_columns)
    table, seq_lens = pool.table.clamp(min=0).to(dev), i32(list(lens), dev)
    g = torch.Generator().manual_seed(len(lens))
    caches = []
    for _ in range(layers):
        both = torch.randint(-2 ** 15, 2 ** 15, (pool.k.shape[0], 2, *pool.k.shape[1:]), generator=g, dtype=torch.int16)
        x = both.view(dtype).to(dev)
        k, v = (x[:, 0], x[:, 1]) if joint else (x[:, 0].contiguous(), x[:, 1].contiguous())
        caches.append(PagedKVCache(k, v, table, seq_lens))
    return PagedLayers(caches)


def contents(layers):
    """[layers, 2, pages, kv_heads, page, d] as whole numbers, on the host."""
    return torch.stack([torch.stack((bits(c.k_pages), bits(c.v_pages))) for c in layers.layers])


# ---- accept ---------------------------------------------------------------------
def drafted(trees, seed, vocabulary=4):
    """Ids and answers of a small vocabulary, so that paths of several rows are confirmed, and equals occur."""
    r = random.Random(seed)
    n = sum(map(len, trees))
    return [r.randrange(vocabulary) for _ in range(n)], [r.randrange(vocabulary) for _ in range(n)]


def check_accept(dev, trees, ids, answers, dtype=torch.int64, pad=0, bad=False):
    layers = layers_of(dev, [1] * len(trees), layers=1)
    cu, parents = packed(trees)
    kept, counts, token = layers.accept(i32(cu, dev), i32(parents + [0] * pad, dev),
                                        torch.tensor(ids + [0] * pad, dtype=dtype, device=dev),
                                        torch.tensor(answers + [0] * pad, dtype=dtype, device=dev))
    assert kept.dtype == counts.dtype == torch.int32 and token.dtype == dtype
    want_kept, want_counts, want_token = [], [], []
    for b, tree in enumerate(trees):
        here = slice(cu[b], cu[b + 1])
        path, last = accepted(tree, ids[here], answers[here])
        want_kept += path + [-1] * (len(tree) - len(path))
        want_counts.append(len(path))
        want_token.append(last)
    assert kept.tolist() == want_kept + [-1] * pad
    assert counts.tolist() == want_counts
    assert token.tolist() == want_token
    if bad:
        with pytest.raises(ValueError, match="parent"):
            layers.check_status()
    layers.check_status()
    return want_counts


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("vocabulary", [1, 2, 4, 50])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 127, 300, 1024, 1025, 2600])
def test_accept_sizes(cuda_device, n, vocabulary, dtype):
    trees = [random_tree(n, n), random_tree(max(1, n // 3), 5, roots=2)]
    check_accept(cuda_device, trees, *drafted(trees, n, vocabulary), dtype)


@pytest.mark.parametrize("n", [40, 1500])
def test_accept_chains_and_stars(cuda_device, n):
    for tree in (chain(n), [-1] + [0] * (n - 1), [-1] * n):
        ids, answers = [3] * n, [3] * n
        check_accept(cuda_device, [tree], ids, answers)
        if n > 20:
            answers[n // 2] = 4  # a chain that breaks half way
            check_accept(cuda_device, [tree, tree], ids * 2, answers * 2)


def test_accept_batches_idle_sequences_and_rows_behind(cuda_device):
    for batch in (1, 33, 300):
        trees = [random_tree((b * 13) % 40 if b % 5 != 4 else 0, b) for b in range(batch)]
        counts = check_accept(cuda_device, trees, *drafted(trees, batch, 2), pad=batch % 7)
        assert max(counts) > 1 or batch == 1
    check_accept(cuda_device, [[], []], [], [], pad=5)
    check_accept(cuda_device, [[], []], [], [])


def test_accept_wide_tokens(cuda_device):
    """Tokens of 64 bits that agree in their lower half only are different."""
    check_accept(cuda_device, [chain(3)], [0, 5, 7], [5 + 2 ** 40, 7, -2 ** 62])
    check_accept(cuda_device, [chain(3)], [0, 5 + 2 ** 40, 7], [5 + 2 ** 40, 7, -2 ** 62])


@pytest.mark.parametrize("n", [50, 1300])
def test_accept_bad_parents_confirm_nothing(cuda_device, n):
    tree = random_tree(n, 2)
    for at, up in ((0, 0), (5, 5), (9, n - 1), (17, -2), (33, 2 ** 31 - 1), (40, -2 ** 31)):
        tree[at] = up
    check_accept(cuda_device, [tree, chain(4)], [1] * (n + 4), [1] * (n + 4), bad=True)


def test_accept_bad_boundaries(cuda_device):
    """What lies outside the rows is no sequence's; nothing is written elsewhere."""
    dev = cuda_device
    layers = layers_of(dev, [1, 1, 1], layers=1)
    one = torch.ones(9, dtype=torch.int64, device=dev)
    for bounds, counts in (((0, 3, 20, 30), [3, 0, 0]), ((-4, 3, 6, 9), [0, 3, 3]), ((5, 7, 8, 9), [2, 1, 1]),
                           ((0, 2 ** 31 - 1, -2 ** 31, 4), [0, 0, 0])):
        kept, got, token = layers.accept(i32(bounds, dev), i32([-1, 0, 1] * 3, dev), one, one)
        first = i32(bounds, dev)
        want = []
        for b in range(3):
            lo, hi = bounds[b], bounds[b + 1]
            rows = ([-1, 0, 1] * 3)[lo:hi] if 0 <= lo <= hi <= 9 else []
            want.append(len(accepted(rows, [1] * 9, [1] * 9)[0]))
        assert got.tolist() == want
        assert kept.min() >= -1 and kept.max() < 9 and first.tolist() == list(bounds)
        with pytest.raises(ValueError):
            layers.check_status()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("n", [1, 2, 7])
def test_accept_results_are_tensors_of_their_own(cuda_device, dtype, n):
    dev = cuda_device
    trees = [chain(n)] * 3
    layers = layers_of(dev, [1] * 3, layers=1)
    cu, parents = packed(trees)
    ids = torch.ones(3 * n, dtype=dtype, device=dev)
    for inference in (False, True):
        with torch.inference_mode(inference):
            got = layers.accept(i32(cu, dev), i32(parents, dev), ids, ids)
            want = [list(range(n)) * 3, [n] * 3, [1] * 3]
            assert [x.tolist() for x in got] == want
            assert all(x.is_contiguous() and not x._is_view() and x.is_inference() == inference for x in got)
            before = [0 if inference else x._version for x in got]
            for k, x in enumerate(got):  # a write reaches one of them only
                x.fill_(-9)
                want[k] = [-9] * len(want[k])
                assert [y.tolist() for y in got] == want
                assert inference or [y._version - v for y, v in zip(got, before)] == [int(j <= k) for j in range(3)]
        kept = got[0].clone()
        del got
        assert kept.tolist() == [-9] * (3 * n)


def test_accept_refusals(cuda_device):
    dev = cuda_device
    layers = layers_of(dev, [9, 9], layers=1)
    cu, up = i32([0, 2, 6], dev), i32([-1] * 6, dev)
    x = torch.zeros(6, dtype=torch.int64, device=dev)
    for args in ((cu[:2], up, x, x), (cu.long(), up, x, x), (cu, up[:5], x, x), (cu, up, x[:5], x), (cu, up, x, x.int()),
                 (cu, up, x.float(), x.float()), (cu, up, x.cpu(), x.cpu()), (cu, up, x[None], x[None]), (cu, up.cpu(), x, x)):
        with pytest.raises((ValueError, AttributeError)):
            layers.accept(*args)
    wide = torch.zeros(12, dtype=torch.int64, device=dev)
    kept, counts, token = layers.accept(cu, up, wide[::2], wide[1::2])  # read through a copy
    assert counts.tolist() == [1, 1] and kept.tolist() == [0, -1, 0, -1, -1, -1] and token.tolist() == [0, 0]


# ---- keep -------------------------------------------------------------------------
def check_keep(dev, new, total, paths, *, lens_out=False, **more):
    layers = layers_of(dev, total, **more)
    c = layers.layers[0]
    want = contents(layers)
    before = want.clone()
    table, page = c.page_table.cpu(), c.page_size
    cu, _ = packed([[0] * n for n in new])
    flat = []
    for n, path in zip(new, paths):
        flat += path + [-7] * (n - len(path))
    for b, path in enumerate(paths):
        base = total[b] - new[b]
        for i, k in enumerate(path):
            (p0, s0), (p1, s1) = divmod(base + k, page), divmod(base + i, page)
            want[:, :, table[b, p1], :, s1] = before[:, :, table[b, p0], :, s0]
    out = torch.full((len(new),), -5, dtype=torch.int32, device=dev) if lens_out else None
    got = layers.keep(i32(cu, dev), i32(flat, dev), i32([len(p) for p in paths], dev), lens_out=out)
    layers.check_status()
    lens = [t - n + len(p) for t, n, p in zip(total, new, paths)]
    assert got.tolist() == lens
    assert got is (out if lens_out else layers.seq_lens)
    assert layers.seq_lens.tolist() == (list(total) if lens_out else lens)
    assert torch.equal(contents(layers), want)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("d,kv_heads,layers", [(64, 1, 1), (128, 4, 28), (128, 2, 2), (64, 32, 5)])
def test_keep_paths(cuda_device, d, kv_heads, layers, page):
    trees = [random_tree(26, 1), random_tree(1, 2), random_tree(40, 3)]
    paths = [path_to(trees[0], 25), [0], path_to(trees[2], 39)]
    check_keep(cuda_device, [26, 1, 40], [75, 1, 40], paths, d=d, kv_heads=kv_heads, layers=layers, page=page)


@pytest.mark.parametrize("name,n,path", [
    ("none", 5, []), ("all", 40, list(range(40))), ("last", 30, [29]), ("every second", 60, list(range(0, 60, 2))),
    ("all but the first", 70, list(range(1, 70))), ("all but one inside", 70, [i for i in range(70) if i != 33]),
    ("far", 300, [0, 1, 298, 299]), ("many", 700, list(range(1, 700))), ("many, some", 900, list(range(100, 900, 3))),
    ("as many as are held", 300, list(range(44, 300))), ("one more", 300, list(range(43, 300)))])
@pytest.mark.parametrize("joint", [True, False])
def test_keep_overlapping_moves(cuda_device, name, n, path, joint):
    check_keep(cuda_device, [n], [n + 21], [path], joint=joint)
    check_keep(cuda_device, [n, 3], [n, 20], [path, [0, 2]], joint=joint, lens_out=True, dtype=F16, layers=1)


def test_keep_batches(cuda_device):
    for batch in (1, 40, 200):
        trees = [random_tree((b * 13) % 30 if b % 5 != 4 else 0, b) for b in range(batch)]
        paths = [path_to(t, len(t) - 1 - b % 2) if len(t) > 1 else [] for b, t in enumerate(trees)]
        check_keep(cuda_device, [len(t) for t in trees], [len(t) + (b * 7) % 50 if t else 0 for b, t in enumerate(trees)],
                   paths, layers=2, lens_out=batch == 40)


BAD_KEEP = {"falling": dict(kept=[0, 3, 2, -1]), "twice": dict(kept=[1, 1, -1, -1], count=2), "below": dict(kept=[-1, 2, 3, -1]),
            "beyond": dict(kept=[0, 4, -1, -1], count=2), "far": dict(kept=[0, 2 ** 31 - 1, -1, -1], count=2),
            "count below": dict(count=-1), "count beyond": dict(count=5), "count far": dict(count=2 ** 31 - 1),
            "length below": dict(length=3), "length negative": dict(length=-4), "length beyond": dict(length=49),
            "length far": dict(length=2 ** 31 - 1), "source page": dict(page=(2, 1000)), "page below": dict(page=(2, -1)),
            "destination page": dict(page=(1, 1000)), "boundaries": dict(cu=[0, 4, 9]), "fall": dict(cu=[4, 3, 8]),
            "start": dict(cu=[1, 5, 8])}


def good_keep(cu, b, rows, kept, count, length, table, page, num_pages):
    """The path of sequence b, or None when anything of it is wrong."""
    lo, hi = cu[b], cu[b + 1]
    if not 0 <= lo <= hi <= rows or (b == 0 and lo != 0) or not 0 <= count <= hi - lo or not hi - lo <= length <= 48:
        return None
    path = kept[lo:lo + count]
    if any(not last < k < hi - lo for last, k in zip([-1] + path, path)):
        return None
    base = length - (hi - lo)
    if any(not 0 <= table[b][(base + at) // page] < num_pages for at in path + list(range(count))):
        return None
    return path


@pytest.mark.parametrize("lens_out", [False, True])
@pytest.mark.parametrize("case", BAD_KEEP)
def test_keep_leaves_a_bad_sequence(cuda_device, case, lens_out):
    """A sequence with anything wrong stays as it was, its length too; the other is done."""
    dev = cuda_device
    given = dict(kept=[0, 2, 3, -1], count=3, length=35, page=None, cu=[0, 4, 8])
    given.update(BAD_KEEP[case])
    layers = layers_of(dev, [35, 35], layers=2)
    layers.seq_lens[0] = given["length"]
    if given["page"]:
        layers.page_table[0, given["page"][0]] = given["page"][1]
    before = contents(layers)
    want, lens, table = before.clone(), layers.seq_lens.tolist(), layers.page_table.tolist()
    kept, counts = given["kept"] + [1, 3, -1, -1], [given["count"], 2]
    want_lens, left = list(lens), 0
    for b in range(2):
        path = good_keep(given["cu"], b, 8, kept, counts[b], lens[b], table, 16, before.shape[2])
        if path is None:
            left += 1
            continue
        base = lens[b] - (given["cu"][b + 1] - given["cu"][b])
        for i, k in enumerate(path):
            (p0, s0), (p1, s1) = divmod(base + k, 16), divmod(base + i, 16)
            want[:, :, table[b][p1], :, s1] = before[:, :, table[b][p0], :, s0]
        want_lens[b] = base + len(path)
    assert left >= 1
    out = torch.zeros(2, dtype=torch.int32, device=dev) if lens_out else None
    got = layers.keep(i32(given["cu"], dev), i32(kept, dev), i32(counts, dev), lens_out=out)
    assert got.tolist() == want_lens
    assert layers.seq_lens.tolist() == (lens if lens_out else want_lens)
    with pytest.raises(ValueError):
        layers.check_status()
    assert torch.equal(contents(layers), want)


def test_keep_refusals(cuda_device):
    dev = cuda_device
    layers = layers_of(dev, [30, 30])
    cu, kept, counts = i32([0, 4, 8], dev), i32([0] * 8, dev), i32([1, 1], dev)
    before = contents(layers)
    for args, more in (((cu[:2], kept, counts), {}), ((cu, kept.long(), counts), {}), ((cu, kept, counts[:1]), {}),
                       ((cu, kept.cpu(), counts), {}), ((cu, kept[None], counts), {}), ((cu, kept, counts), {"lens_out": counts[:1]}),
                       ((cu, kept, counts), {"lens_out": counts.long()}), ((cu, kept, None), {}), ((None, kept, counts), {})):
        with pytest.raises(ValueError):
            layers.keep(*args, **more)
    with pytest.raises(Exception, match="abft_kv_keep"):  # a part of the lengths themselves
        both = torch.zeros(3, dtype=torch.int32, device=dev)
        PagedLayers([PagedKVCache(c.k_pages, c.v_pages, c.page_table, both[:2]) for c in layers.layers]).keep(
            cu, kept, counts, lens_out=both[1:])
    assert torch.equal(contents(layers), before)


# ---- fork -------------------------------------------------------------------------
def check_fork(dev, lens, pairs, *, pages=None, bad=None, undone=(), rows=None, **more):
    """``pairs``: (source, destination); pairs in ``undone`` change nothing."""
    rows = rows or len(lens)
    layers = layers_of(dev, lens, spare=len(pairs) + 1, **more)
    c = layers.layers[0]
    page = c.page_size
    used = set(c.page_table.cpu().flatten().tolist()[:0])
    table, want_lens = c.page_table.cpu().clone(), layers.seq_lens.tolist()
    for b, n in enumerate(lens):
        used |= set(table[b, : -(-n // page)].tolist())
    free = [p for p in range(c.num_pages) if p not in used]
    pages = free[:len(pairs)] if pages is None else pages(free, table)
    want = contents(layers)
    before, old_table, old_lens = want.clone(), table.clone(), list(want_lens)
    for i, (s, d) in enumerate(pairs):
        if i in undone:
            continue
        n = old_lens[s]
        full, rest = divmod(n, page)
        table[d, :full] = old_table[s, :full]
        want_lens[d] = n
        if rest:
            table[d, full] = pages[i]
            want[:, :, pages[i], :, :rest] = before[:, :, old_table[s, full], :, :rest]
    src, dst = (i32([p[k] for p in pairs], dev) for k in (0, 1))
    assert layers.fork(src, dst, i32(pages, dev)) is None
    if bad is None:
        layers.check_status()
    else:
        with pytest.raises(ValueError, match=bad):
            layers.check_status()
    assert layers.seq_lens.tolist() == want_lens
    assert torch.equal(c.page_table.cpu(), table)
    assert torch.equal(contents(layers), want)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("d,kv_heads,layers", [(64, 1, 1), (128, 4, 28), (64, 32, 3)])
@pytest.mark.parametrize("length", [0, 1, 15, 16, 127, 128, 300])
def test_fork_lengths(cuda_device, length, d, kv_heads, layers, page):
    check_fork(cuda_device, [length, 300, 0, 40], [(0, 2), (0, 3)], d=d, kv_heads=kv_heads, layers=layers, page=page)


def test_fork_many(cuda_device):
    lens = [(7 * b) % 90 for b in range(20)] + [0] * 60
    check_fork(cuda_device, lens, [(i % 20, 20 + i) for i in range(60)], joint=False)
    check_fork(cuda_device, lens, [(0, 79)], dtype=F16, extra_columns=3000)
    r = random.Random(1)
    check_fork(cuda_device, lens, [(r.randrange(20), d) for d in r.sample(range(20, 80), 33)])
    lens = [33] * 5 + [0] * 700
    check_fork(cuda_device, lens, [(i % 5, 5 + i) for i in range(700)], layers=1)


def test_fork_without_pair(cuda_device):
    check_fork(cuda_device, [20, 30, 40, 0], [(0, 3), (-1, 1), (2, -1), (-1, -1)], undone=(1, 2, 3))
    # a place without a pair is in nobody's way
    check_fork(cuda_device, [20, 30, 40, 0], [(0, 3), (-1, 3), (3, -1)], undone=(1, 2),
               pages=lambda free, table: [free[0], free[0], -1])
    layers = layers_of(cuda_device, [3, 0])
    none = i32([], cuda_device)
    layers.fork(none, none, none)
    layers.check_status()


@pytest.mark.parametrize("pairs,undone", [
    ([(0, 2), (1, 2)], (0, 1)), ([(0, 1), (1, 2)], (0,)), ([(0, 0), (1, 3)], (0,)), ([(0, 2), (0, 2)], (0, 1)),
    ([(0, 1), (1, 0)], (0, 1)), ([(4, 2), (0, 3)], (0,)), ([(0, 4), (1, 2)], (0,)), ([(-2, 2), (1, 3)], (0,)),
    ([(0, -5), (1, 3)], (0,)), ([(2 ** 31 - 1, 2), (1, 3)], (0,)), ([(0, 2 ** 31 - 1), (1, 3)], (0,))])
def test_fork_refuses_pairs_that_meet(cuda_device, pairs, undone):
    check_fork(cuda_device, [20, 30, 0, 0], pairs, bad="fork", undone=undone)


def test_fork_pages(cuda_device):
    """A page named twice is refused where it is needed; one that is not needed is not looked at; bad ones are told."""
    dev, lens = cuda_device, [20, 48, 30, 0, 0, 0]
    check_fork(dev, lens, [(0, 3), (2, 4)], pages=lambda free, table: [free[0], free[0]], bad="fork", undone=(0, 1))
    check_fork(dev, lens, [(0, 3), (1, 4)], pages=lambda free, table: [free[0], -1])
    check_fork(dev, lens, [(1, 3), (0, 4)], pages=lambda free, table: [10 ** 9, free[1]])
    check_fork(dev, lens, [(0, 3), (2, 4)], pages=lambda free, table: [-1, free[0]], bad="page", undone=(0,))
    check_fork(dev, lens, [(0, 3), (2, 4)], pages=lambda free, table: [10 ** 9, free[0]], bad="page", undone=(0,))
    check_fork(dev, lens, [(0, 3), (2, 4)], pages=lambda free, table: [int(table[0, 1]), free[0]], bad="page", undone=(0,))


@pytest.mark.parametrize("length,entry,bad", [(-1, None, "length"), (49, None, "length"), (2 ** 31 - 1, None, "length"),
                                              (20, 99999, "page"), (20, -1, "page")])
def test_fork_leaves_bad_sources(cuda_device, length, entry, bad):
    dev = cuda_device
    layers = layers_of(dev, [40, 33, 0, 0], spare=4)
    layers.seq_lens[0] = length
    if entry is not None:
        layers.page_table[0, 1] = entry
    before, table, lens = contents(layers), layers.page_table.cpu(), layers.seq_lens.tolist()
    layers.fork(i32([0], dev), i32([2], dev), i32([5], dev))
    with pytest.raises(ValueError, match=bad):
        layers.check_status()
    assert torch.equal(contents(layers), before) and torch.equal(layers.page_table.cpu(), table)
    assert layers.seq_lens.tolist() == lens


def test_fork_refusals_and_layers_that_do_not_match(cuda_device):
    dev = cuda_device
    layers = layers_of(dev, [30, 30])
    x = i32([0], dev)
    for args in ((x.long(), x, x), (x, i32([0, 1], dev), x), (x, x, x[None]), (x, x, x.cpu()), (None, x, x)):
        with pytest.raises(ValueError):
            layers.fork(*args)
    with pytest.raises(TypeError):
        PagedLayers([])
    with pytest.raises(TypeError):
        PagedLayers([layers])
    one, other = layers.layers[0], layers_of(dev, [30, 30]).layers[0]
    with pytest.raises(ValueError, match="share"):
        PagedLayers([one, other])
    with pytest.raises(ValueError, match="own"):
        PagedLayers([one, one])
    with pytest.raises(ValueError, match="own"):
        PagedLayers([PagedKVCache(one.k_pages, one.k_pages, one.page_table, one.seq_lens)])


@pytest.mark.parametrize("layers", [64, 65, 512])
def test_many_layers(cuda_device, layers):
    check_keep(cuda_device, [30, 2], [40, 20], [[0, 3, 4, 29], [1]], layers=layers, kv_heads=1)
    check_fork(cuda_device, [21, 30, 0, 0], [(0, 2), (1, 3)], layers=layers, kv_heads=1)


def test_more_layers_are_refused(cuda_device):
    with pytest.raises(ValueError, match="512"):
        PagedLayers(layers_of(cuda_device, [3], layers=1).layers * 513)


def test_the_object_may_go_while_its_calls_run(cuda_device):
    """Nothing of the object's is read by the GPU."""
    dev = cuda_device
    layers = layers_of(dev, [400] * 8, layers=28, d=128, kv_heads=4)
    caches = layers.layers
    path = list(range(1, 200))
    before = contents(layers)
    stream = torch.cuda.Stream()
    cu, kept, counts = i32([200 * i for i in range(9)], dev), i32((path + [-1]) * 8, dev), i32([199] * 8, dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(2_000_000)
        layers.keep(cu, kept, counts)
    del layers
    junk = [torch.full((1 << 16,), -1, dtype=torch.int64, device=dev) for _ in range(64)]
    torch.cuda.synchronize()
    del junk
    layers = PagedLayers(caches)
    table, want = layers.page_table.cpu(), before.clone()
    for b in range(8):
        for i, k in enumerate(path):
            (p0, s0), (p1, s1) = divmod(200 + k, 16), divmod(200 + i, 16)
            want[:, :, table[b, p1], :, s1] = before[:, :, table[b, p0], :, s0]
    assert torch.equal(contents(layers), want) and layers.seq_lens.tolist() == [399] * 8
