"""The paged cache operators run together, as a decoder uses them: chunks and
single tokens of a batch, CUDA graphs, streams, large pools, the model."""
import contextlib

import pytest
import torch

from vla_abft_estimate_b200.abft import AbftConfig, AbftInjector, AbftStatsCollector, CheapSumChecker
from vla_abft_estimate_b200.paged import PagedKVCache, rope_table
from vla_abft_estimate_b200.workloads import build_qwen2

from .paged_reference import Pool, attention, rotated
from .test_gpu_paged import BF16, F16, bits, close, owners_of

pytestmark = pytest.mark.gpu


def stored(cache):
    """The cache's content as a Pool, for the 64-bit reference."""
    pool = Pool.__new__(Pool)
    pool.k, pool.v, pool.table = cache.k_pages.cpu(), cache.v_pages.cpu(), cache.page_table.cpu()
    pool.page, pool.d, pool.kv_heads, pool.dtype = cache.page_size, cache.head_dim, cache.kv_heads, cache.dtype
    return pool


@pytest.mark.parametrize("heads,kv_heads,d,page,dtype", [(28, 4, 128, 16, BF16), (8, 8, 64, 32, F16)])
def test_chunks_then_tokens(cuda_device, heads, kv_heads, d, page, dtype):
    """Ragged prompts in two chunks, then single tokens: every step's keys,
    values and outputs against the formulas on what the cache holds."""
    dev = cuda_device
    batch, per = 4, -(-400 // page)
    g = torch.Generator().manual_seed(5)
    table = torch.randperm(batch * per, generator=g).int().view(batch, per).to(dev)
    lens = torch.zeros(batch, dtype=torch.int32, device=dev)
    nan = float("nan")
    cache = PagedKVCache(torch.full((batch * per, kv_heads, page, d), nan, dtype=dtype, device=dev),
                         torch.full((batch * per, kv_heads, page, d), nan, dtype=dtype, device=dev), table, lens)
    rope = rope_table(400, d, device=dev)
    total = [0] * batch
    steps = [[100, 1, 257, 0], [60, 130, 3, 16]] + [None] * 3
    for new in steps:
        one = new is None
        new = [1] * batch if one else new
        total = [t + n for t, n in zip(total, new)]
        lens.copy_(torch.tensor(total, dtype=torch.int32))
        tokens = sum(new)
        q, k, v = (torch.randn(tokens, h, d, generator=g).to(dtype) for h in (heads, kv_heads, kv_heads))
        cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device=dev)
        rq = cache.append(q.to(dev), k.to(dev), v.to(dev), rope, cu_seqlens=None if one else cu)
        out = cache.decode(rq) if one else cache.prefill(rq, cu)
        cache.check_status()
        pos = torch.tensor([t - n + i for n, t in zip(new, total) for i in range(n)])
        close(rq, *rotated(q, pos))
        owner = torch.tensor([b for b, n in enumerate(new) for _ in range(n)], dtype=torch.int64)
        page_of = table.cpu()[owner, pos // page].long()
        close(cache.k_pages.cpu()[page_of, :, pos % page], *rotated(k, pos))
        assert torch.equal(bits(cache.v_pages.cpu()[page_of, :, pos % page]), bits(v))
        close(out, *attention(stored(cache), rq.cpu(), owners_of(new, total)))


def decode_state(dev, seed=0, lens=(40, 700, 3)):
    pool = Pool([n + 20 for n in lens], 4, 16, 128, BF16, seed=seed)
    cache = pool.device_cache(dev, PagedKVCache)
    cache.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(len(lens), h, 128, generator=g).to(BF16).to(dev) for h in (28, 4, 4))
    return cache, q, k, v, rope_table(800, 128, device=dev)


def test_captured_decode_step_follows_the_lengths(cuda_device):
    """append + decode in a graph, the lengths advanced in it, against eager steps."""
    dev = cuda_device

    def step(cache, q, k, v, rope):
        cache.seq_lens.add_(1)
        return cache.decode(cache.append(q, k, v, rope))

    eager = decode_state(dev)
    want = [step(*eager).clone() for _ in range(6)]
    state = decode_state(dev)
    step(*state)  # first calls outside the capture, then the lengths as they were
    state[0].seq_lens.sub_(1)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(*state)
    for w in want:
        g.replay()
        assert torch.equal(out, w)
    state[0].check_status()


def test_two_graphs_replay_at_once(cuda_device):
    """Scratch belongs to each captured call: two graphs on two streams give what each gives alone."""
    dev = cuda_device
    runs = []
    for seed in range(2):
        cache, q, *_ = decode_state(dev, seed, (5000, 300, 9000))
        cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev)
        want = cache.decode(q).clone(), cache.prefill(q, cu, num_splits=8).clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(4):
                got = cache.decode(q), cache.prefill(q, cu, num_splits=8)
        runs.append((g, got, want, torch.cuda.Stream(), (cache, q, cu)))  # what the graph reads stays alive
    torch.cuda.synchronize()
    for _ in range(10):
        for g, _, _, stream, _ in runs:
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for _, got, want, _, _ in runs:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_calls_on_two_streams_at_once(cuda_device):
    dev = cuda_device
    runs = []
    for seed in range(2):
        cache, q, *_ = decode_state(dev, seed, (5000, 300, 9000))
        cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev)
        runs.append((cache, q, cu, cache.decode(q), cache.prefill(q, cu, num_splits=8), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (cache, q, cu, _, _, stream) in enumerate(runs):
            with torch.cuda.stream(stream):
                got[i].append((cache.decode(q), cache.prefill(q, cu, num_splits=8)))
    torch.cuda.synchronize()
    for (_, _, _, a, b, _), outs in zip(runs, got):
        assert all(torch.equal(x, a) and torch.equal(y, b) for x, y in outs)


def test_offsets_beyond_32_bits(cuda_device):
    """Pages 2^31 elements into the pool: three pages of a strided 4.3 GB buffer."""
    dev = cuda_device
    stride = (1 << 30) + 4096
    flat = torch.empty(2 * stride + 2 * 4 * 16 * 128 + 64, dtype=BF16, device=dev)  # only the pages are touched
    shape, inner = (3, 4, 16, 128), (16 * 128, 128, 1)
    k = flat.as_strided(shape, (stride,) + inner)
    v = flat.as_strided(shape, (stride,) + inner, 4 * 16 * 128)
    pool = Pool([48], 4, 16, 128, BF16, spare=0)
    cache = PagedKVCache(k, v, pool.table.to(dev), torch.tensor([48], dtype=torch.int32, device=dev))
    k.copy_(pool.k)
    v.copy_(pool.v)
    q = torch.randn(3, 28, 128, generator=torch.Generator().manual_seed(1)).to(BF16)
    want, tol = attention(pool, q, [(0, 46), (0, 47), (0, 48)])
    cu = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    close(cache.prefill(q.to(dev), cu), want, tol)
    close(cache.decode(q[2:].to(dev)), want[2:], tol[2:])
    new = torch.randn(48, 4, 128, generator=torch.Generator().manual_seed(2)).to(BF16).to(dev)
    cache.append(None, new, new, cu_seqlens=torch.tensor([0, 48], dtype=torch.int32, device=dev))
    held = pool.table[0].long()
    assert torch.equal(k[held.to(dev)].transpose(1, 2).reshape(48, 4, 128), new)
    cache.check_status()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_scores_stay_in_the_rows_that_see_them(cuda_device, value):
    """A key that is not finite makes the rows that see it (of its kv head)
    what 64-bit arithmetic makes them, and no other row."""
    dev = cuda_device
    pool = Pool([300, 200], 2, 16, 64, F16)
    at = pool.table[0, 150 // 16].long().item()
    pool.k[at, 1, 150 % 16, 7] = value
    cache = pool.device_cache(dev, PagedKVCache)
    q = torch.randn(200, 6, 64, generator=torch.Generator().manual_seed(4)).to(F16)
    cu = torch.tensor([0, 199, 200], dtype=torch.int32, device=dev)
    owners = [(0, 102 + i) for i in range(199)] + [(1, 200)]
    got = cache.prefill(q.to(dev), cu).cpu()
    one = cache.decode(torch.stack((q[198], q[199])).to(dev)).cpu()
    want, tol = attention(pool, q, owners)
    for have, ref, t in ((got, want, tol), (one, want[198:], tol[198:])):
        assert torch.equal(torch.isnan(have), torch.isnan(ref))
        fine = ~torch.isnan(ref)
        close(have[fine], ref[fine], t[fine])
    assert torch.isfinite(got[:48]).all() and torch.isfinite(got[:, :3]).all() and torch.isfinite(got[199]).all()


def test_captured_prefill_follows_boundaries_and_lengths(cuda_device):
    """One capture over 60 packed rows, replayed as other batches come: other
    chunk lengths, empty chunks, rows behind the last one."""
    dev = cuda_device
    pool = Pool([900, 120, 400], 2, 16, 64, BF16)
    cache = pool.device_cache(dev, PagedKVCache)
    q = torch.randn(60, 14, 64, generator=torch.Generator().manual_seed(8)).to(BF16)
    dq, out = q.to(dev), torch.empty(60, 14, 64, dtype=BF16, device=dev)
    cu = torch.tensor([0, 20, 40, 60], dtype=torch.int32, device=dev)
    cache.prefill(dq, cu, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.prefill(dq, cu, out=out)
    for new, total in (((20, 20, 20), (900, 120, 400)), ((60, 0, 0), (61, 5, 0)), ((1, 1, 1), (900, 1, 33)),
                       ((0, 50, 7), (0, 50, 399))):
        cu.copy_(torch.tensor([0, *torch.tensor(new).cumsum(0)], dtype=torch.int32))
        cache.seq_lens.copy_(torch.tensor(total, dtype=torch.int32))
        out.fill_(7.0)
        g.replay()
        want, tol = attention(pool, q[:sum(new)], owners_of(new, total))
        close(out[:sum(new)], want, tol)
        assert (out[sum(new):] == 7.0).all()
    cache.check_status()


def test_many_sequences(cuda_device):
    """A batch of 1,000 sequences: every scan over the batch takes many rounds."""
    dev = cuda_device
    total = [(i * 29) % 61 for i in range(1000)]
    pool = Pool(total, 1, 16, 64, F16)
    cache = pool.device_cache(dev, PagedKVCache)
    q = torch.randn(1000, 3, 64, generator=torch.Generator().manual_seed(9)).to(F16)
    want, tol = attention(pool, q, list(enumerate(total)))
    close(cache.decode(q.to(dev)), want, tol)
    new = [min(1, t) for t in total]
    rows = [b for b, n in enumerate(new) if n]
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0)], dtype=torch.int32, device=dev)
    close(cache.prefill(q[rows].to(dev), cu), want[rows], tol[rows])
    k = torch.randn(1000, 1, 64, generator=torch.Generator().manual_seed(10)).to(F16).to(dev)
    cache.append(None, k, k)
    last = torch.tensor([t - 1 for t in total if t])
    page_of = pool.table[torch.tensor(rows), last // 16].long()
    assert torch.equal(cache.v_pages.cpu()[page_of, 0, last % 16], k.cpu()[rows, 0])
    cache.check_status()


@pytest.mark.parametrize("batch", [33, 129, 2100])
def test_batches_that_a_warp_scans_in_parts(cuda_device, batch):
    """More sequences than lanes, than boundaries counted at once, and than 32
    for each lane: empty ones, and none, one or several new tokens each."""
    dev = cuda_device
    total = [(i * 29) % 47 for i in range(batch)]
    new = [min(t, (0, 1, 3)[i % 3]) for i, t in enumerate(total)]
    pool = Pool(total, 1, 16, 64, BF16)
    cache = pool.device_cache(dev, PagedKVCache)
    g = torch.Generator().manual_seed(12)
    q = torch.randn(batch, 2, 64, generator=g).to(BF16)
    want, tol = attention(pool, q, list(enumerate(total)))
    close(cache.decode(q.to(dev)), want, tol)
    close(cache.decode(q.to(dev), num_sms=3), want, tol)
    rows = sum(new)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0)], dtype=torch.int32, device=dev)
    q = torch.randn(rows + 5, 2, 64, generator=g).to(BF16)
    want, tol = attention(pool, q[:rows], owners_of(new, total))
    for splits in (0, 2):
        out = torch.full_like(q, 7.0).to(dev)
        cache.prefill(q.to(dev), cu, out=out, num_splits=splits)
        close(out[:rows], want, tol)
        assert (out[rows:] == 7.0).all()
    v = torch.randn(rows + 5, 1, 64, generator=g).to(BF16)
    cache.append(None, v.to(dev), v.to(dev), cu_seqlens=cu)
    place = [(b, t - n + i) for b, (n, t) in enumerate(zip(new, total)) for i in range(n)]
    b, pos = torch.tensor(place).unbind(1)
    stored = cache.v_pages.cpu()[pool.table[b, pos // 16].long(), 0, pos % 16]
    assert torch.equal(stored, v[:rows, 0])
    cache.check_status()


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("kv_heads,group", [(1, 3), (2, 12), (4, 7), (1, 24)])
@pytest.mark.parametrize("lens", [(510,), (0,), (1, 33, 0), (500, 130, 31, 257, 64, 448, 5), [37 * i % 513 for i in range(16)]])
def test_decode_by_clusters(cuda_device, lens, kv_heads, group, d, dtype):
    """Tables of 512 slots: clusters of 8, 4 or 2 CTAs a segment by the number of
    segments (1 to 64); lengths that leave CTAs, or all, without a tile."""
    dev = cuda_device
    pool = Pool(lens, kv_heads, 16, d, dtype, extra_columns=32 - max(1, (max(lens) + 15) // 16))
    cache = pool.device_cache(dev, PagedKVCache)
    assert cache.max_pages == 32
    q = torch.randn(len(lens), kv_heads * group, d, generator=torch.Generator().manual_seed(13)).to(dtype)
    want, tol = attention(pool, q, list(enumerate(lens)))
    x = q.to(dev)
    for sms in (0, 1, 9):  # 1: the list on one SM
        close(cache.decode(x, num_sms=sms), want, tol)
    first = cache.decode(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.decode(x)
    for _ in range(3):
        out.fill_(7.0)
        graph.replay()
        assert torch.equal(out, first)
    cache.check_status()


@pytest.mark.parametrize("kv_heads,group,d,lens,new", [
    (1, 7, 128, (5000, 3, 700), (9, 3, 5)),             # one sequence cut, the others whole
    (4, 2, 64, (4097,), (70,)),                          # blocks of unlike length
    (2, 16, 128, (2300, 2299, 0, 1), (1, 20, 0, 1)),
    (1, 4, 64, [3000] + [40 + i for i in range(39)], [33] + [1 + i % 3 for i in range(39)]),  # two sequences a lane
])
def test_pieces_chosen_for_the_lengths(cuda_device, kv_heads, group, d, lens, new):
    """Tables far wider than the sequences; lengths that change between the
    replays of a graph, whose pieces are chosen each time."""
    dev = cuda_device
    pool = Pool(lens, kv_heads, 16, d, BF16, extra_columns=1500)
    cache = pool.device_cache(dev, PagedKVCache)
    rows = sum(new)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0)], dtype=torch.int32, device=dev)
    q = torch.randn(rows + 3, kv_heads * group, d, generator=torch.Generator().manual_seed(14)).to(BF16)
    x, out = q.to(dev), torch.empty_like(q, device=dev)
    cache.prefill(x, cu, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.prefill(x, cu, out=out)
    for short in (0, 1, 0):
        now = [max(n, t - short * 900) for t, n in zip(lens, new)]
        cache.seq_lens.copy_(torch.tensor(now, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        want, tol = attention(pool, q[:rows], owners_of(new, now))
        close(out[:rows], want, tol)
        assert (out[rows:] == 7.0).all()
    cache.check_status()
    cache.seq_lens.zero_()  # rows without keys
    graph.replay()
    assert (out[:rows] == 0).all()
    with pytest.raises(ValueError, match="length"):
        cache.check_status()


def test_result_over_q_and_a_slice_of_a_wider_table(cuda_device):
    dev = cuda_device
    pool = Pool([2000, 77, 300], 4, 16, 128, BF16)
    wide = torch.full((5, 400), -1, dtype=torch.int32, device=dev)
    wide[1:4, 7:7 + pool.table.shape[1]] = pool.table.to(dev)
    cache = PagedKVCache(pool.k.to(dev), pool.v.to(dev), wide[1:4, 7:7 + pool.table.shape[1]],
                         torch.tensor([0, 2000, 77, 300], dtype=torch.int32, device=dev)[1:])
    q = torch.randn(43, 28, 128, generator=torch.Generator().manual_seed(8)).to(BF16)
    new = (40, 1, 2)
    cu = torch.tensor([0, 40, 41, 43], dtype=torch.int32, device=dev)
    want, tol = attention(pool, q, owners_of(new, (2000, 77, 300)))
    for splits in (1, 4):
        x = q.to(dev)
        assert cache.prefill(x, cu, out=x, num_splits=splits) is x
        close(x, want, tol)
    newest = [39, 40, 42]
    for sms in (0, 5):
        x = q[newest].to(dev)
        assert cache.decode(x, out=x, num_sms=sms) is x
        close(x, want[newest], tol[newest])
    with pytest.raises(AttributeError):
        cache.seq_lens = torch.zeros(3, dtype=torch.int32, device=dev)


def test_misaligned_rows_are_copied(cuda_device):
    cache, q, k, v, rope = decode_state(cuda_device)
    want_q = cache.append(q, k, v, rope)
    want = cache.decode(want_q)
    kept = bits(cache.k_pages)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)

    got = cache.append(shifted(q), shifted(k), shifted(v), rope)
    assert torch.equal(got, want_q) and torch.equal(bits(cache.k_pages), kept)
    assert torch.equal(cache.decode(shifted(want_q)), want)
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=cuda_device)
    assert torch.equal(cache.prefill(shifted(want_q), cu), cache.prefill(want_q, cu))
    with pytest.raises(ValueError, match="aligned"):
        cache.decode(want_q, out=shifted(want))


def test_python_refusals(cuda_device):
    cache, q, k, v, rope = decode_state(cuda_device)
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=cuda_device)
    dev = cuda_device
    for bad in (q[:2], q.float(), q[:, :27], q[..., :64], q.cpu(), q.half(), q[0], q[:, :0]):
        with pytest.raises(ValueError):
            cache.decode(bad)
    for bad in (k[:2], k[:, :3], k.float(), k.cpu()):
        with pytest.raises(ValueError):
            cache.append(q, bad, v, rope)
        with pytest.raises(ValueError):
            cache.append(q, k, bad, rope)
    for bad in (rope.half(), rope[:, :32], rope[::2], rope[:0], rope.cpu(), rope[..., 0]):
        with pytest.raises(ValueError):
            cache.append(q, k, v, bad)
    for bad in (cu[:3], cu.long(), cu.cpu(), cu[None], torch.zeros(8, dtype=torch.int32, device=dev)[::2]):
        with pytest.raises(ValueError):
            cache.prefill(q, bad)
        with pytest.raises(ValueError):
            cache.append(q, k, v, rope, cu_seqlens=bad)
    with pytest.raises(ValueError):
        cache.append(q[:2], k[:2], v[:2], rope)  # one row per sequence without cu_seqlens
    with pytest.raises(ValueError):
        cache.append(None, k, v, rope, q_out=q)
    with pytest.raises(TypeError):
        cache.decode([1.0])
    with pytest.raises(ValueError):
        cache.decode(q, out=torch.empty(3, 28, 64, dtype=BF16, device=dev))
    with pytest.raises(ValueError):
        cache.decode(q, out=torch.empty(1, 28, 128, dtype=BF16, device=dev).expand(3, 28, 128))
    with pytest.raises(ValueError):
        cache.decode(q, scale=float("inf"))
    with pytest.raises(ValueError):
        cache.prefill(q, cu, num_splits=-1)
    with pytest.raises(ValueError):
        cache.decode(q, num_sms=-1)
    wants_grad = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        cache.decode(wants_grad)
    with torch.no_grad():
        assert torch.equal(cache.decode(wants_grad), cache.decode(q))
    pages, table, lens = cache.k_pages, cache.page_table, cache.seq_lens
    for args in ((pages, pages, table.long(), lens), (pages, pages, table, lens[:2]), (pages, pages, table.cpu(), lens),
                 (pages.transpose(1, 2).contiguous().transpose(1, 2), pages, table, lens), (pages[:0], pages[:0], table, lens),
                 (pages, pages, table[:, :0], lens), (pages, pages, table.t().contiguous().t(), lens),
                 (pages[:1].expand(3, -1, -1, -1), pages[:3], table, lens)):
        with pytest.raises(ValueError):
            PagedKVCache(*args)


TINY = dict(hidden=256, inter=512, layers=2, heads=4, kv_heads=2, head_dim=64, vocab=512, rope_theta=10000.0, eps=1e-6)


@pytest.mark.parametrize("checked", [False, True])
def test_model_over_paged_caches(cuda_device, checked):
    """Two prompts and their next tokens, one batch over the paged caches,
    against each sequence alone over its dense cache. Both round activations
    to bf16 at the same places but one (the dense path rounds cos and sin):
    a dozen roundings of 2^-8 at most per layer bound the logits' relative
    distance by 2 * 12 * 2^-8 = 0.09."""
    dev = cuda_device
    model = build_qwen2(TINY, dev, seed=0)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 512, (n,), generator=g).to(dev) for n in (37, 150)]
    tokens = [torch.randint(0, 512, (2,), generator=g).to(dev) for _ in range(3)]
    cfg = AbftConfig(enable=True, checker_backend="b200", detect_only=False)
    stats = AbftStatsCollector()
    injector = AbftInjector(cfg, CheapSumChecker(cfg), stats, defer_reports=True)
    with torch.no_grad(), (injector if checked else contextlib.nullcontext()):
        caches = model.new_paged_caches(2, 160)
        caches.lens.copy_(torch.tensor([37, 150], dtype=torch.int32))
        cu = torch.tensor([0, 37, 187], dtype=torch.int32, device=dev)
        got = [model.forward_paged(torch.cat(prompts), caches, cu)]
        for t in tokens:
            caches.lens.add_(1)
            got.append(model.forward_paged(t, caches))
        for c in caches.layers:
            c.check_status()
        if checked:
            injector.flush()
    if checked:
        summary = stats.export_summary()["abft"]["faults"]
        assert summary["detected_total"] == 0
    with torch.no_grad():
        for b, prompt in enumerate(prompts):
            dense = model.new_caches(160)
            want = model(prompt, dense, 0)
            have = got[0][(0, 37)[b]:(37, 187)[b]]
            assert (have - want).float().norm() <= 0.09 * want.float().norm()
            for i, t in enumerate(tokens):
                want = model(t[b:b + 1], dense, len(prompt) + i)
                assert (got[1 + i][b] - want[0]).float().norm() <= 0.09 * want.float().norm()
