"""Paged cache operators on the GPU against plain 64-bit forms."""
import pytest
import torch

from vla_abft_estimate_b200.paged import PagedKVCache, rope_table

from .paged_reference import Pool, attention, rotated

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def close(got, want, tol):
    got = got.double().cpu()
    off = (got - want).abs()
    assert torch.isfinite(got).all()
    worst = (off - tol).max().item()
    assert worst <= 0, f"off by {off.max().item():.3g}, {worst:.3g} beyond the tolerance"


def bits(t):
    return t.cpu().contiguous().view(torch.int16)


# ---- append -------------------------------------------------------------------
def run_append(dev, new, total, heads, kv_heads, d, page, dtype, *, cu=True, pad=0, rope=True, joint=False, seed=0):
    """Appends, and compares q, the appended slots and every other slot."""
    pool = Pool(total, kv_heads, page, d, dtype, seed=seed, joint=joint)
    cache = pool.device_cache(dev, PagedKVCache)
    before = bits(cache.k_pages), bits(cache.v_pages)
    tokens = sum(new) if cu else len(total)
    g = torch.Generator().manual_seed(seed + 1)
    qkv = torch.randn(tokens + pad, (heads + 2 * kv_heads) * d, generator=g).to(dtype)
    q, k, v = (x.view(tokens + pad, -1, d) for x in qkv.split([heads * d, kv_heads * d, kv_heads * d], -1))
    dq, dk, dv = (x.view(tokens + pad, -1, d)
                  for x in qkv.to(dev).split([heads * d, kv_heads * d, kv_heads * d], -1))
    table = rope_table(max(total) + 1, d, device=dev) if rope else None
    bounds = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device=dev) if cu else None
    q_out = torch.full((tokens + pad, heads, d), 7.0, dtype=dtype, device=dev)
    got = cache.append(dq, dk, dv, table, cu_seqlens=bounds, q_out=q_out)
    assert got is q_out
    cache.check_status()
    owner, pos = [], []
    for b, (n, t) in enumerate(zip(new, total)):
        owner += [b] * n
        pos += range(t - n, t)
    rows = list(range(tokens)) if cu else [b for b, n in enumerate(new) if n]
    position = torch.tensor(pos, dtype=torch.int64)
    if rope:
        want_q, tol_q = rotated(q[rows], position)
        want_k, tol_k = rotated(k[rows], position)
    else:
        want_q, want_k = q[rows].double(), k[rows].double()
        tol_q = tol_k = 0.0 * want_q.abs().max()
    close(q_out[rows], want_q, tol_q)
    rest = [i for i in range(tokens + pad) if i not in set(rows)]
    assert (q_out[rest] == 7.0).all()
    page_of = pool.table[torch.tensor(owner, dtype=torch.int64), position // page].long()
    slot = position % page
    close(cache.k_pages.cpu()[page_of, :, slot], want_k, tol_k)
    assert torch.equal(bits(cache.v_pages.cpu()[page_of, :, slot]), bits(v[rows]))
    for now, was in ((bits(cache.k_pages), before[0]), (bits(cache.v_pages), before[1])):
        now, was = now.clone(), was.clone()
        now[page_of, :, slot] = 0
        was[page_of, :, slot] = 0
        assert torch.equal(now, was), "a slot of no appended token changed"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (28, 4), (32, 32), (64, 1), (6, 3)])
def test_append_head_layouts(cuda_device, heads, kv_heads, d, dtype):
    run_append(cuda_device, [3, 1, 17], [20, 1, 33], heads, kv_heads, d, 16, dtype)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("new,total", [([1], [1]), ([1], [513]), ([129], [129]), ([16, 16], [16, 32]),
                                       ([5, 0, 0, 40], [700, 3, 0, 40])])
def test_append_lengths(cuda_device, new, total, page):
    run_append(cuda_device, new, total, 7, 1, 128, page, BF16)


def test_append_rows_of_no_sequence_are_left(cuda_device):
    run_append(cuda_device, [2, 3], [9, 100], 8, 2, 64, 16, F16, pad=6)
    run_append(cuda_device, [1, 0, 1, 0], [9, 0, 100, 0], 8, 2, 64, 16, F16, cu=False)


def test_append_many_sequences(cuda_device):
    total = [(i * 37) % 90 + 1 for i in range(70)]
    run_append(cuda_device, [1] * 70, total, 8, 8, 128, 32, BF16, cu=True)
    run_append(cuda_device, [1] * 70, total, 8, 8, 128, 32, BF16, cu=False)
    run_append(cuda_device, [min(t, i % 5) for i, t in enumerate(total)], total, 8, 8, 128, 32, BF16)


def test_append_without_rotation_and_joint_pool(cuda_device):
    run_append(cuda_device, [4, 30], [50, 30], 14, 2, 128, 16, BF16, rope=False, joint=True)
    run_append(cuda_device, [4, 30], [50, 30], 14, 2, 128, 16, F16, joint=True)


def test_append_far_positions(cuda_device):
    """A position near 2^20 rotates as exactly as a near one."""
    run_append(cuda_device, [2], [1 << 20], 2, 1, 64, 128, F16)


def test_append_in_place_other_strides_and_no_q(cuda_device):
    pool = Pool([40, 25], 2, 16, 64, BF16)
    cache = pool.device_cache(cuda_device, PagedKVCache)
    rope = rope_table(64, 64, device=cuda_device)
    q = torch.randn(2, 4, 64, device=cuda_device).to(BF16)
    k, v = (torch.randn(2, 64, 2, device=cuda_device).to(BF16).transpose(1, 2) for _ in range(2))  # stride 2 inside
    want = cache.append(q, k, v, rope)
    kept = bits(cache.k_pages)
    assert cache.append(q, k, v, rope, q_out=q) is q
    assert torch.equal(q, want) and torch.equal(bits(cache.k_pages), kept)
    cache.v_pages.zero_()
    assert cache.append(None, k, v, rope) is None
    assert torch.equal(bits(cache.k_pages), kept)
    assert torch.equal(cache.v_pages[pool.table[0, 2], :, 39 - 32], v[0])


def test_append_skips_bad_entries(cuda_device):
    """Device-side errors: nothing outside the slots is written, the status says what was met."""
    def attempt(lens=None, entry=None, positions=64):
        pool = Pool([40, 25], 2, 16, 64, BF16)
        cache = pool.device_cache(cuda_device, PagedKVCache)
        before = bits(cache.k_pages), bits(cache.v_pages)
        if lens is not None:
            cache.seq_lens[0] = lens
        if entry is not None:
            cache.page_table[0, 2] = entry
        k = torch.randn(2, 2, 64, device=cuda_device).to(BF16)
        q = torch.randn(2, 4, 64, device=cuda_device).to(BF16)
        out = torch.full_like(q, 5.0)
        cache.append(q, k, k, rope_table(positions, 64, device=cuda_device), q_out=out)
        assert (out[0] == 5.0).all() and (out[1] != 5.0).any()
        with pytest.raises(ValueError) as e:
            cache.check_status()
        cache.check_status()  # cleared
        now = bits(cache.k_pages), bits(cache.v_pages)
        for a, b in zip(now, before):  # sequence 1's slot 24 alone
            a, b = a.clone(), b.clone()
            a[pool.table[1, 1].item(), :, 8] = b[pool.table[1, 1].item(), :, 8]
            assert torch.equal(a, b)
        return str(e.value)

    assert "page_table" in attempt(entry=1000)
    assert "page_table" in attempt(entry=-1)
    assert "length" in attempt(lens=49)  # the table has 3 pages: 48 slots
    assert "length" in attempt(lens=-5)
    assert "length" in attempt(lens=2147483647)
    assert "rotation" in attempt(positions=39)


# ---- decode -------------------------------------------------------------------
def run_decode(dev, lens, heads, kv_heads, d, page, dtype, *, seed=0, sms=0, spread=1.5, joint=False, extra=0,
               scale=None):
    pool = Pool(lens, kv_heads, page, d, dtype, seed=seed, joint=joint, extra_columns=extra)
    cache = pool.device_cache(dev, PagedKVCache)
    q = (torch.randn(len(lens), heads, d, generator=torch.Generator().manual_seed(seed + 9)) * spread).to(dtype)
    got = cache.decode(q.to(dev), num_sms=sms, scale=scale)
    cache.check_status()
    want, tol = attention(pool, q, list(enumerate(lens)), scale)
    close(got, want, tol)
    return cache, q.to(dev), got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (28, 4), (5, 5), (16, 2), (9, 1), (32, 2), (17, 1), (64, 1)])
def test_decode_head_layouts(cuda_device, heads, kv_heads, d, dtype):
    run_decode(cuda_device, [77, 300], heads, kv_heads, d, 16, dtype)


@pytest.mark.parametrize("sms", [0, 1, 2, 3, 7, 1000])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("lens", [[1], [2], [15, 16, 17], [31, 32, 33], [0, 1, 127, 128, 129, 0], [1000, 3, 513]])
def test_decode_lengths_and_shares(cuda_device, lens, page, sms):
    """Shares of any size: segments within a warp, across warps and across CTAs."""
    run_decode(cuda_device, lens, 7, 1, 128, page, BF16, sms=sms)


@pytest.mark.parametrize("sms", [1, 5, 0])
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (36, 3), (40, 2)])
def test_decode_many_sequences(cuda_device, heads, kv_heads, sms):
    """More sequences than a warp scans at once, empty ones among them."""
    run_decode(cuda_device, [(i * 53) % 170 if i % 7 else 0 for i in range(75)], heads, kv_heads, 64, 32, F16, sms=sms)
    run_decode(cuda_device, [0] * 40 + [333] + [0] * 40, heads, kv_heads, 128, 16, BF16, sms=sms)


def test_decode_long_and_peaked(cuda_device):
    run_decode(cuda_device, [20011], 7, 1, 128, 32, BF16)
    run_decode(cuda_device, [3000, 5000], 8, 4, 64, 64, F16, spread=30.0)  # scores of +-100: one key has all the weight
    run_decode(cuda_device, [3000, 5000], 8, 4, 64, 64, F16, scale=0.0)  # all keys alike


def test_decode_wide_table_joint_pool(cuda_device):
    """Columns behind a sequence's pages are never read, other page strides."""
    run_decode(cuda_device, [100, 17, 0], 12, 4, 128, 16, F16, joint=True, extra=50)


def test_decode_empty_batch_and_all_idle(cuda_device):
    cache = PagedKVCache(torch.zeros(2, 1, 16, 64, dtype=BF16, device=cuda_device),
                         torch.zeros(2, 1, 16, 64, dtype=BF16, device=cuda_device),
                         torch.zeros(0, 4, dtype=torch.int32, device=cuda_device),
                         torch.zeros(0, dtype=torch.int32, device=cuda_device))
    assert cache.decode(torch.zeros(0, 2, 64, dtype=BF16, device=cuda_device)).shape == (0, 2, 64)
    _, _, got = run_decode(cuda_device, [0, 0], 2, 1, 64, 16, BF16)
    assert (got == 0).all()
    _, _, got = run_decode(cuda_device, [0, 0], 2, 1, 64, 16, BF16, extra=100)
    assert (got == 0).all()


def test_decode_same_bits_twice_and_other_strides(cuda_device):
    cache, q, got = run_decode(cuda_device, [900, 1234, 77], 28, 4, 128, 16, BF16)
    assert torch.equal(cache.decode(q), got)
    wide = torch.zeros(3, 28, 256, dtype=BF16, device=cuda_device)
    wide[:, :, 128:] = q
    assert torch.equal(cache.decode(wide[:, :, 128:]), got)  # read in place
    assert torch.equal(cache.decode(q.transpose(1, 2).contiguous().transpose(1, 2)), got)  # copied
    out = torch.full((3, 28, 136), 3.0, dtype=BF16, device=cuda_device)
    assert torch.equal(cache.decode(q, out=out[:, :, :128]), got)
    assert (out[:, :, 128:] == 3.0).all()


def test_decode_shared_pages(cuda_device):
    """Two sequences with the same first pages."""
    pool = Pool([64, 64], 2, 16, 64, BF16)
    pool.table[1, :3] = pool.table[0, :3]
    cache = pool.device_cache(cuda_device, PagedKVCache)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(3)).to(BF16)
    want, tol = attention(pool, q, [(0, 64), (1, 64)])
    close(cache.decode(q.to(cuda_device)), want, tol)


def test_decode_bad_entries(cuda_device):
    """A bad page reads as zeros, lengths are cut to the table; the status tells."""
    def attempt(lens=None, entry=None, column=1):
        pool = Pool([48, 25], 2, 16, 64, BF16)
        cache = pool.device_cache(cuda_device, PagedKVCache)
        seen = 48
        if lens is not None:
            cache.seq_lens[0] = lens
            seen = max(0, min(48, lens))
        if entry is not None:
            cache.page_table[0, column] = entry
            at = pool.table[0, column].long().item()
            pool.k[at] = 0
            pool.v[at] = 0
        q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(3)).to(BF16)
        got = cache.decode(q.to(cuda_device))
        want, tol = attention(pool, q, [(0, seen), (1, 25)])
        close(got, want, tol)
        with pytest.raises(ValueError) as e:
            cache.check_status()
        return str(e.value)

    assert "page_table" in attempt(entry=5000)
    assert "page_table" in attempt(entry=-2, column=0)
    assert "length" in attempt(lens=-1)
    assert "length" in attempt(lens=49)
    assert "length" in attempt(lens=2147483647)


# ---- prefill ------------------------------------------------------------------
def owners_of(new, total):
    return [(b, t - n + i + 1) for b, (n, t) in enumerate(zip(new, total)) for i in range(n)]


def run_prefill(dev, new, total, heads, kv_heads, d, page, dtype, *, seed=0, splits=0, spread=1.5, joint=False, extra=0,
                scale=None, pad=0):
    pool = Pool(total, kv_heads, page, d, dtype, seed=seed, joint=joint, extra_columns=extra)
    cache = pool.device_cache(dev, PagedKVCache)
    tokens = sum(new)
    q = (torch.randn(tokens + pad, heads, d, generator=torch.Generator().manual_seed(seed + 9)) * spread).to(dtype)
    cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device=dev)
    out = torch.full((tokens + pad, heads, d), 7.0, dtype=dtype, device=dev)
    got = cache.prefill(q.to(dev), cu, num_splits=splits, scale=scale, out=out)
    assert got is out
    cache.check_status()
    want, tol = attention(pool, q[:tokens], owners_of(new, total), scale)
    close(got[:tokens], want, tol)
    assert (out[tokens:] == 7.0).all()
    return cache, q.to(dev), cu, out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (28, 4), (5, 5), (16, 2), (9, 1), (17, 1), (64, 1)])
def test_prefill_head_layouts(cuda_device, heads, kv_heads, d, dtype):
    run_prefill(cuda_device, [77, 3], [77, 300], heads, kv_heads, d, 16, dtype)


@pytest.mark.parametrize("splits", [0, 1, 2, 5])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("new,total", [([1], [1]), ([2], [2]), ([17], [17]), ([1], [513]), ([129, 5], [129, 128]),
                                       ([16, 16], [128, 144]), ([5, 0, 0, 40], [700, 3, 0, 40]),
                                       ([255, 256, 257], [255, 256, 257])])
def test_prefill_lengths(cuda_device, new, total, page, splits):
    run_prefill(cuda_device, new, [max(n, t) for n, t in zip(new, total)], 7, 1, 128, page, BF16, splits=splits)


def test_prefill_longer_and_peaked(cuda_device):
    run_prefill(cuda_device, [700], [1500], 7, 1, 128, 32, BF16)
    run_prefill(cuda_device, [300, 20], [700, 2000], 8, 4, 64, 64, F16, spread=30.0)
    run_prefill(cuda_device, [300, 20], [700, 2000], 8, 4, 64, 64, F16, scale=0.0)
    run_prefill(cuda_device, [300, 20], [700, 2000], 8, 4, 64, 64, BF16, scale=-0.2)


def test_prefill_rows_of_no_sequence_joint_pool_wide_table(cuda_device):
    run_prefill(cuda_device, [30, 0, 100], [30, 0, 117], 12, 4, 128, 16, F16, joint=True, extra=50, pad=9)
    run_prefill(cuda_device, [2, 1], [900, 17], 12, 4, 128, 16, F16, joint=True, extra=50, pad=200, splits=3)


def test_prefill_rising_maximum(cuda_device):
    """Scores that rise by far more than 2^8 from step to step: every step rescales."""
    pool = Pool([900], 1, 16, 64, BF16)
    held = pool.table[0, :57].long()
    ramp = torch.arange(57 * 16).view(57, 1, 16, 1) / 900.0
    pool.k[held] = (ramp * 20 * torch.ones(64)).to(BF16)
    pool.k[held[-1], :, 4:] = float("nan")
    cache = pool.device_cache(cuda_device, PagedKVCache)
    q = torch.full((100, 2, 64), 3.0).to(BF16)
    want, tol = attention(pool, q, owners_of([100], [900]), 1.0)
    cu = torch.tensor([0, 100], dtype=torch.int32, device=cuda_device)
    close(cache.prefill(q.to(cuda_device), cu, scale=1.0), want, tol)
    want, tol = attention(pool, -q, owners_of([100], [900]), 1.0)  # falling
    close(cache.prefill(-q.to(cuda_device), cu, scale=1.0), want, tol)


def test_prefill_same_bits_twice_other_strides_and_decode(cuda_device):
    cache, q, cu, got = run_prefill(cuda_device, [90, 1, 33], [900, 1234, 33], 28, 4, 128, 16, BF16)
    assert torch.equal(cache.prefill(q, cu), got)
    wide = torch.zeros(124, 28, 256, dtype=BF16, device=cuda_device)
    wide[:, :, 128:] = q
    assert torch.equal(cache.prefill(wide[:, :, 128:], cu), got)
    assert torch.equal(cache.prefill(q.transpose(1, 2).contiguous().transpose(1, 2), cu), got)
    # the newest tokens again, one per sequence
    newest = (cu[1:] - 1).long()
    one = cache.decode(q[newest])
    assert (one.float() - got[newest].float()).abs().max() <= 2.0 ** -6 * got.float().abs().max()


def test_prefill_bad_entries(cuda_device):
    def attempt(lens=None, entry=None, column=1, new=(20, 25)):
        pool = Pool([48, 25], 2, 16, 64, BF16)
        cache = pool.device_cache(cuda_device, PagedKVCache)
        total = [48, 25]
        if lens is not None:
            cache.seq_lens[0] = lens
            total[0] = max(0, min(48, lens))
        if entry is not None:
            cache.page_table[0, column] = entry
            at = pool.table[0, column].long().item()
            pool.k[at] = 0
            pool.v[at] = 0
        q = torch.randn(sum(new), 4, 64, generator=torch.Generator().manual_seed(3)).to(BF16)
        cu = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=cuda_device)
        got = cache.prefill(q.to(cuda_device), cu)
        want, tol = attention(pool, q, owners_of(new, total))
        close(got, want, tol)
        with pytest.raises(ValueError) as e:
            cache.check_status()
        return str(e.value)

    assert "page_table" in attempt(entry=5000)
    assert "page_table" in attempt(entry=-2, column=0)
    assert "length" in attempt(lens=-1)
    assert "length" in attempt(lens=49)
    assert "length" in attempt(lens=7)  # fewer than the new tokens: the first 13 see nothing
    assert "length" in attempt(lens=2147483647)
