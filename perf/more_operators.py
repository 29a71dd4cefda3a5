"""Operators of drafted trees over the paged cache: what is measured, and their plain forms.

What a serving step with drafted tokens runs around the paged cache of
``perf/operators.py``, in its order:

* ``append`` with positions of its own: tokens go to the slots behind the cache
  and are rotated by the position they stand for, which for image and video
  tokens has several axes and for drafted ones is their depth in the tree;
* ``tree``: attention of a tree of drafted tokens over the cached tokens and
  their own ancestors;
* ``accept``: which of the drafted tokens the model's answers confirm (the
  longest confirmed path from a root, the lowest last row among equals);
* ``keep``: the confirmed tokens' keys and values move up to the slots behind the
  cache, in all layers;
* ``fork``: sequences go on from others' caches (shared full pages, a copy of the
  last, partial one), in all layers.

A case gives the head layout, the page size, the type, and how long the
sequences are: ``new`` tokens of this call (at most) after ``past`` cached ones
(at most). ``ragged`` spreads both over the batch; ``idle`` leaves every fifth
slot of a batch without a sequence. ``run`` with ``own`` false computes in
elementary torch operations, in 32 bits.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _case(name, op, batch, new, past, heads=0, kv_heads=0, head_dim=0, page=0, dtype="", ragged=False, idle=False,
          sections="", layers=0):
    return dict(name=name, op=op, batch=batch, new=new, past=past, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                page=page, dtype=dtype, ragged=ragged, idle=idle, sections=sections, layers=layers)


def listed():
    return [
        # one decoded token behind images, rotated on three axes: launch latency
        _case("append_one", "append", 1, 1, 528, 28, 4, 128, 16, "bf16", sections="16,24,24"),
        # prompts with eight images of 256 patches and 32 tokens of text each
        _case("append_media", "append", 5, 2080, 1000, 28, 4, 128, 16, "bf16", sections="16,24,24"),
        # the first tree drafted after a 512-token prompt
        _case("tree_one", "tree", 1, 16, 512, 28, 4, 128, 16, "bf16"),
        # a serving batch: trees and caches of unlike size, some slots without a sequence
        _case("tree_batch", "tree", 24, 26, 4096, 28, 4, 128, 16, "bf16", ragged=True, idle=True),
        # no shared heads, heads of 64, larger pages
        _case("tree_heads", "tree", 12, 13, 3001, 32, 32, 64, 64, "f16", ragged=True),
        # a large tree behind one long document
        _case("tree_long", "tree", 1, 64, 131008, 28, 4, 128, 32, "bf16"),
        # one sequence's tree, and a serving batch's
        _case("accept_one", "accept", 1, 16, 0),
        _case("accept_batch", "accept", 256, 61, 0, ragged=True),
        # the kept path of one tree, in the caches of 28 layers, and those of a batch
        _case("keep_one", "keep", 1, 26, 100, 28, 4, 128, 16, "bf16", layers=28),
        _case("keep_batch", "keep", 64, 26, 100, 28, 4, 128, 16, "bf16", ragged=True, layers=28),
        # three more samples of one prompt, and the beams of a batch on large pages
        _case("fork_one", "fork", 3, 1, 507, 28, 4, 128, 16, "bf16", layers=28),
        _case("fork_beams", "fork", 32, 1, 2000, 32, 4, 128, 128, "f16", ragged=True, layers=28),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    while True:
        op = rng.choice(["append", "tree", "tree", "accept", "keep", "fork"])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 16, 32])
        group = rng.choice([1, 2, 3, 4, 6, 7, 8, 12, 16])
        d = rng.choice([64, 128, 128])
        case = dict(op=op, heads=kv_heads * group, kv_heads=kv_heads, head_dim=d, page=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice(["bf16", "f16"]), ragged=rng.random() < 0.6, idle=False, sections="", layers=0)
        if op == "append":
            cuts = sorted(rng.sample(range(1, d // 2), rng.choice([0, 1, 2, 2, 3])))
            sizes = [b - a for a, b in zip([0] + cuts, cuts + [d // 2])]
            case.update(batch=_log_int(rng, 1, 96), new=_log_int(rng, 1, 4096), past=_log_int(rng, 1, 4096) - 1,
                        sections=",".join(map(str, sizes)))
        elif op == "tree":
            case.update(batch=_log_int(rng, 1, 64), new=_log_int(rng, 1, 128), past=_log_int(rng, 1, 131072) - 1,
                        idle=rng.random() < 0.3)
        elif op == "accept":
            case.update(batch=_log_int(rng, 1, 256), new=_log_int(rng, 1, 200), past=0, heads=0, kv_heads=0, head_dim=0,
                        page=0, dtype="")
            if case["batch"] * case["new"] > 256 * 61:
                continue
            return case
        elif op == "keep":
            case.update(batch=_log_int(rng, 1, 64), new=_log_int(rng, 1, 128), past=_log_int(rng, 1, 200) - 1,
                        layers=rng.choice([1, 6, 28]))
        else:
            case.update(batch=_log_int(rng, 1, 48), new=1, past=_log_int(rng, 1, 4000) - 1, layers=rng.choice([1, 6, 28]))
        if case["heads"] > 64:
            continue
        slots = case["batch"] * (case["new"] + case["past"])
        if op in ("append", "tree") and slots * kv_heads * d * 4 > (1.0e9 if op == "append" else 2.7e8):
            continue  # the cache's bytes
        tokens = case["batch"] * case["new"]
        if op == "append" and (tokens * (case["heads"] + 2 * kv_heads) * d * 2 > 9.0e7 or tokens > 30000):
            continue  # the new tokens'
        if op == "tree" and case["batch"] * case["heads"] * case["new"] * (case["new"] + case["past"]) > 2.3e8:
            continue
        rows = case["batch"] * (math.log2(case["new"]) + 1 if op == "keep" else case["page"])
        if op in ("keep", "fork") and rows * case["layers"] * kv_heads * d > (6.0e6 if op == "keep" else 5.0e7):
            continue
        if op == "keep" and (slots + case["batch"] * case["page"]) * case["layers"] * kv_heads * d > 3.0e8:
            continue
        return case


def _by_case(case):
    """Random numbers that are a function of the case alone."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case):
    """(new, total) tokens of each sequence, and the generator for what follows."""
    r = _by_case(case)
    new, total = [], []
    for b in range(case["batch"]):
        n, p = case["new"], case["past"]
        if case["ragged"] and b:
            n, p = _log_int(r, 1, n), _log_int(r, 1, p + 1) - 1
        if case["idle"] and b % 5 == 4:
            n, p = 0, 0
        new.append(n)
        total.append(n + p)
    return new, total, r


def _trees(new, r):
    """Each sequence's parents: a row's is drawn from the rows before it; row 0 has none."""
    return [[-1 if i == 0 else r.randrange(i) for i in range(n)] for n in new]


def _paths(trees, r):
    """A path from the root to a row of the tree's deeper half, in each tree."""
    out = []
    for parents in trees:
        paths = []
        for i, p in enumerate(parents):
            paths.append([i] if p < 0 else paths[p] + [i])
        paths.sort(key=len)
        out.append(r.choice(paths[len(paths) // 2:]) if paths else [])
    return out


def _packed(lists, pad=None):
    """One int32 tensor of the lists one after another; ``pad``: each filled up to its length in ``pad`` with -1."""
    flat = []
    for k, x in enumerate(lists):
        flat += x + ([-1] * (pad[k] - len(x)) if pad else [])
    return torch.tensor(flat, dtype=torch.int32)


def _pool(case, total, layers, dt, g, dev, extra):
    """Pools [layers, pages, 2, kv_heads, page, head_dim] of every layer's keys and values and a page table, pages handed
    out in no order, as after many requests have come and gone."""
    page, hk, d = case["page"], case["kv_heads"], case["head_dim"]
    count = [-(-n // page) for n in total]
    pages = sum(count) + extra
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32).cpu()
    table = torch.zeros(len(total), max(1, max(count)), dtype=torch.int32)
    at = 0
    for b, c in enumerate(count):
        table[b, :c] = order[at:at + c]
        at += c
    pools = torch.empty(layers, pages, 2, hk, page, d, dtype=dt, device=dev).normal_(generator=g)
    return pools, table, order[at:]


def _media_positions(new, total, axes, r):
    """[axes, tokens]: each run of 256 tokens is an image of 16 x 16 patches (time, height, width, its place), text behind
    it moves all axes on by one; positions are below the slots' as images take fewer positions than tokens."""
    out = [[] for _ in range(axes)]
    for n, t in zip(new, total):
        at = (t - n) // 2
        for i in range(n):
            image = n - i > n % 256  # the first whole images, then text
            k = i % 256
            here = (at, at + k // 16, at + k % 16, at + k // 32) if image else (at, at, at, at)
            for a in range(axes):
                out[a].append(here[a])
            if not image or k == 255:
                at += 16 if image else 1
    return torch.tensor(out, dtype=torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    new, total, r = _lengths(case)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    state = dict(op=case["op"], max_new=max(new), cu=torch.tensor(cu, dtype=torch.int32, device=dev))
    if case["op"] == "accept":
        return _prepare_accept(state, _trees(new, r), cu[-1], seed, dev)
    dt = _DTYPES[case["dtype"]]
    heads, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "fork":
        return _prepare_fork(state, case, total, r, dt, g, dev)
    layers = max(1, case["layers"])
    pools, table, _ = _pool(case, total, layers, dt, g, dev, 3)
    state.update(pools=pools, table=table.to(dev), lens=torch.tensor(total, dtype=torch.int32, device=dev))
    if case["op"] == "append":
        # q, k, v are the fused projection's output, as the layer's linear gives it
        qkv = torch.empty(cu[-1], (heads + 2 * hk) * d, dtype=dt, device=dev).normal_(generator=g)
        q, k, v = qkv.split([heads * d, hk * d, hk * d], dim=-1)
        state.update(q=q.view(-1, heads, d), k=k.view(-1, hk, d), v=v.view(-1, hk, d))
        sections = tuple(int(x) for x in case["sections"].split(","))
        positions = _media_positions(new, total, len(sections), r)
        angle = torch.outer(torch.arange(max(total) + 16, device=dev, dtype=torch.float64), _inverse(d, dev))
        state.update(sections=sections, positions=positions.to(dev),
                     rope=torch.stack((angle.cos(), angle.sin()), dim=-1).float())  # [positions, d / 2, 2]
    else:
        trees = _trees(new, r)
        state["parents"] = _packed(trees).to(dev)
        if case["op"] == "tree":
            # scores spread by about 1.5, as trained heads' do before the softmax
            state["q"] = (1.5 * torch.randn(cu[-1], heads, d, generator=g, device=dev)).to(dt)
        else:
            paths = _paths(trees, r)
            state["kept"] = _packed(paths, new).to(dev)
            state["counts"] = torch.tensor([len(p) for p in paths], dtype=torch.int32, device=dev)
            state["lens_out"] = torch.empty_like(state["lens"])
    if own:
        _handles(state)
    return state


def _prepare_accept(state, trees, tokens, seed, dev):
    """Drafted ids of a vocabulary of 152,064; of every ten rows six would be their parent's answer, which the last such
    child gets."""
    g = torch.Generator().manual_seed(seed)
    parents = _packed(trees)
    ids = torch.randint(0, 152064, (tokens,), generator=g)
    answers = torch.randint(0, 152064, (tokens,), generator=g)
    agree = torch.rand(tokens, generator=g) < 0.6
    at = 0
    for tree in trees:
        for i, p in enumerate(tree):
            if p >= 0 and agree[at + i]:
                answers[at + p] = ids[at + i]
        at += len(tree)
    state.update(parents=parents.to(dev), ids=ids.to(dev), answers=answers.to(dev))
    if own:
        # one small cache stands for the model's: what is accepted does not look at it
        batch = state["cu"].shape[0] - 1
        state["pools"] = torch.zeros(1, 1, 2, 1, 16, 64, dtype=torch.bfloat16, device=dev)
        state.update(table=torch.zeros(batch, 1, dtype=torch.int32, device=dev),
                     lens=torch.zeros(batch, dtype=torch.int32, device=dev))
        _handles(state)
    return state


def _fork_pairs(case, r):
    """(sources, rows of the batch): every source has one to three children; a child is a row behind the sources."""
    batch, at, src = case["batch"], 0, []
    while len(src) < batch:
        src += [at] * min(batch - len(src), r.randrange(1, 4) if case["ragged"] else 3)
        at += 1
    return src, at


def _prepare_fork(state, case, total, r, dt, g, dev):
    src, sources = _fork_pairs(case, r)
    pairs, page = len(src), case["page"]
    lens = total[:sources] + [0] * pairs
    width = max(1, max(-(-n // page) for n in lens))
    # the pages before a sequence's last are read by no fork: sequences share eight of them here
    pages = 8 + sources + pairs
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32).cpu()
    table = torch.full((sources + pairs, width), 0, dtype=torch.int32)
    for b in range(sources):
        held = -(-lens[b] // page)
        for j in range(held):
            table[b, j] = order[8 + b] if j == held - 1 else order[(b + j) % 8]
    state.update(pools=torch.empty(case["layers"], pages, 2, case["kv_heads"], page, case["head_dim"], dtype=dt,
                                   device=dev).normal_(generator=g),
                 table=table.to(dev), lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                 src=torch.tensor(src, dtype=torch.int32, device=dev),
                 dst=torch.arange(sources, sources + pairs, dtype=torch.int32, device=dev),
                 pages=order[8 + sources:].to(dev))
    if own:
        _handles(state)
    return state


def _handles(state):
    """What a program keeps beside its pools: the caches of the layers, and the object for all of them."""
    from vla_abft_estimate_b200.paged import PagedKVCache, PagedLayers

    state["caches"] = [PagedKVCache(p[:, 0], p[:, 1], state["table"], state["lens"]) for p in state["pools"]]
    state["layers"] = PagedLayers(state["caches"])


def _inverse(d, dev):
    return 1.0e6 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)


def run(s):
    if not own:
        return {"append": _plain_append, "tree": _plain_tree, "accept": _plain_accept, "keep": _plain_keep,
                "fork": _plain_fork}[s["op"]](s)
    if s["op"] == "append":
        q = s["caches"][0].append(s["q"], s["k"], s["v"], s["rope"], cu_seqlens=s["cu"], positions=s["positions"],
                                  sections=s["sections"])
        return q, s["pools"]
    if s["op"] == "tree":
        return s["caches"][0].tree(s["q"], s["cu"], s["parents"])
    if s["op"] == "accept":
        return s["layers"].accept(s["cu"], s["parents"], s["ids"], s["answers"])
    if s["op"] == "keep":
        s["layers"].keep(s["cu"], s["kept"], s["counts"], lens_out=s["lens_out"])
        return s["pools"], s["lens_out"]
    s["layers"].fork(s["src"], s["dst"], s["pages"])
    return s["pools"], s["table"], s["lens"]


def _owners(cu, tokens):
    """The sequence of each packed token, and its place among that sequence's new tokens."""
    t = torch.arange(tokens, device=cu.device)
    seq = (t[:, None] >= cu[None, 1:]).sum(1)
    return seq, t - cu[seq]


def _plain_append(s):
    tokens, _, d = s["q"].shape
    seq, place = _owners(s["cu"], tokens)
    count = s["cu"][1:] - s["cu"][:-1]
    slot_of = s["lens"][seq] - count[seq] + place
    axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device=seq.device),
                                   torch.tensor(s["sections"], device=seq.device), output_size=d // 2)
    pair = torch.arange(d // 2, device=seq.device)
    turn = s["rope"][s["positions"].long()[axis].T, pair][:, None]  # [tokens, 1, d / 2, 2]
    cos, sin = turn[..., 0], turn[..., 1]

    def rotated(x):
        a, b = x.float().chunk(2, dim=-1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).to(x.dtype)

    pool = s["pools"][0]
    size = pool.shape[3]
    page, slot = s["table"][seq, slot_of // size].long(), (slot_of % size).long()
    pool[page, 0, :, slot] = rotated(s["k"])
    pool[page, 1, :, slot] = s["v"]
    return rotated(s["q"]), s["pools"]


def _gathered(pages, table):
    """[batch, kv_heads, slots, d] in 32 bits, in the sequences' order."""
    x = pages[table.long()].float()  # [batch, pages, kv_heads, size, d]
    b, n, h, size, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, n * size, d)


def _padded_parents(s):
    """[batch, most, most]: row i has its parent's column; and where the packed rows are in it."""
    seq, place = _owners(s["cu"], s["parents"].shape[0])
    batch, n = s["cu"].shape[0] - 1, s["max_new"]
    up = torch.zeros(batch, n, n + 1, dtype=torch.float64, device=seq.device)  # column 0: no parent
    up[seq, place, (s["parents"] + 1).long()] = 1
    return up[:, :, 1:], seq, place


def _ancestors(up):
    """[batch, most, most]: row i has itself and all rows above it. (I + up)^most counts the ways, 0 where there are none."""
    n = up.shape[-1]
    return torch.linalg.matrix_power(up + torch.eye(n, dtype=up.dtype, device=up.device), n) > 0


def _plain_tree(s):
    q = s["q"]
    tokens, heads, d = q.shape
    up, seq, place = _padded_parents(s)
    above = _ancestors(up)
    k, v = _gathered(s["pools"][0, :, 0], s["table"]), _gathered(s["pools"][0, :, 1], s["table"])
    b, hk, slots = k.shape[0], k.shape[1], k.shape[2]
    n = s["max_new"]
    padded = torch.zeros(b, n, heads, d, device=q.device)
    padded[seq, place] = q.float()
    # slot j of a sequence is drafted row j - (length - count); before those all slots are seen
    row = torch.arange(slots, device=q.device)[None] - (s["lens"] - (s["cu"][1:] - s["cu"][:-1]))[:, None]
    among = torch.gather(above, 2, row.clamp(0, n - 1)[:, None].expand(b, n, slots))
    seen = (row < 0)[:, None] | (among & (row < n)[:, None])
    x = torch.matmul(padded.view(b, n, hk, heads // hk, d).permute(0, 2, 3, 1, 4), k[:, :, None].transpose(-1, -2))
    x = torch.where(seen[:, None, None], x / math.sqrt(d), -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, v[:, :, None]) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, heads, d)[seq, place].to(q.dtype)


def _plain_accept(s):
    up, seq, place = _padded_parents(s)
    above = _ancestors(up)
    batch, n = up.shape[0], up.shape[1]
    first = s["cu"][seq]
    parent = s["parents"].long()
    confirmed = (parent < 0) | (s["ids"] == s["answers"][(first + parent).clamp(min=0)])
    good = torch.zeros(batch, n, dtype=torch.bool, device=up.device)
    good[seq, place] = confirmed
    taken = good & ~(above & ~good[:, None]).any(-1)
    depth = torch.where(taken, above.sum(-1), 0)
    # the deepest, the lowest among equals
    best = (depth * n + (n - 1 - torch.arange(n, device=up.device))).argmax(-1)
    counts = depth.gather(1, best[:, None])[:, 0]
    path = above[torch.arange(batch, device=up.device), best] & (counts > 0)[:, None]
    rank = torch.where(path, path.cumsum(-1) - 1, n)
    rows = torch.full((batch, n + 1), -1, dtype=torch.int32, device=up.device)
    rows.scatter_(1, rank, torch.arange(n, dtype=torch.int32, device=up.device).expand(batch, n))
    last = torch.where(counts > 0, s["answers"][(s["cu"][:-1] + best).clamp(max=s["answers"].shape[0] - 1)], -1)
    return rows[seq, place], counts.to(torch.int32), last


def _plain_keep(s):
    seq, place = _owners(s["cu"], s["kept"].shape[0])
    count = s["cu"][1:] - s["cu"][:-1]
    before = (s["lens"] - count)[seq]
    # rows behind the kept ones stay where they are
    source = torch.where(place < s["counts"][seq], s["kept"], place)
    size = s["pools"].shape[4]
    pool = s["pools"]

    def at(i):
        return s["table"][seq, (before + i) // size].long(), ((before + i) % size).long()

    (from_page, from_slot), (to_page, to_slot) = at(source), at(place)
    pool[:, to_page, :, :, to_slot] = pool[:, from_page, :, :, from_slot]
    s["lens_out"].copy_(s["lens"] - count + s["counts"])
    return pool, s["lens_out"]


def _plain_fork(s):
    size = s["pools"].shape[4]
    src, dst, new, pool, table = s["src"].long(), s["dst"].long(), s["pages"].long(), s["pools"], s["table"]
    n = s["lens"][src]
    full, rest = n // size, n % size
    old = table[src, torch.clamp(full, max=table.shape[1] - 1).long()].long()
    copied = (torch.arange(size, device=src.device)[None] < rest[:, None])[None, :, None, None, :, None]
    pool[:, new] = torch.where(copied, pool[:, old], pool[:, new])
    column = torch.arange(table.shape[1], device=src.device)[None]
    row = torch.where(column < full[:, None], table[src], table[dst])
    table[dst] = torch.where((column == full[:, None]) & (rest > 0)[:, None], s["pages"][:, None], row)
    s["lens"][dst] = n
    return pool, table, s["lens"]


def work(case):
    new, total, r = _lengths(case)
    heads, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    tokens = sum(new)
    if case["op"] == "append":  # q, k, v in; q and the new slots out; each token's angles and positions
        axes = case["sections"].count(",") + 1
        return {"bytes": 2 * tokens * (heads + 2 * hk) * d * 2 + tokens * (d + axes) * 4, "flops": 3 * tokens * (heads + hk) * d}
    if case["op"] == "tree":  # the caches' valid slots, q in and out, parents; a row's own slots are the cached ones and its depth's
        pairs = sum(n * (t - n) for n, t in zip(new, total))
        pairs += sum(_sum_depths(tree) for tree in _trees(new, r))
        return {"bytes": sum(total) * hk * d * 4 + 2 * tokens * heads * d * 2 + 4 * tokens, "flops": 4 * pairs * heads * d}
    if case["op"] == "accept":  # parents, ids and answers in; rows, counts and the next token out
        return {"bytes": tokens * (4 + 8 + 8 + 4) + case["batch"] * 16, "flops": tokens}
    row = 2 * case["layers"] * hk * d * 2  # bytes of a slot's keys and values
    if case["op"] == "keep":  # the rows that move, in and out
        moved = sum(k != i for p in _paths(_trees(new, r), r) for i, k in enumerate(p))
        return {"bytes": 2 * moved * row + tokens * 4 + case["batch"] * 16, "flops": 0}
    src, _ = _fork_pairs(case, r)  # the partial pages' slots in and out, and the tables' rows
    rest = sum(total[a] % case["page"] for a in src)
    return {"bytes": 2 * rest * row + sum(8 * (total[a] // case["page"] + 3) for a in src), "flops": 0}


def _sum_depths(tree):
    depth = []
    for p in tree:
        depth.append(1 if p < 0 else depth[p] + 1)
    return sum(depth)


def exact(case, seed):
    """In 64 bits, sequence by sequence, from the definition. What accept gives is whole numbers."""
    if case["op"] == "accept":
        return None
    s = prepare(case, seed)
    new, total, r = _lengths(case)
    pools, table, size = s["pools"].double(), s["table"].tolist(), case["page"]
    if case["op"] == "fork":
        src, sources = _fork_pairs(case, r)
        for i, a in enumerate(src):
            rest = total[a] % size
            if rest:
                pools[:, int(s["pages"][i]), :, :, :rest] = pools[:, table[a][total[a] // size], :, :, :rest]
        return pools, None, None
    if case["op"] == "keep":
        for b, path in enumerate(_paths(_trees(new, r), r)):
            base = total[b] - new[b]
            for i, k in enumerate(path):
                there, here = divmod(base + k, size), divmod(base + i, size)
                pools[:, table[b][here[0]], :, :, here[1]] = pools[:, table[b][there[0]], :, :, there[1]]
        return pools, None
    d, hk, heads, at = case["head_dim"], case["kv_heads"], case["heads"], 0
    if case["op"] == "append":
        q_out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        bounds = [0]
        for n in s["sections"]:
            bounds.append(bounds[-1] + n)
        for b, (n, t) in enumerate(zip(new, total)):
            here = slice(at, at + n)
            p = torch.empty(n, d // 2, dtype=torch.float64, device="cuda")
            for a in range(len(s["sections"])):
                p[:, bounds[a]:bounds[a + 1]] = s["positions"][a, here, None].double()
            z = torch.polar(torch.ones_like(p), p * _inverse(d, "cuda"))[:, None]

            def turn(x):
                x = x.double()
                w = torch.complex(x[..., : d // 2], x[..., d // 2:]) * z
                return torch.cat((w.real, w.imag), dim=-1)

            slot = torch.arange(t - n, t, device="cuda")
            held = torch.tensor(table[b], device="cuda")[slot // size]
            q_out[here] = turn(s["q"][here])
            pools[0, held, 0, :, slot % size] = turn(s["k"][here])
            pools[0, held, 1, :, slot % size] = s["v"][here].double()
            at += n
        return q_out, pools
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, tree in enumerate(_trees(new, r)):
        n, t = new[b], total[b]
        if n == 0:
            continue
        hidden = torch.ones(n, t, dtype=torch.bool)
        hidden[:, : t - n] = False
        for i in range(n):
            j = i
            while j >= 0:
                hidden[i, t - n + j] = False
                j = tree[j]
        hidden = hidden.cuda()
        held = torch.tensor(table[b][: -(-t // size)], device="cuda")
        for h in range(hk):
            k, v = (pools[0, held, c, h].reshape(-1, d)[:t] for c in (0, 1))
            for j in range(h * heads // hk, (h + 1) * heads // hk):
                x = s["q"][at:at + n, j].double() @ k.T * d ** -0.5
                out[at:at + n, j] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ v
        at += n
    return out
