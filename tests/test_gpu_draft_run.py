"""Drafted trees run together, as a serving loop uses them: append by depth, tree
attention, accept, keep, fork; in CUDA graphs, on streams, in the model."""
import random

import pytest
import torch

from vla_abft_estimate_b200 import paged
from vla_abft_estimate_b200.paged import PagedKVCache, PagedLayers, rope_table
from vla_abft_estimate_b200.workloads import build_qwen2

from .draft_reference import accepted, attention_over, i32, packed, path_to, random_tree, visible_slots
from .test_gpu_paged import BF16, F16, bits, close
from .test_gpu_paged_run import stored

pytestmark = pytest.mark.gpu

HEADS, KV, D, PAGE = 14, 2, 128, 16


def new_layers(dev, batch, slots, n, dtype=BF16, fill=0.0, extra_rows=0):
    """``n`` layers of empty caches; row b of the table has pages b, b + batch, ..."""
    per = -(-slots // PAGE)
    rows = batch + extra_rows
    table = torch.arange(per * rows, dtype=torch.int32, device=dev).view(per, rows).t().contiguous()
    lens = torch.zeros(rows, dtype=torch.int32, device=dev)
    pools = [torch.full((per * rows + 8, 2, KV, PAGE, D), fill, dtype=dtype, device=dev) for _ in range(n)]
    return PagedLayers([PagedKVCache(p[:, 0], p[:, 1], table, lens) for p in pools])


def depth_of(parents):
    return [len(path_to(parents, i)) - 1 for i in range(len(parents))]


def slots_of(layers, layer, b, n):
    """Keys and values of sequence b's first n slots, as bits."""
    c = layers.layers[layer]
    held = c.page_table[b, : -(-n // PAGE)].long()
    return [bits(x[held].transpose(0, 1).reshape(KV, -1, D)[:, :n]) for x in (c.k_pages, c.v_pages)]


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_drafted_steps_leave_what_single_tokens_leave(cuda_device, dtype):
    """Prompts, then steps of drafted trees of which a path is kept, in three layers:
    every attention against the formula, and the caches bit for bit those of the same
    tokens appended one by one."""
    dev, batch, n_layers = cuda_device, 3, 3
    g, r = torch.Generator().manual_seed(1), random.Random(2)
    drafted, plain = (new_layers(dev, batch, 600, n_layers, dtype, fill=float("nan")) for _ in range(2))
    rope = rope_table(700, D, device=dev)

    def rows(n):
        return [torch.randn(n, h, D, generator=g).to(dtype).to(dev) for h in (HEADS, KV, KV)]

    total = [40, 130, 5]
    cu = i32([0, 40, 170, 175], dev)
    for x in (drafted, plain):
        x.seq_lens.copy_(i32(total, dev))
    for layer in range(n_layers):
        q, k, v = rows(175)
        for x in (drafted, plain):
            x.layers[layer].append(q, k, v, rope, cu_seqlens=cu)
    for step in range(6):
        trees = [random_tree(r.randrange(1, 40), r.random()) for _ in range(batch)]
        cu, parents = packed(trees)
        positions = [total[b] + d for b, t in enumerate(trees) for d in depth_of(t)]
        dcu, dup, dpos = i32(cu, dev), i32(parents, dev), i32(positions, dev)
        drafted.seq_lens.copy_(i32([t + len(x) for t, x in zip(total, trees)], dev))
        ids = torch.tensor([r.randrange(3) for _ in parents], device=dev)
        answers = torch.tensor([r.randrange(3) for _ in parents], device=dev)
        paths = [accepted(t, ids[a:b].tolist(), answers[a:b].tolist())[0] for t, a, b in zip(trees, cu, cu[1:])]
        for layer in range(n_layers):
            cache = drafted.layers[layer]
            q, k, v = rows(cu[-1])
            rq = cache.append(q, k, v, rope, cu_seqlens=dcu, positions=dpos)
            out = cache.tree(rq, dcu, dup)
            held = stored(cache)
            held.lens = [t + len(x) for t, x in zip(total, trees)]
            want = [(b, visible_slots(t, i, held.lens[b])) for b, t in enumerate(trees) for i in range(len(t))]
            close(out, *attention_over(held, rq.cpu(), want))
            for b, path in enumerate(paths):  # the same tokens, one by one
                for i, row in enumerate(path):
                    lens = list(total)
                    lens[b] = total[b] + i + 1
                    plain.seq_lens.copy_(i32([n if c == b else 0 for c, n in enumerate(lens)], dev))
                    at = cu[b] + row
                    one = [x[at:at + 1].expand(batch, -1, -1).contiguous() for x in (q, k, v)]
                    plain.layers[layer].append(*one, rope)
        kept, counts, token = drafted.accept(dcu, dup, ids, answers)
        assert counts.tolist() == [len(p) for p in paths]
        drafted.keep(dcu, kept, counts)
        total = [t + len(p) for t, p in zip(total, paths)]
        assert drafted.seq_lens.tolist() == total
        for layer in range(n_layers):
            for b in range(batch):
                for have, want in zip(slots_of(drafted, layer, b, total[b]), slots_of(plain, layer, b, total[b])):
                    assert torch.equal(have, want), (step, layer, b)
    drafted.check_status()
    plain.check_status()


def test_forked_sequences_go_their_own_ways(cuda_device):
    """Two samples of one prompt: shared full pages, a page each from the fork on."""
    dev = cuda_device
    layers = new_layers(dev, 2, 200, 2, extra_rows=2)
    rope = rope_table(300, D, device=dev)
    g = torch.Generator().manual_seed(3)
    layers.seq_lens.copy_(i32([70, 45, 0, 0], dev))
    cu = i32([0, 70, 115, 115, 115], dev)
    for c in layers.layers:
        q, k, v = (torch.randn(115, h, D, generator=g).to(BF16).to(dev) for h in (HEADS, KV, KV))
        c.append(q, k, v, rope, cu_seqlens=cu)
    spare = layers.layers[0].num_pages
    layers.fork(i32([0, 0], dev), i32([2, 3], dev), i32([spare - 1, spare - 2], dev))
    layers.check_status()
    table = layers.page_table.tolist()
    assert table[2][:5] == table[0][:4] + [spare - 1] and table[3][:5] == table[0][:4] + [spare - 2]
    before = [[slots_of(layers, layer, b, 70) for b in (0, 2, 3)] for layer in range(2)]
    for layer in before:
        for x in layer[1:]:
            assert all(torch.equal(a, b) for a, b in zip(x, layer[0]))
    layers.seq_lens.add_(i32([1, 0, 1, 1], dev))
    cu = i32([0, 1, 1, 2, 3], dev)
    for layer, c in enumerate(layers.layers):
        q, k, v = (torch.randn(3, h, D, generator=g).to(BF16).to(dev) for h in (HEADS, KV, KV))
        rq = c.append(q, k, v, rope, cu_seqlens=cu)
        held = stored(c)
        held.lens = layers.seq_lens.tolist()
        close(c.prefill(rq, cu), *attention_over(held, rq.cpu(), [(b, list(range(71))) for b in (0, 2, 3)]))
        for b, was in zip((0, 2, 3), before[layer]):
            assert all(torch.equal(x, y) for x, y in zip(slots_of(layers, layer, b, 70), was))
    layers.check_status()


def tree_state(dev, seed, sizes=(26, 1, 0, 40), total=(500, 1, 0, 90), columns=0):
    layers = new_layers(dev, len(sizes), max(total) + 16 * columns + 60, 2)
    g = torch.Generator().manual_seed(seed)
    for c in layers.layers:
        c.k_pages.copy_(torch.randn(c.k_pages.shape, generator=g).to(BF16))
        c.v_pages.copy_(torch.randn(c.v_pages.shape, generator=g).to(BF16))
    layers.seq_lens.copy_(i32(total, dev))
    cu, parents = packed([random_tree(n, seed + i) for i, n in enumerate(sizes)])
    q, k, v = (torch.randn(cu[-1], h, D, generator=g).to(BF16).to(dev) for h in (HEADS, KV, KV))
    ids, answers = (torch.randint(0, 2, (cu[-1],), generator=g).to(dev) for _ in range(2))
    positions = torch.randint(0, 600, (cu[-1],), generator=g, dtype=torch.int32).to(dev)
    return dict(layers=layers, q=q, k=k, v=v, cu=i32(cu, dev), parents=i32(parents, dev), ids=ids, answers=answers,
                positions=positions, rope=rope_table(600, D, device=dev))


def tree_step(s):
    """A whole step; everything it gives."""
    out = []
    for c in s["layers"].layers:
        q = c.append(s["q"], s["k"], s["v"], s["rope"], cu_seqlens=s["cu"], positions=s["positions"])
        out += [q, c.tree(q, s["cu"], s["parents"])]
    kept, counts, token = s["layers"].accept(s["cu"], s["parents"], s["ids"], s["answers"])
    s["layers"].keep(s["cu"], kept, counts)
    return out + [kept, counts, token]


def everything(s, out):
    return [x.clone() for x in out] + [x.clone() for c in s["layers"].layers for x in (c.k_pages, c.v_pages)] + \
        [s["layers"].seq_lens.clone()]


@pytest.mark.parametrize("columns", [0, 600])
def test_a_captured_step_follows_trees_lengths_and_answers(cuda_device, columns):
    """By cluster and by list: one graph, replayed for other trees, boundaries, lengths and answers."""
    dev = cuda_device
    state = tree_state(dev, 0, (26, 1, 0, 40), (700, 700, 700, 700), columns=columns)
    lens = state["layers"].seq_lens.clone()
    tree_step(state)  # first calls outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tree_step(state)
    state["layers"].seq_lens.copy_(lens)
    g = torch.Generator().manual_seed(9)
    for seed, (sizes, total) in enumerate([((26, 1, 0, 40), (500, 1, 0, 90)), ((0, 30, 30, 7), (0, 30, 600, 8)),
                                           ((67, 0, 0, 0), (300, 9, 0, 40)), ((5, 50, 4, 8), (700, 699, 650, 8)),
                                           ((1, 1, 1, 1), (64, 65, 128, 1))]):
        cu, parents = packed([random_tree(n, seed + n) for n in sizes])
        state["cu"].copy_(i32(cu))
        state["parents"][:cu[-1]].copy_(i32(parents))
        state["layers"].seq_lens.copy_(i32(total))
        for key in ("ids", "answers"):
            state[key].copy_(torch.randint(0, 2, state[key].shape, generator=g))
        state["q"].normal_()
        for _ in range(2):
            table, lens = state["layers"].page_table, state["layers"].seq_lens.clone()
            eager = dict(state, layers=PagedLayers([PagedKVCache(c.k_pages.clone(), c.v_pages.clone(), table, lens)
                                                    for c in state["layers"].layers]))
            want = everything(eager, tree_step(eager))
            graph.replay()
            got = everything(state, out)
            for k, (a, b) in enumerate(zip(got, want)):
                if k < 4:  # rows of q and results behind the last sequence are anybody's
                    a, b = a[:cu[-1]], b[:cu[-1]]
                assert torch.equal(a, b), (seed, k)
            state["layers"].check_status()
            state["layers"].seq_lens.copy_(i32(total))


@pytest.mark.parametrize("graphs", [False, True])
def test_steps_on_two_streams_at_once(cuda_device, graphs):
    """Eager, or two graphs: scratch belongs to each call."""
    dev = cuda_device
    runs = []
    for seed in range(2):
        s = tree_state(dev, seed, (30, 9, 50, 3), (3000, 800, 2000, 20), columns=300)
        one = s["layers"].layers[0]
        want = one.tree(s["q"], s["cu"], s["parents"]).clone()
        accept = [x.clone() for x in s["layers"].accept(s["cu"], s["parents"], s["ids"], s["answers"])]
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()

        def step(s=s, one=one):
            return [one.tree(s["q"], s["cu"], s["parents"]),
                    *s["layers"].accept(s["cu"], s["parents"], s["ids"], s["answers"])]

        got = None
        if graphs:
            with torch.cuda.graph(graph):
                for _ in range(3):
                    got = step()
        runs.append((stream, graph, step, got, [want] + accept))
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(10):
        for i, (stream, graph, step, got, _) in enumerate(runs):
            with torch.cuda.stream(stream):
                if graphs:
                    graph.replay()
                else:
                    results[i].append(step())
    torch.cuda.synchronize()
    for i, (_, _, _, got, want) in enumerate(runs):
        for out in [got] if graphs else results[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_the_long_way_gives_the_same(cuda_device, monkeypatch):
    """Without the extension, calls go through ctypes to the same kernels."""
    def outputs():
        s = tree_state(cuda_device, 5)
        out = everything(s, tree_step(s))
        s["layers"].layers[0].append(None, s["k"], s["v"], s["rope"], cu_seqlens=s["cu"],
                                     positions=s["positions"].expand(2, -1), sections=[60, 4])
        layers = s["layers"]
        layers.fork(i32([0], cuda_device), i32([2], cuda_device), i32([layers.layers[0].num_pages - 1], cuda_device))
        lens = layers.keep(s["cu"], torch.zeros_like(s["parents"]), torch.zeros_like(layers.seq_lens),
                           lens_out=torch.empty_like(layers.seq_lens))
        out += everything(s, [layers.page_table, lens])
        out.append(layers.layers[1].tree(s["q"], s["cu"], s["parents"], scale=0.3, num_sms=3, out=torch.empty_like(s["q"])))
        return out

    want = outputs()
    monkeypatch.setattr(paged, "_HOST", paged._LongWay)
    got = outputs()
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_what_autograd_and_tracers_are_told(cuda_device):
    s = tree_state(cuda_device, 6)
    layers = s["layers"]
    cache = layers.layers[0]
    calls = {"append": lambda: cache.append(s["q"], s["k"], s["v"], s["rope"], cu_seqlens=s["cu"], positions=s["positions"]),
             "tree": lambda: cache.tree(s["q"], s["cu"], s["parents"]),
             "keep": lambda: layers.keep(s["cu"], torch.zeros_like(s["parents"]), torch.zeros_like(layers.seq_lens)),
             "fork": lambda: layers.fork(i32([-1], cuda_device), i32([-1], cuda_device), i32([-1], cuda_device))}
    # what a call writes counts as modified
    watched = dict(k=cache.k_pages, v=cache.v_pages, last=layers.layers[1].v_pages, lens=layers.seq_lens, table=layers.page_table)
    for name, written in (("append", "k v"), ("keep", "k v last lens"), ("fork", "k v last lens table"), ("tree", "")):
        before = {key: x._version for key, x in watched.items()}
        calls[name]()
        assert {key for key, x in watched.items() if x._version > before[key]} == set(written.split()), name
    out = torch.empty_like(s["q"])
    cache.tree(s["q"], s["cu"], s["parents"], out=out)
    assert out._version == 1
    # gradients and traces are refused
    for which in ("q", "k", "v", "rope"):
        kept = s[which]
        s[which] = kept.clone().requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            calls["append"]()
        with torch.no_grad():
            calls["append"]()
        s[which] = kept
    layers.layers[1].k_pages.requires_grad_()
    for name in ("keep", "fork"):
        with pytest.raises(ValueError, match="gradient"):
            calls[name]()
        with torch.no_grad():
            calls[name]()
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(lambda x: cache.tree(x, s["cu"], s["parents"]), (s["q"],), check_trace=False)
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(lambda x: layers.accept(s["cu"], s["parents"], x, s["answers"])[0], (s["ids"],), check_trace=False)
    with torch.inference_mode():
        calls["append"]()
        calls["tree"]()


SMALL = dict(hidden=256, inter=512, layers=3, heads=4, kv_heads=2, head_dim=64, vocab=211, rope_theta=10000.0, eps=1e-6)


def test_the_model_over_drafted_trees(cuda_device):
    """Sequences go on by known tokens, which trees hold among wrong ones: on the path
    that is kept the logits are those of the same tokens one at a time. Both ways
    round activations to bf16 at the same places, a dozen roundings of 2^-8 at most per
    layer of weights' and scores' sums in another order: 3 * 12 * 2^-8 = 0.14 relative."""
    dev, batch = cuda_device, 3
    model = build_qwen2(SMALL, dev, seed=3)
    g, r = torch.Generator().manual_seed(4), random.Random(5)
    prompts = [torch.randint(0, 211, (n,), generator=g).to(dev) for n in (17, 40, 3)]
    goes_on = torch.randint(0, 211, (batch, 40), generator=g)
    with torch.no_grad():
        plain, caches = (model.new_paged_caches(batch, 200) for _ in range(2))
        for c in (plain, caches):
            c.lens.copy_(i32([17, 40, 3], dev))
            model.forward_paged(torch.cat(prompts), c, i32([0, 17, 57, 60], dev))
        logits = []
        for i in range(40):
            plain.lens.add_(1)
            logits.append(model.forward_paged(goes_on[:, i].to(dev), plain).float())
        done, total, longest = [0] * batch, [17, 40, 3], 0
        for _ in range(5):
            trees, ids, answers = [], [], []
            for b in range(batch):
                # the sampled token, then a branch of the known tokens among wrong ones
                tree, words, branch = [-1], [int(goes_on[b, done[b]])], [0]
                for i in range(1, 14):
                    if r.random() < 0.3:
                        words.append(int(goes_on[b, done[b] + len(branch)]))
                        tree.append(branch[-1])
                        branch.append(i)
                    else:
                        tree.append(r.randrange(i))
                        words.append(211)  # no known token
                trees.append(tree)
                ids.append(words)
                answers.append([int(goes_on[b, done[b] + branch.index(i) + 1]) if i in branch else -1 for i in range(14)])
            cu, parents = packed(trees)
            positions = [total[b] + d for b, t in enumerate(trees) for d in depth_of(t)]
            drafted = torch.tensor(sum(ids, []), device=dev)
            caches.lens.copy_(i32([t + 14 for t in total], dev))
            got = model.forward_paged(drafted.clamp(max=210), caches, i32(cu, dev), i32(parents, dev), i32(positions, dev)).float()
            kept, counts, token = caches.together.accept(i32(cu, dev), i32(parents, dev), drafted,
                                                         torch.tensor(sum(answers, []), device=dev))
            caches.together.keep(i32(cu, dev), kept, counts)
            for b in range(batch):
                path = kept[cu[b]:cu[b] + int(counts[b])].tolist()
                assert [ids[b][a] for a in path] == goes_on[b, done[b]:done[b] + len(path)].tolist()
                for i, row in enumerate(path):
                    want = logits[done[b] + i][b]
                    assert (got[cu[b] + row] - want).norm() <= 0.14 * want.norm()
                longest = max(longest, len(path))
                total[b] += len(path)
                done[b] += len(path)
                assert int(token[b]) == int(goes_on[b, done[b]])
            assert caches.lens.tolist() == total
        assert longest >= 4
        caches.together.check_status()
        with pytest.raises(ValueError, match="cu_seqlens"):
            model.forward_paged(drafted[:3], caches, parents=i32([-1] * 3, dev))


def test_the_model_rotates_by_several_axes(cuda_device):
    """Positions that are the slots' on every axis give what slots give; others do not."""
    dev = cuda_device
    model = build_qwen2(dict(SMALL, rope_sections=(8, 12, 12)), dev, seed=3)
    ids = torch.randint(0, 211, (50,), generator=torch.Generator().manual_seed(6)).to(dev)
    cu, place = i32([0, 50], dev), torch.arange(50, dtype=torch.int32, device=dev)
    with torch.no_grad():
        out = []
        for positions in (None, place.repeat(3, 1), torch.stack((place, place // 7, place % 7))):
            caches = model.new_paged_caches(1, 64)
            caches.lens.fill_(50)
            out.append(model.forward_paged(ids, caches, cu, positions=positions))
            caches.together.check_status()
    assert torch.equal(out[0], out[1]) and not torch.equal(out[0], out[2])
