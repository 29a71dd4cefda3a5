"""Paged key-value cache operators: what is measured, and their plain forms.

Three operators that a decoder layer runs one after another on the same cache:

* ``append``: the new tokens' keys and values go into the pages, q and k
  rotated by position on the way;
* ``decode``: attention of one new token per sequence over its pages;
* ``prefill``: causal attention of prompt chunks over the pages.

A case gives the head layout, the page size, the type, and how long the
sequences are: ``new`` tokens of this call (at most) after ``past`` cached ones
(at most). ``ragged`` spreads both over the batch; ``idle`` leaves every fifth
slot of a decode batch without a sequence (length 0), as a batch of fixed
size has them. ``run`` with ``own`` false computes in elementary torch
operations in 32 bits.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _case(name, op, batch, new, past, heads, kv_heads, head_dim, page, dtype, ragged=False, idle=False):
    return dict(name=name, op=op, batch=batch, new=new, past=past, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, page=page, dtype=dtype, ragged=ragged, idle=idle)


def listed():
    return [
        # one decoded token of one sequence: launch latency
        _case("append_one", "append", 1, 1, 512, 28, 4, 128, 16, "bf16"),
        # a decode step of a serving batch
        _case("append_step", "append", 64, 1, 4096, 32, 32, 128, 64, "f16", ragged=True),
        # several prompts written at once
        _case("append_prompts", "append", 5, 2048, 1000, 28, 4, 128, 16, "bf16"),
        # the first decoded tokens after a 512-token prompt
        _case("decode_one", "decode", 1, 1, 528, 28, 4, 128, 16, "bf16"),
        # a serving batch of unlike lengths, some slots without a sequence
        _case("decode_batch", "decode", 37, 1, 4096, 28, 4, 128, 16, "bf16", ragged=True, idle=True),
        # no shared heads, larger pages, a dialogue's length
        _case("decode_heads", "decode", 8, 1, 2047, 32, 32, 128, 64, "f16"),
        # one long document
        _case("decode_long", "decode", 1, 1, 131071, 28, 4, 128, 32, "bf16"),
        # a full serving batch
        _case("decode_full", "decode", 64, 1, 8191, 28, 4, 128, 16, "bf16"),
        # the 512-token prompt
        _case("prefill_512", "prefill", 1, 512, 0, 28, 4, 128, 16, "bf16"),
        # one long prompt
        _case("prefill_long", "prefill", 1, 8192, 0, 28, 4, 128, 16, "bf16"),
        # prompts and chunks of unlike length behind cached prefixes, no shared heads
        _case("prefill_ragged", "prefill", 7, 1500, 1111, 32, 32, 64, 32, "f16", ragged=True),
        # a few draft tokens per sequence, looked at behind long caches
        _case("prefill_drafts", "prefill", 9, 5, 7777, 28, 4, 128, 16, "bf16", ragged=True),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    while True:
        op = rng.choice(["append", "decode", "prefill"])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 16, 32])
        group = rng.choice([1, 2, 3, 4, 6, 7, 8, 12, 16])
        head_dim = rng.choice([64, 128, 128])
        case = dict(op=op, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                    page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "f16"]),
                    ragged=rng.random() < 0.6, idle=False)
        if op == "append":
            case.update(batch=_log_int(rng, 1, 96), new=_log_int(rng, 1, 4096), past=_log_int(rng, 1, 4096) - 1)
        elif op == "decode":
            case.update(batch=_log_int(rng, 1, 128), new=1, past=_log_int(rng, 1, 131072) - 1,
                        idle=rng.random() < 0.3)
        else:
            case.update(batch=_log_int(rng, 1, 16), new=_log_int(rng, 1, 4096), past=_log_int(rng, 1, 16384) - 1)
        if case["heads"] > 64:
            continue
        slots = case["batch"] * (case["new"] + case["past"])
        if slots * kv_heads * head_dim * 4 > 1.0e9:  # the cache's bytes
            continue
        if case["batch"] * case["new"] * (case["heads"] + 2 * kv_heads) * head_dim * 2 > 1.0e8:  # the new tokens'
            continue
        if op == "prefill" and case["batch"] * case["heads"] * case["new"] * (case["new"] + case["past"]) > 1.5e9:
            continue
        return case


def _lengths(case):
    """(new, total) tokens of each sequence: a function of the case alone."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    new, total = [], []
    for b in range(case["batch"]):
        n, p = case["new"], case["past"]
        if case["ragged"] and b:
            n, p = _log_int(r, 1, n), _log_int(r, 1, p + 1) - 1
        if case["idle"] and b % 5 == 4:
            n, p = 0, 0
        new.append(n)
        total.append(n + p)
    return new, total


def prepare(case, seed):
    dev = torch.device("cuda")
    dt = _DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    new, total = _lengths(case)
    page, heads, hk, d = case["page"], case["heads"], case["kv_heads"], case["head_dim"]
    count = [-(-n // page) for n in total]
    width = max(1, max(count))
    pages = sum(count) + 3  # a few that no sequence holds
    # pages are handed out in no order, as after many requests have come and gone
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32).cpu()
    table = torch.zeros(case["batch"], width, dtype=torch.int32)
    at = 0
    for b, c in enumerate(count):
        table[b, :c] = order[at:at + c]
        at += c
    tokens = sum(new) if case["op"] != "decode" else case["batch"]
    state = dict(op=case["op"], max_new=max(new), k_pages=torch.empty(pages, hk, page, d, dtype=dt, device=dev).normal_(generator=g),
                 v_pages=torch.empty(pages, hk, page, d, dtype=dt, device=dev).normal_(generator=g),
                 table=table.to(dev), lens=torch.tensor(total, dtype=torch.int32, device=dev), cu=None, rope=None)
    if case["op"] == "append":
        # q, k, v are the fused projection's output, as the layer's linear gives it
        qkv = torch.empty(tokens, (heads + 2 * hk) * d, dtype=dt, device=dev).normal_(generator=g)
        q, k, v = qkv.split([heads * d, hk * d, hk * d], dim=-1)
        state.update(q=q.view(tokens, heads, d), k=k.view(tokens, hk, d), v=v.view(tokens, hk, d))
        angle = torch.outer(torch.arange(max(total), device=dev, dtype=torch.float64), _inverse(d, dev))
        state["rope"] = torch.stack((angle.cos(), angle.sin()), dim=-1).float()  # [positions, d / 2, 2]
    else:
        # scores spread by about 1.5, as trained heads' do before the softmax
        state["q"] = (1.5 * torch.randn(tokens, heads, d, generator=g, device=dev)).to(dt)
    if case["op"] != "decode":
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        state["cu"] = torch.tensor(cu, dtype=torch.int32, device=dev)
    if own:
        from vla_abft_estimate_b200.paged import PagedKVCache

        state["cache"] = PagedKVCache(state["k_pages"], state["v_pages"], state["table"], state["lens"])
    return state


def _inverse(d, dev):
    return 1.0e6 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)


def run(state):
    if own:
        cache = state["cache"]
        if state["op"] == "append":
            q = cache.append(state["q"], state["k"], state["v"], state["rope"], cu_seqlens=state["cu"])
            return q, state["k_pages"], state["v_pages"]
        if state["op"] == "decode":
            return cache.decode(state["q"])
        return cache.prefill(state["q"], state["cu"])
    return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill}[state["op"]](state)


def _owners(cu, tokens):
    """The sequence of each packed token, and its place among that sequence's new tokens."""
    t = torch.arange(tokens, device=cu.device)
    seq = (t[:, None] >= cu[None, 1:]).sum(1)
    return seq, t - cu[seq]


def _plain_append(s):
    seq, place = _owners(s["cu"], s["q"].shape[0])
    count = s["cu"][1:] - s["cu"][:-1]
    pos = s["lens"][seq] - count[seq] + place
    turn = s["rope"][pos][:, None]  # [tokens, 1, d / 2, 2]
    cos, sin = turn[..., 0], turn[..., 1]

    def rotated(x):
        a, b = x.float().chunk(2, dim=-1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).to(x.dtype)

    size = s["k_pages"].shape[2]
    page, slot = s["table"][seq, pos // size].long(), (pos % size).long()
    s["k_pages"][page, :, slot] = rotated(s["k"])
    s["v_pages"][page, :, slot] = s["v"]
    return rotated(s["q"]), s["k_pages"], s["v_pages"]


def _gathered(pages, table):
    """[batch, kv_heads, slots, d] in 32 bits, in the sequences' order."""
    x = pages[table.long()].float()  # [batch, pages, kv_heads, size, d]
    b, n, h, size, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, n * size, d)


def _attend(q, k, v, seen):
    """q [b, h, g, n, d] over k, v [b, h, slots, d]; ``seen`` [b, n, slots]. A row that sees nothing gives 0."""
    x = torch.matmul(q, k[:, :, None].transpose(-1, -2)) / math.sqrt(q.shape[-1])
    x = torch.where(seen[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = x.sum(-1, keepdim=True)
    return torch.matmul(x, v[:, :, None]) / torch.where(total == 0, 1.0, total)


def _plain_decode(s):
    q = s["q"]
    b, heads, d = q.shape
    k, v = _gathered(s["k_pages"], s["table"]), _gathered(s["v_pages"], s["table"])
    hk = k.shape[1]
    seen = torch.arange(k.shape[2], device=q.device)[None, None] < s["lens"][:, None, None]
    o = _attend(q.float().view(b, hk, heads // hk, 1, d), k, v, seen)
    return o.reshape(b, heads, d).to(q.dtype)


def _plain_prefill(s):
    q = s["q"]
    tokens, heads, d = q.shape
    seq, place = _owners(s["cu"], tokens)
    count = s["cu"][1:] - s["cu"][:-1]
    k, v = _gathered(s["k_pages"], s["table"]), _gathered(s["v_pages"], s["table"])
    b, hk, n = k.shape[0], k.shape[1], s["max_new"]
    padded = torch.zeros(b, n, heads, d, device=q.device)
    padded[seq, place] = q.float()
    last = (s["lens"] - count)[:, None] + torch.arange(n, device=q.device)
    seen = torch.arange(k.shape[2], device=q.device)[None, None] <= last[:, :, None]
    o = _attend(padded.view(b, n, hk, heads // hk, d).permute(0, 2, 3, 1, 4), k, v, seen)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, heads, d)[seq, place].to(q.dtype)


def work(case):
    new, total = _lengths(case)
    heads, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    tokens = sum(new)
    if case["op"] == "append":  # q, k, v in; q and the new slots out; each token's row of the rotation table
        return {"bytes": 2 * tokens * (heads + 2 * hk) * d * 2 + tokens * d * 4, "flops": 3 * tokens * (heads + hk) * d}
    if case["op"] == "decode":  # the caches' valid slots, q in and out (idle slots' rows too)
        return {"bytes": sum(total) * hk * d * 4 + 2 * case["batch"] * heads * d * 2, "flops": 4 * sum(total) * heads * d}
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    return {"bytes": sum(total) * hk * d * 4 + 2 * tokens * heads * d * 2, "flops": 4 * pairs * heads * d}


def exact(case, seed):
    """In 64 bits, sequence by sequence, from the definition."""
    s = prepare(case, seed)
    new, total = _lengths(case)
    size, hk, d, heads = case["page"], case["kv_heads"], case["head_dim"], case["heads"]
    table = s["table"].tolist()
    if case["op"] == "append":
        q_out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        k_out, v_out = s["k_pages"].double(), s["v_pages"].double()
        at = 0
        for b, (n, t) in enumerate(zip(new, total)):
            p = torch.arange(t - n, t, device="cuda")
            z = torch.polar(torch.ones(n, d // 2, dtype=torch.float64, device="cuda"), torch.outer(p.double(), _inverse(d, "cuda")))[:, None]

            def turn(x):
                x = x.double()
                w = torch.complex(x[..., : d // 2], x[..., d // 2:]) * z
                return torch.cat((w.real, w.imag), dim=-1)

            q_out[at:at + n] = turn(s["q"][at:at + n])
            held = torch.tensor(table[b], device="cuda")[p // size]
            k_out[held, :, p % size] = turn(s["k"][at:at + n])
            v_out[held, :, p % size] = s["v"][at:at + n].double()
            at += n
        return q_out, k_out, v_out
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (n, t) in enumerate(zip(new, total)):
        rows = slice(b, b + 1) if case["op"] == "decode" else slice(at, at + n)
        at += n
        if n == 0:
            continue
        held = table[b][: -(-t // size)]
        for h in range(hk):
            k = torch.cat([s["k_pages"][held[i:i + 512], h].double() for i in range(0, len(held), 512)]).reshape(-1, d)[:t]
            v = torch.cat([s["v_pages"][held[i:i + 512], h].double() for i in range(0, len(held), 512)]).reshape(-1, d)[:t]
            for j in range(h * heads // hk, (h + 1) * heads // hk):
                x = s["q"][rows, j].double() @ k.T * d ** -0.5
                hidden = torch.arange(t, device="cuda")[None] > torch.arange(t - n, t, device="cuda")[:, None]
                w = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1)
                out[rows, j] = w @ v
    return out
