"""The operators of serving over a pool of cache pages, as cases that a timing harness can run: rotary positions, appending the new
tokens of ragged sequences to their pages, attention of new tokens over the pages, and the pages' own maintenance (beams that follow their
parents and copy on write, page copies, compaction).

    listed()             the cases by name
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  the tensors that a serving program holds before the call, on the GPU
    run(state)           one pass: in plain torch, or with `own` through the framework's entry points
    exact(case, seed)    what that pass computes, in 64 bits
    work(case)           the bytes and floating-point operations that one pass cannot do without

A pool is [planes, pages, key heads, page tokens, head size]: a plane each for the keys and the values of every layer. Row b of the page table
lists the pages of sequence b in order, -1 behind the last.
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One decoding step of a batch: the queries and keys of one token a request, far into long contexts (frequencies stretched for them).
        {"name": "rotary_bf16_t64_far", "kind": "rotary", "dtype": "bf16", "tokens": 64, "heads": 32, "kv_heads": 8, "d": 128, "rotary": 128,
         "interleaved": False, "reach": 500000, "stretch": 8.0, "scale": 1.2},
        # The prompts of a packed batch, pairs side by side, half of every head turned.
        {"name": "rotary_f16_t15000_part", "kind": "rotary", "dtype": "f16", "tokens": 15000, "heads": 16, "kv_heads": 16, "d": 64, "rotary": 32,
         "interleaved": True, "reach": 2048, "stretch": 1.0, "scale": 1.0},
        # A decoding step of many requests: their new keys are turned and filed, the queries turned, in one pass.
        {"name": "append_bf16_b200_step", "kind": "append", "dtype": "bf16", "batch": 200, "new_low": 1, "new_high": 1, "past_low": 0, "past_high": 700,
         "heads": 32, "kv_heads": 8, "d": 128, "page": 16, "rotary": 128, "interleaved": False},
        # Prompts of different lengths filed behind what their conversations already hold.
        {"name": "append_f16_b9_prompts", "kind": "append", "dtype": "f16", "batch": 9, "new_low": 150, "new_high": 1800, "past_low": 0, "past_high": 600,
         "heads": 32, "kv_heads": 8, "d": 128, "page": 64, "rotary": 64, "interleaved": True},
        # One user's next token over a long conversation: the smallest call of the attention, latency.
        {"name": "attend_bf16_b1_k8000", "kind": "attend", "dtype": "bf16", "batch": 1, "new_low": 1, "new_high": 1, "past_low": 8000, "past_high": 8000,
         "heads": 32, "kv_heads": 8, "d": 128, "page": 16, "causal": True},
        # A decoding step of a batch of GPT-2's head layout, lengths all over the place.
        {"name": "attend_f16_b64_heads12", "kind": "attend", "dtype": "f16", "batch": 64, "new_low": 1, "new_high": 1, "past_low": 20, "past_high": 4000,
         "heads": 12, "kv_heads": 12, "d": 64, "page": 16, "causal": True},
        # A few proposed tokens a request, checked together: more rows than one, eight query heads to a key head.
        {"name": "attend_bf16_b16_n5", "kind": "attend", "dtype": "bf16", "batch": 16, "new_low": 3, "new_high": 6, "past_low": 1000, "past_high": 16000,
         "heads": 64, "kv_heads": 8, "d": 128, "page": 32, "causal": True},
        # Prompts of a ragged batch, some of which continue a cached beginning.
        {"name": "attend_f16_b6_prompts", "kind": "attend", "dtype": "f16", "batch": 6, "new_low": 200, "new_high": 2000, "past_low": 0, "past_high": 3000,
         "heads": 16, "kv_heads": 16, "d": 64, "page": 64, "causal": True},
        # A chunk of one long prompt over what was read of it so far: the largest.
        {"name": "attend_bf16_b1_n4000_k12000", "kind": "attend", "dtype": "bf16", "batch": 1, "new_low": 4000, "new_high": 4000, "past_low": 12000,
         "past_high": 12000, "heads": 32, "kv_heads": 8, "d": 128, "page": 16, "causal": True},
        # A beam search's step between two passes: the beams follow their parents, some requests end, every beam gets room for its next token and a page
        # of its own where it shares the one that it would write to.
        {"name": "beams_f16_b64", "kind": "beams", "dtype": "f16", "batch": 64, "past_low": 40, "past_high": 500, "planes": 24, "kv_heads": 12, "d": 64,
         "page": 16, "width": 64, "spare": 200},
        # Pages of a prefix duplicated in every layer.
        {"name": "copy_bf16_p300", "kind": "copy", "dtype": "bf16", "pages": 900, "copies": 301, "planes": 24, "kv_heads": 8, "d": 128, "page": 16},
        # A pool after many requests have come and gone, packed to its front so that its rear can be given back.
        {"name": "compact_f16_p3000", "kind": "compact", "dtype": "f16", "batch": 48, "past_low": 10, "past_high": 900, "pages": 3001, "planes": 16, "kv_heads": 8,
         "d": 64, "page": 16, "width": 64},
    ]


def _spread(rng, low, high):
    """A whole number from [low, high], uniform over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(max(low, 1)), math.log(max(high, 1))))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend", "attend", "beams", "copy", "compact"])
    case = {"kind": kind, "dtype": rng.choice(["f16", "bf16"]), "page": rng.choice([16, 16, 32, 64, 128])}
    kv_heads, d = rng.choice([(1, 128), (2, 128), (8, 64), (8, 128), (12, 64), (16, 64), (5, 64)])
    case |= {"kv_heads": kv_heads, "d": d}
    if kind == "rotary":
        del case["page"]
        case |= {"dtype": rng.choice(["f16", "bf16", "f32"]), "tokens": _spread(rng, 1, 15000), "heads": kv_heads * rng.choice([1, 2, 4]),
                 "rotary": rng.choice([d, d, d // 2, d // 4]), "interleaved": rng.random() < 0.5, "reach": _spread(rng, 100, 1000000),
                 "stretch": rng.choice([1.0, 4.0, 16.0]), "scale": rng.choice([1.0, 1.1])}
    elif kind == "append":
        steps = rng.random() < 0.5
        high = 1 if steps else _spread(rng, 2, 1500)
        case |= {"batch": _spread(rng, 1, 200 if steps else 8), "new_low": 1 if steps else rng.randint(1, high), "new_high": high, "past_low": 0,
                 "past_high": _spread(rng, 1, 700), "heads": kv_heads * rng.choice([1, 2, 4]), "rotary": rng.choice([d, d, d // 2]),
                 "interleaved": rng.random() < 0.5}
    elif kind == "attend":
        heads = kv_heads * rng.choice([1, 2, 4, 7, 8] if kv_heads < 12 else [1])
        high = rng.choice([1, 1, rng.randint(2, 8), _spread(rng, 9, 200), _spread(rng, 200, 3000)])
        past = _spread(rng, 1, 16000)
        # the scores of the padded batch and its keys stay within what the largest listed cases hold
        most = min(int(1e9 / (heads * high * (past + high))), int(1e9 / (kv_heads * d * (past + high))), 100)
        case |= {"batch": _spread(rng, 1, max(1, most)), "new_low": rng.randint(1, high) if high > 1 else 1, "new_high": high,
                 "past_low": rng.choice([0, past // 10, past]), "past_high": past, "heads": heads, "causal": rng.random() < 0.85}
    elif kind == "beams":
        past = _spread(rng, 10, 500)
        case |= {"batch": _spread(rng, 2, 64), "past_low": rng.randint(1, past), "past_high": past, "planes": rng.choice([2, 8, 24]), "page": rng.choice([16, 32]),
                 "width": 64, "spare": rng.randint(70, 200)}
    elif kind == "copy":
        pages = _spread(rng, 8, 900) if case["page"] <= 32 else _spread(rng, 8, 200)
        case |= {"pages": pages, "copies": rng.randint(1, pages // 3), "planes": rng.choice([2, 8, 24])}
    else:
        past, batch = _spread(rng, 10, 900), _spread(rng, 1, 48)
        case |= {"batch": batch, "past_low": rng.randint(1, past), "past_high": past, "pages": batch * (past // case["page"] + 1) + rng.randint(5, 200),
                 "planes": rng.choice([2, 8, 16]), "width": past // case["page"] + 5}
    return case


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
def _lengths(case):
    """(new tokens, cached tokens) of every sequence: they belong to the case, as its work does."""
    rng = random.Random("%(batch)d %(past_low)d %(past_high)d" % case)
    past = [rng.randint(case["past_low"], case["past_high"]) for _ in range(case["batch"])]
    return [rng.randint(case.get("new_low", 1), case.get("new_high", 1)) for _ in range(case["batch"])], past


def _frequencies(case):
    half = case["rotary"] // 2
    exponents = torch.arange(half, dtype=torch.float64, device=DEVICE) / half
    return 10000.0 ** -exponents / case.get("stretch", 1.0)


def _values(g, *shape, dtype):
    return torch.randn(*shape, device=DEVICE, generator=g, dtype=dtype)


def _table(g, tokens, page, pages, width):
    """A page table over scattered pages: (table [B, width] int32, references [pages] int32)."""
    tokens = torch.tensor(tokens, device=DEVICE)
    counts = (tokens + page - 1) // page
    order = torch.randperm(pages, device=DEVICE, generator=g)
    column = torch.arange(width, device=DEVICE)
    taken = (counts.cumsum(0) - counts)[:, None] + column
    live = column < counts[:, None]
    table = torch.where(live, order[taken.clamp(max=pages - 1)], -1).to(torch.int32)
    refs = torch.zeros(pages, device=DEVICE, dtype=torch.int32)
    refs[table[live].long()] = 1
    return table, refs


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"case": dict(case)}
    if kind == "rotary":
        T, Hq, Hk, d = case["tokens"], case["heads"], case["kv_heads"], case["d"]
        rows = _values(g, T, (Hq + 2 * Hk) * d, dtype=dtype)  # what the projection leaves: queries | keys | values
        return state | {"q": rows[:, :Hq * d].view(T, Hq, d), "k": rows[:, Hq * d:(Hq + Hk) * d].view(T, Hk, d), "freqs": _frequencies(case),
                        "positions": torch.randint(0, case["reach"], (T,), device=DEVICE, generator=g)}
    if kind in ("append", "attend"):
        new, past = _lengths(case)
        T, Hq, Hk, d, page = sum(new), case["heads"], case["kv_heads"], case["d"], case["page"]
        most = max(n + p for n, p in zip(new, past))
        pages = sum((n + p + page - 1) // page for n, p in zip(new, past)) + 3
        table, _ = _table(g, [n + p for n, p in zip(new, past)], page, pages, (most + page - 1) // page + 2)
        pool = _values(g, 2, pages, Hk, page, d, dtype=dtype)
        cu = torch.tensor([0] + new, device=DEVICE).cumsum(0).to(torch.int32)
        state |= {"keys": pool[0], "values": pool[1], "table": table, "cu": cu, "past": torch.tensor(past, device=DEVICE, dtype=torch.int32),
                  "max_new": max(new), "max_keys": most}
        rows = _values(g, T, (Hq + 2 * Hk) * d, dtype=dtype)
        state |= {"q": rows[:, :Hq * d].view(T, Hq, d)}
        if kind == "append":
            state |= {"k": rows[:, Hq * d:(Hq + Hk) * d].view(T, Hk, d), "v": rows[:, (Hq + Hk) * d:].view(T, Hk, d), "freqs": _frequencies(case)}
        return state
    Hk, d, page = case["kv_heads"], case["d"], case["page"]
    if kind == "copy":
        pool = _values(g, case["planes"], case["pages"], Hk, page, d, dtype=dtype)
        order = torch.randperm(case["pages"], device=DEVICE, generator=g)[:2 * case["copies"]]
        return state | {"pool": pool, "copies": order.view(-1, 2).to(torch.int32)}
    _, past = _lengths(case)
    pages = case["pages"] if kind == "compact" else sum((p + page - 1) // page for p in past) + case["spare"]
    table, refs = _table(g, past, page, pages, case["width"])
    state |= {"pool": _values(g, case["planes"], pages, Hk, page, d, dtype=dtype), "table": table, "refs": refs}
    if kind == "beams":
        B = case["batch"]
        parents = torch.randint(0, B, (B,), device=DEVICE, generator=g)
        alone = torch.rand(B, device=DEVICE, generator=g)
        parents = torch.where(alone < 0.4, torch.arange(B, device=DEVICE), parents)  # many a beam goes on by itself
        parents = torch.where(alone > 0.95, -1, parents).to(torch.int32)             # a few requests have ended
        state |= {"lens": torch.tensor(past, device=DEVICE, dtype=torch.int32), "parents": parents, "new": (parents >= 0).to(torch.int32)}
    return state


# ---------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------
def _turn(x, positions, freqs, interleaved, scale):
    angles = positions.double()[:, None] * freqs
    cos, sin = (angles.cos() * scale).float()[:, None], (angles.sin() * scale).float()[:, None]
    half, y = freqs.numel(), x.float()
    a, b = (y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if interleaved else (y[..., :half], y[..., half:2 * half])
    turned = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((turned, y[..., 2 * half:]), -1).to(x.dtype)


def _owners(cu, tokens):
    """(sequence, place in its new tokens) of every token."""
    at = torch.arange(tokens, device=cu.device)
    owner = torch.searchsorted(cu, at, right=True) - 1
    return owner, at - cu[owner]


def _append(s, interleaved, scale):
    owner, i = _owners(s["cu"], s["k"].shape[0])
    position, page = s["past"][owner] + i, s["keys"].shape[2]
    to, slot = s["table"][owner, position // page].long(), position % page
    s["keys"][to, :, slot] = _turn(s["k"], position, s["freqs"], interleaved, scale)
    s["values"][to, :, slot] = s["v"]
    return _turn(s["q"], position, s["freqs"], interleaved, scale), s["keys"], s["values"]


def _attend(s, causal, scale):
    q, cu, past = s["q"], s["cu"].long(), s["past"].long()
    page, (T, Hq, d), Hk, B = s["keys"].shape[2], q.shape, s["keys"].shape[1], past.numel()
    used, M = (s["max_keys"] + page - 1) // page, s["max_new"]
    pages, new = s["table"][:, :used].clamp(min=0).long(), cu.diff()
    key = torch.arange(used * page, device=q.device)
    there = key < (past + new)[:, None]
    k = s["keys"][pages].permute(0, 2, 1, 3, 4).reshape(B, Hk, used * page, d).float()
    v = s["values"][pages].permute(0, 2, 1, 3, 4).reshape(B, Hk, used * page, d).float().masked_fill(~there[:, None, :, None], 0)
    rows = (cu[:-1, None] + torch.arange(M, device=q.device)).clamp(max=T - 1)
    x = q[rows].view(B, M, Hk, Hq // Hk, d).permute(0, 2, 3, 1, 4).reshape(B, Hk, Hq // Hk * M, d).float()
    scores = (x @ k.transpose(-1, -2) * scale).view(B, Hk, Hq // Hk, M, used * page)
    seen = there[:, None]
    if causal:
        seen = seen & (key <= (past[:, None] + torch.arange(M, device=q.device))[..., None])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores = (scores - scores.amax(-1, keepdim=True)).exp_()
    out = (scores / scores.sum(-1, keepdim=True)).view(B, Hk, Hq // Hk * M, used * page) @ v
    owner, i = _owners(cu, T)
    return out.view(B, Hk, Hq // Hk, M, d).permute(0, 3, 1, 2, 4).reshape(B, M, Hq, d)[owner, i].to(q.dtype)


def _count(refs, table, sign):
    flat = table.flatten().long()
    refs.index_add_(0, flat.clamp(min=0), torch.where(flat >= 0, sign, 0).to(torch.int32))


def _fork(table, lens, refs, parents):
    kept, ended = table[parents.clamp(min=0).long()], parents < 0
    kept = kept.masked_fill(ended[:, None], -1)
    _count(refs, kept, 1)
    _count(refs, table, -1)
    table.copy_(kept)
    lens.copy_(lens[parents.clamp(min=0).long()].masked_fill(ended, 0))


def _reserve(table, lens, refs, new, page):
    """Pages for `new` more tokens of every row, the lowest free ones in the rows' order. A row that would write to a page it shares gets one of its own in
    its place: of rows that are all a page's holders, the last keeps it. From the first row on that the pages do not suffice for, nothing is granted."""
    B, width = table.shape
    row, writes = torch.arange(B, device=table.device), new > 0
    fits = (lens + new + page - 1) // page <= width
    have, want = (lens + page - 1) // page, (lens + new + page - 1) // page
    last = table.gather(1, (have - 1).clamp(min=0).long()[:, None])[:, 0]
    open_ = writes & fits & (lens % page != 0) & (last >= 0)
    at = last.clamp(min=0).long()
    sharers = torch.zeros_like(refs).index_add_(0, at, open_.to(torch.int32))
    keeper = torch.full_like(refs, -1).scatter_reduce_(0, at, torch.where(open_, row, -1).to(torch.int32), "amax")
    copies = open_ & (refs[at] > 1) & ~((sharers[at] == refs[at]) & (keeper[at] == row))
    need = torch.where(writes & fits, want - have + copies.to(torch.int32), 0)
    until = need.cumsum(0)
    free = torch.sort((refs > 0).to(torch.int32), stable=True).indices.to(torch.int32)
    count = (refs <= 0).sum()
    granted = ~writes | (fits & (until <= count))
    copies &= granted
    column = torch.arange(width, device=table.device)
    first = torch.where(copies, have - 1, have)
    gets = (granted & writes)[:, None] & (column >= first[:, None]) & (column < want[:, None])
    taken = (until - need)[:, None] + column - first[:, None]
    fresh = torch.where(gets, free[taken.clamp(0, refs.numel() - 1)], table)
    refs.index_add_(0, at, -copies.to(torch.int32))
    refs.index_add_(0, fresh.flatten().clamp(min=0).long(), gets.flatten().to(torch.int32))
    pairs = torch.stack((last, fresh.gather(1, (have - 1).clamp(min=0).long()[:, None])[:, 0]), 1)
    order = torch.sort((~copies).to(torch.int32), stable=True).indices
    pairs = torch.where(copies[order, None], pairs[order], -1)
    table.copy_(fresh)
    return granted.to(torch.int32), pairs.to(torch.int32)


def _copy(pool, pairs):
    """Page pairs[i, 1] of every plane becomes a copy of page pairs[i, 0]; pairs of -1 are left out."""
    at = pairs[pairs[:, 0] >= 0].long()
    pool[:, at[:, 1]] = pool[:, at[:, 0]]


def _compact(table, refs, pool):
    """The pages in use move to the front: those behind it, in order, into the free ones within it, in order."""
    live = refs > 0
    count, at = live.sum(), torch.arange(refs.numel(), device=refs.device)
    out, hole = (live & (at >= count)).nonzero()[:, 0], (~live & (at < count)).nonzero()[:, 0]
    pool[:, hole] = pool[:, out]
    to = at.scatter(0, out, hole)
    refs[hole] = refs[out]
    refs[out] = 0
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    return count.to(torch.int32)


def run(state):
    if own:
        import turbotransformers_b200 as tt
    s, case = state, state["case"]
    kind, scale = case["kind"], case.get("scale", 1.0)
    if kind == "rotary":
        if own:
            return tt.rotary(s["q"], s["k"], s["positions"], s["freqs"], interleaved=case["interleaved"], scale=scale)
        return tuple(_turn(s[x], s["positions"], s["freqs"], case["interleaved"], scale) for x in ("q", "k"))
    if kind == "append":
        if own:
            q = tt.paged_append(s["k"], s["v"], s["keys"], s["values"], s["table"], s["cu"], s["past"], q=s["q"], freqs=s["freqs"],
                                interleaved=case["interleaved"], scale=scale)
            return q, s["keys"], s["values"]
        return _append(s, case["interleaved"], scale)
    if kind == "attend":
        if own:
            return tt.paged_attention(s["q"], s["keys"], s["values"], s["table"], s["cu"], s["past"], causal=case["causal"])
        return _attend(s, case["causal"], case["d"] ** -0.5)
    if kind == "copy":
        tt.paged_copy(s["pool"], s["copies"]) if own else _copy(s["pool"], s["copies"])
        return s["pool"]
    # what these change of the table is made anew for every pass, so that each has the same to do
    table, refs = s["table"].clone(), s["refs"].clone()
    if kind == "compact":
        count = tt.paged_compact(table, refs, s["pool"]) if own else _compact(table, refs, s["pool"])
        return table, refs, s["pool"], count.reshape(())
    lens = s["lens"].clone()
    if own:
        tt.paged_fork(table, lens, refs, s["parents"])
        granted, copies = tt.paged_reserve(table, lens, refs, s["new"], case["page"])
        tt.paged_copy(s["pool"], copies)
    else:
        _fork(table, lens, refs, s["parents"])
        granted, copies = _reserve(table, lens, refs, s["new"], case["page"])
        _copy(s["pool"], copies)
    return table, lens, refs, granted, copies, s["pool"]


# ---------------------------------------------------------------------------------------------------
# the definition in 64 bits, one sequence, head, row or page after the other
# ---------------------------------------------------------------------------------------------------
def _turn64(x, positions, freqs, interleaved, scale):
    """Pairs as complex numbers, multiplied by scale * e^(i angle)."""
    x, n = x.double().clone(), freqs.numel()
    turn = torch.polar(torch.full((positions.numel(), n), scale, dtype=torch.float64, device=x.device), positions.double()[:, None] * freqs)[:, None]
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    kind, scale = case["kind"], case.get("scale", 1.0)
    if kind == "rotary":
        return tuple(_turn64(s[x], s["positions"], s["freqs"], case["interleaved"], scale) for x in ("q", "k"))
    if kind == "append":
        new, past = _lengths(case)
        table, page, t = s["table"].tolist(), case["page"], 0
        position = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)]).to(DEVICE)
        k = _turn64(s["k"], position, s["freqs"], case["interleaved"], scale)
        keys, values = s["keys"].double(), s["values"].double()
        for b, (n, p) in enumerate(zip(new, past)):
            for j in range(p, p + n):
                keys[table[b][j // page], :, j % page], values[table[b][j // page], :, j % page] = k[t], s["v"][t].double()
                t += 1
        return _turn64(s["q"], position, s["freqs"], case["interleaved"], scale), keys, values
    if kind == "attend":
        new, past = _lengths(case)
        group, t, out = case["heads"] // case["kv_heads"], 0, torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
        for b, (n, p) in enumerate(zip(new, past)):
            pages = s["table"][b, :(n + p + case["page"] - 1) // case["page"]].long()
            hidden = torch.arange(n + p, device=DEVICE) > (p + torch.arange(n, device=DEVICE) if case["causal"] else torch.full((n,), n + p, device=DEVICE))[:, None]
            for h in range(case["kv_heads"]):
                k, v = (s[x][pages, h].reshape(-1, case["d"])[:n + p].double() for x in ("keys", "values"))
                for g in range(h * group, (h + 1) * group):
                    scores = (s["q"][t:t + n, g].double() @ k.T * case["d"] ** -0.5).masked_fill_(hidden, -math.inf)
                    out[t:t + n, g] = torch.softmax(scores, -1) @ v
            t += n
        return out
    pool = s["pool"]  # pages are moved as they are: their values have no rounding
    if kind == "copy":
        source = pool.clone()
        for a, b in s["copies"].tolist():
            pool[:, b] = source[:, a]
        return pool.double()
    table, refs = s["table"].tolist(), s["refs"].tolist()
    if kind == "compact":
        count = sum(r > 0 for r in refs)
        holes, to = iter([p for p in range(count) if refs[p] <= 0]), {}
        for p in range(count, len(refs)):
            if refs[p] > 0:
                to[p] = next(holes)
                pool[:, to[p]] = pool[:, p]
                refs[to[p]], refs[p] = refs[p], 0
        table = [[to.get(p, p) for p in row] for row in table]
        return torch.tensor(table), torch.tensor(refs), pool.double(), torch.tensor(count)
    page, lens, new = case["page"], s["lens"].tolist(), s["new"].tolist()
    parents = s["parents"].tolist()
    before, table = table, [list(table[p]) if p >= 0 else [-1] * case["width"] for p in parents]
    lens = [lens[p] if p >= 0 else 0 for p in parents]
    for rows, sign in ((table, 1), (before, -1)):
        for p in (p for row in rows for p in row if p >= 0):
            refs[p] += sign
    free, copies, granted, stopped = [p for p, r in enumerate(refs) if r <= 0], [], [], False
    for b, row in enumerate(table):
        have, want = -(-lens[b] // page), -(-(lens[b] + new[b]) // page)
        shared = new[b] > 0 and lens[b] % page and refs[row[have - 1]] > 1
        stopped |= want - have + bool(shared) > len(free)
        granted.append(int(not stopped or not new[b]))
        if stopped or not new[b]:
            continue
        if shared:
            refs[row[have - 1]] -= 1
            copies.append([row[have - 1], free[0]])
            row[have - 1] = free.pop(0)
            refs[row[have - 1]] += 1
        for c in range(have, want):
            row[c] = free.pop(0)
            refs[row[c]] += 1
    for a, b in copies:
        pool[:, b] = pool[:, a]
    copies += [[-1, -1]] * (len(table) - len(copies))
    return torch.tensor(table), torch.tensor(lens), torch.tensor(refs), torch.tensor(granted), torch.tensor(copies), pool.double()


# ---------------------------------------------------------------------------------------------------
def work(case):
    size, kind = 4 if case["dtype"] == "f32" else 2, case["kind"]
    if kind == "rotary":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["d"] * size + case["tokens"] * 8, "flops": 3 * n * case["rotary"]}
    if kind == "append":
        new, _ = _lengths(case)
        n = sum(new) * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * (n + sum(new) * case["kv_heads"]) * case["d"] * size, "flops": 3 * n * case["rotary"]}
    if kind == "attend":
        new, past = _lengths(case)
        kept = sum(n + p for n, p in zip(new, past))
        seen = sum(n * p + (n * (n + 1) // 2 if case["causal"] else n * n) for n, p in zip(new, past))
        return {"bytes": 2 * size * case["d"] * (kept * case["kv_heads"] + sum(new) * case["heads"]), "flops": 4 * case["d"] * case["heads"] * seen}
    page = size * case["planes"] * case["kv_heads"] * case["page"] * case["d"]
    if kind == "copy":
        return {"bytes": 2 * page * case["copies"], "flops": 0}
    _, past = _lengths(case)
    used = sum((p + case["page"] - 1) // case["page"] for p in past)
    if kind == "compact":  # of the pages in use, those behind the front, as pages lie by chance
        return {"bytes": 2 * page * used * (1 - used / case["pages"]) + 8 * used, "flops": 0}
    # a beam in three shares the page that it goes on in with others and copies it
    return {"bytes": 2 * page * (case["batch"] / 3) + 16 * used, "flops": 0}
