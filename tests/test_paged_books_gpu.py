"""The books of a pool of cache pages, over runs in which rows keep fewer tokens than they reserved, give tokens back, are refused and ask again: reference counts say how many
rows list a page at all times, and nothing is lost."""
import random

import pytest
import torch

import turbotransformers_b200 as tt
from turbotransformers_b200 import _capi
from turbotransformers_b200._cxx import cxx

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)
DEV = torch.device("cuda:0")


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def status():
    return cxx.device_status(0)


class Ledger:
    """Page tables kept by the rules of include/ttb.h, one row and one column after the other."""

    def __init__(self, B, width, pages, page):
        self.B, self.width, self.pages, self.page = B, width, pages, page
        self.lens, self.table, self.refs = [0] * B, [[-1] * width for _ in range(B)], [0] * pages

    def counted(self):
        refs = [0] * self.pages
        for p in (p for row in self.table for p in row if p >= 0):
            refs[p] += 1
        return refs

    def fork(self, parents):
        self.table = [list(self.table[p]) if p >= 0 else [-1] * self.width for p in parents]
        self.lens = [self.lens[p] if p >= 0 else 0 for p in parents]
        self.refs = self.counted()

    def reserve(self, new):
        before, free = list(self.refs), [p for p, r in enumerate(self.refs) if r == 0]
        granted, copies, stopped = [], [], False
        for b, n in enumerate(new):
            if n == 0:
                granted.append(1)
                continue
            have, want = -(-self.lens[b] // self.page), -(-(self.lens[b] + n) // self.page)
            if want > self.width:
                granted.append(0)
                continue
            begun = self.lens[b] % self.page != 0
            listed = lambda p: 0 <= p < self.pages and before[p] > 0  # noqa: E731
            takes = [c for c in range(have - begun, want) if not listed(self.table[b][c]) or self.refs[self.table[b][c]] > 1]
            stopped |= len(takes) > len(free)
            granted.append(0 if stopped else 1)
            if stopped:
                continue
            for c in takes:
                old, fresh = self.table[b][c], free.pop(0)
                if begun and c == have - 1:
                    copies.append([old, fresh])
                if listed(old):
                    self.refs[old] -= 1
                self.table[b][c] = fresh
                self.refs[fresh] = 1
        assert self.refs == self.counted()
        return granted, copies + [[-1, -1]] * (self.B - len(copies))

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        to = dict(zip([p for p in range(used, self.pages) if self.refs[p] > 0], [p for p in range(used) if self.refs[p] == 0]))
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        self.refs = self.counted()
        return used


def same(ledger, tensors):
    table, lens, refs = (x.tolist() for x in tensors)
    assert table == ledger.table and lens == ledger.lens and refs == ledger.refs


def test_rows_that_keep_fewer_tokens_than_they_reserved_lose_no_page():
    """15 tokens cached, 5 proposed three times and none kept, then the row is freed."""
    t = ints([[-1] * 4]), ints([0]), ints([0] * 6)
    tt.paged_reserve(*t, ints([15]), 16)
    t[1].fill_(15)
    for _ in range(3):
        granted, copies = tt.paged_reserve(*t, ints([5]), 16)
        assert granted.tolist() == [1] and copies.tolist() == [[-1, -1]]
        assert t[0].tolist() == [[0, 1, -1, -1]] and t[2].tolist() == [1, 1, 0, 0, 0, 0]
    tt.paged_fork(*t, ints([-1]))
    assert t[2].tolist() == [0] * 6 and status() == _capi.OK


def test_pages_reserved_and_then_shared_are_each_rows_own_when_written():
    """A row with pages in hand is forked: of the two that go on, the first gets its own in their place, the last keeps them."""
    ledger = Ledger(3, 5, 12, 16)
    t = ints(ledger.table), ints(ledger.lens), ints(ledger.refs)
    for new, keep, parents in (([40, 0, 0], [20, 0, 0], [0, 0, 0]), ([30, 30, 0], [1, 13, 0], [0, 1, 2]), ([0, 4, 60], [0, 0, 60], [-1, -1, -1])):
        granted, copies = tt.paged_reserve(*t, ints(new), 16)
        want, pairs = ledger.reserve(new)
        assert granted.tolist() == want == [1, 1, 1] and copies.tolist() == pairs
        same(ledger, t)
        t[1].add_(ints(keep))
        ledger.lens = [a + b for a, b in zip(ledger.lens, keep)]
        tt.paged_fork(*t, ints(parents))
        ledger.fork(parents)
        same(ledger, t)
    assert t[2].tolist() == [0] * 12 and status() == _capi.OK


@pytest.mark.parametrize("B,width,pages,page", [(1, 3, 4, 16), (3, 6, 14, 16), (9, 12, 70, 32), (40, 150, 900, 64), (200, 9, 5000, 256), (1024, 4, 1500, 16)])
def test_reserve_after_fewer_were_kept_and_after_tokens_were_given_back(B, width, pages, page):
    rng = random.Random(B * width + pages)
    ledger = Ledger(B, width, pages, page)
    t = ints(ledger.table).view(B, width), ints(ledger.lens), ints(ledger.refs)
    most = width * page
    for step in range(16):
        new = [rng.choice([0, 1, 5, rng.randint(1, 2 * page), rng.randint(1, most)]) for _ in range(B)]
        granted, copies = tt.paged_reserve(*t, ints(new), page)
        want, pairs = ledger.reserve(new)
        assert granted.tolist() == want and copies.tolist() == pairs
        same(ledger, t)
        keep = [g * rng.choice([n, n, rng.randint(0, n), 0]) for n, g in zip(new, want)]
        lens = [x + k for x, k in zip(ledger.lens, keep)]
        ledger.lens = [rng.choice([x, x, x, rng.randint(0, x)]) for x in lens]  # some tokens are given back
        t[1].copy_(ints(ledger.lens))
        if step % 3 == 1:
            parents = [rng.choice([-1, b, b, b, rng.randrange(B)]) for b in range(B)]
            tt.paged_fork(*t, ints(parents))
            ledger.fork(parents)
            same(ledger, t)
        if step % 5 == 4:
            used = ledger.compact()
            assert tt.paged_compact(t[0], t[2], torch.zeros(1, pages, 4, device=DEV)).tolist() == [used]
            same(ledger, t)
    tt.paged_fork(*t, ints([-1] * B))
    assert (t[2] == 0).all() and (t[0] == -1).all() and status() == _capi.OK


def test_bad_rows_are_not_granted_and_left_alone():
    """Row by row: its last page outside the pool, -1 (begun, and full), a negative number of tokens, a negative length, lengths beyond the table; the good rows among them get theirs."""
    table = [[3, 9], [-1, -1], [-1, -1], [1, -1], [-1, -1], [2, 4], [2, 4], [-1, -1], [1, -1]]
    lens, new, refs = [20, 5, 16, 10, -4, 33, 2 ** 31 - 1, 0, 10], [1, 1, 1, -3, 0, 0, 1, 3, 8], [0, 2, 2, 1, 2, 0]
    t = ints(table), ints(lens), ints(refs)
    granted, copies = tt.paged_reserve(*t, ints(new), 16)
    assert status() == _capi.ERR_BAD_INDEX
    assert granted.tolist() == [0, 0, 0, 0, 0, 0, 0, 1, 0]  # (the last row wants two pages, of which row 7 has left one: it is not bad)
    assert copies.tolist() == [[-1, -1]] * 9
    assert t[0].tolist() == table[:7] + [[0, -1]] + table[8:] and t[1].tolist() == lens and t[2].tolist() == [1, 2, 2, 1, 2, 0]
    for bad in ([-3], [-2 ** 31]):  # so that lens += new * granted never takes tokens away
        t = ints([[0, -1]]), ints([10]), ints([1, 0])
        assert tt.paged_reserve(*t, ints(bad), 16)[0].tolist() == [0] and status() == _capi.ERR_BAD_INDEX


def test_a_table_whose_pages_could_not_be_counted_is_refused(ctx):
    """Rows that want 2^31 pages together: refused before anything is launched (the table that is handed over here has two entries)."""
    table, lens, refs, new, granted = ints([[-1, -1]]), ints([0] * 1024), ints([0]), ints([0] * 1024), ints([0] * 1024)
    copies = ints([[0, 0]] * 1024)
    launches = _capi.lib().ttb_launch_count(ctx.h)
    for B, width, page in ((1024, 1 << 21, 16), (3, (1 << 30) - 1, 1), (33, 1 << 26, 16)):
        assert B * width >= 1 << 31
        tables = dict(table=table, stride=width, B=B, width=width, lens=lens, refs=refs, pages=1)
        with pytest.raises(_capi.TTBError):
            ctx.paged_reserve(tables, new, page, granted, copies)
    assert _capi.lib().ttb_launch_count(ctx.h) == launches


# ---------------------------------------------------------------------------------------------------
# rows that were not granted
# ---------------------------------------------------------------------------------------------------
def rows(g, n, heads, d, dtype):
    return torch.randn(n, heads, d, generator=g, device=DEV, dtype=dtype)


def cumulative(new):
    return ints([sum(new[:i]) for i in range(len(new) + 1)])


@pytest.mark.parametrize("new", [[1, 1, 1], [1, 0, 1], [3, 2, 1], [200, 7, 130], [4, 300, 0]])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_sequences_without_room_are_passed_over(new, d, dtype):
    """Nothing of them is filed, their rows of the outputs are as they were, the others get what they get without them; and no page or length of theirs is reported."""
    heads, kv, page, past = 4, 2, 16, [33, 20, 70]
    g = torch.Generator(DEV).manual_seed(sum(new) + d)
    table = ints([[b * 20 + c for c in range(20)] for b in range(3)])
    table[1] = 2 ** 30  # the row without room has no pages, and more tokens than the table lists
    lens, cu = ints(past), cumulative(new)
    lens[1] = 20 * page - 1
    pool = torch.randn(2, 60, kv, page, d, generator=g, device=DEV, dtype=dtype)
    room, freqs = ints([1, 0, 7]), 10.0 ** -torch.arange(d // 2, dtype=torch.float64, device=DEV)
    q, k, v = (rows(g, sum(new), h, d, dtype) for h in (heads, kv, kv))
    gone = slice(new[0], new[0] + new[1])
    q[gone] = k[gone] = v[gone] = float("nan")
    kept = [i for i in range(sum(new)) if not gone.start <= i < gone.stop]
    out, turned, mine = torch.full_like(q, 3.0), torch.full_like(q, 5.0), pool.clone()
    tt.paged_append(k, v, mine[0], mine[1], table, cu, lens, q=q, freqs=freqs, out=turned, room=room)
    tt.paged_attention(turned, mine[0], mine[1], table, cu, lens, out=out, room=room)
    assert status() == _capi.OK
    assert (turned[gone] == 5.0).all() and (out[gone] == 3.0).all()
    # the same call without them
    two, cu2 = [0, 2], cumulative([new[0], new[2]])
    want_q = tt.paged_append(k[kept], v[kept], pool[0], pool[1], table[two], cu2, lens[two], q=q[kept], freqs=freqs)
    want = tt.paged_attention(want_q, pool[0], pool[1], table[two], cu2, lens[two])
    assert status() == _capi.OK and torch.equal(mine, pool) and torch.equal(turned[kept], want_q)
    # dealt out otherwise: each may be off by half a step of itself and half a step of each probability, 2^-14 for everything in fp32
    u = torch.finfo(dtype).eps / 2
    off = 2 * (u * want.abs().max() + (u + 2.0 ** -14) * pool[1].abs().max()).item()
    assert (out[kept].double() - want.double()).abs().max() <= off


def test_refused_rows_of_a_full_pool_stay_as_they_are_and_go_on_later():
    """Two beams share a begun page and nothing is free: neither writes to it, their lengths and tables stay; when a third request ends they go on, each in a page of its own."""
    kv, d, page, dtype = 2, 64, 16, torch.float16
    cache = tt.PagedKVCache(1, 4, 4, 64, kv, d, page, dtype, DEV)
    g = torch.Generator(DEV).manual_seed(0)
    cache.pool.zero_()

    def play(new):
        granted = cache.reserve(new).tolist()
        k, v = rows(g, sum(new), kv, d, dtype), rows(g, sum(new), kv, d, dtype)
        cu = cumulative(new)
        cache.append(0, k, v, cu)
        out = cache.attend(0, rows(g, sum(new), kv, d, dtype), cu)
        cache.advance(new)
        return granted, out

    assert play([10, 0, 32, 0])[0] == [1] * 4
    cache.fork([0, 0, 2, 3])  # the pool: one page shared by two, two of the third, one free
    assert play([0, 0, 0, 5])[0] == [1] * 4
    before = [x.clone() for x in (cache.table, cache.lens, cache.refs, cache.pool)]
    assert cache.refs.tolist() == [2, 1, 1, 1]
    for new in ([1, 1, 0, 0], [1, 0, 0, 0], [0, 20, 0, 1], [1, 1, 64, 0]):
        granted, _ = play(new)
        assert granted == [int(n == 0) for n in new] and cache.room.tolist() == granted
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.table, cache.lens, cache.refs, cache.pool)))
    assert status() == _capi.OK
    cache.release([2])
    granted, out = play([1, 1, 0, 3])
    assert granted == [1] * 4 and cache.lens.tolist() == [11, 11, 0, 8] and status() == _capi.OK and out.isfinite().all()
    assert cache.refs.tolist() == [1, 1, 0, 1] and cache.table[:, 0].tolist() == [1, 0, -1, 3]
    assert torch.equal(cache.pool[:, 1, :, :10], before[3][:, 0, :, :10]) and torch.equal(cache.pool[:, 0, :, :10], before[3][:, 0, :, :10])
    cache.release(range(4))
    assert (cache.refs == 0).all() and (cache.lens == 0).all()


def test_a_captured_step_goes_by_what_is_granted_when_it_is_replayed():
    """A pool that fills up while a captured step is replayed: the rows stop in their order and go on after one of them is freed, as in the eager run beside it."""
    B, kv, d, page, dtype = 4, 2, 64, 16, torch.bfloat16
    g = torch.Generator(DEV).manual_seed(3)
    q, k, v = (rows(g, B, kv, d, dtype) for _ in range(3))
    cu, ones = cumulative([1] * B), ints([1] * B)

    def step(c, out):
        c.reserve(ones)
        c.append(0, k, v, cu)
        c.attend(0, q, cu, out=out)
        c.advance(ones)

    eager, captured = (tt.PagedKVCache(1, 6, B, 160, kv, d, page, dtype, DEV) for _ in range(2))
    for c in (eager, captured):
        c.pool.zero_()
    outs = [torch.zeros_like(q) for _ in range(2)]
    step(tt.PagedKVCache(1, 6, B, 160, kv, d, page, dtype, DEV), torch.zeros_like(q))  # (a first run loads the kernels, which a capture should not)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    cxx.arena_begin(0, 64 << 20)
    with torch.cuda.graph(graph, stream=side):
        step(captured, outs[1])
    arena = cxx.arena_end(0)[1]
    cxx.set_stream(0, torch.cuda.current_stream().cuda_stream)
    seen = set()
    for i in range(60):
        step(eager, outs[0])
        graph.replay()
        if i == 45:
            for c in (eager, captured):
                c.release([1])
        torch.cuda.synchronize()
        seen.add(tuple(eager.room.tolist()))
        for a, b in zip((eager.table, eager.lens, eager.refs, eager.room, outs[0]), (captured.table, captured.lens, captured.refs, captured.room, outs[1])):
            assert torch.equal(a, b)
    assert (1, 1, 1, 1) in seen and (1, 1, 0, 0) in seen and (0, 0, 0, 0) in seen and status() == _capi.OK
    del graph
    cxx.arena_release(0, arena)


def test_room_through_the_c_interface(ctx):
    """A step of three sequences of which the pool has room for the first: the same entry points with room, without it all rows as before."""
    kv_heads, d, page, dtype = 2, 64, 16, torch.float16
    g = torch.Generator(DEV).manual_seed(8)
    table, lens, refs = ints([[2, -1], [0, -1], [3, -1]]), ints([16, 16, 3]), ints([1, 0, 1, 1])
    granted, room, copies, new = ints([7] * 3), ints([7] * 3), ints([[7, 7]] * 3), ints([1, 1, 1])
    ctx.paged_reserve(dict(table=table, stride=2, B=3, width=2, lens=lens, refs=refs, pages=4), new, page, granted, copies, room=room)
    assert granted.tolist() == room.tolist() == [1, 0, 0] and table.tolist() == [[2, 1], [0, -1], [3, -1]]
    pool = torch.randn(2, 4, kv_heads, page, d, generator=g, device=DEV, dtype=dtype)
    q, k, v = (rows(g, 3, kv_heads, d, dtype) for _ in range(3))
    kv = dict(keys=pool[0], values=pool[1], page_stride=pool.stride(1), pages=4, kv_heads=kv_heads, page_tokens=page, d=d, table=table, table_stride=2, table_width=2,
              cu_seqlens=ints([0, 1, 2, 3]), past_lens=lens, B=3)
    want, out = pool.clone(), torch.full_like(q, 3.0)
    ctx.paged_append(_capi.F16, kv, 3, k, 128, v, 128, room=room)
    want[0, 1, :, 0], want[1, 1, :, 0] = k[0], v[0]
    assert torch.equal(pool, want)
    ctx.paged_attention(_capi.F16, kv, q, 128, 3, kv_heads, 1, 0.125, out, 128, room=room)
    assert ctx.device_status() == _capi.OK and (out[1:] == 3.0).all()
    everything = torch.empty_like(q)
    ctx.paged_attention(_capi.F16, {**kv, "table": ints([[2, 1], [0, 0], [3, 3]])}, q, 128, 3, kv_heads, 1, 0.125, everything, 128)
    assert ctx.device_status() == _capi.OK and everything.isfinite().all()
    # dealt out otherwise: each may be off by half a step of itself and half a step of each probability, 2^-14 for everything in fp32
    u = torch.finfo(dtype).eps / 2
    assert (everything[0].double() - out[0].double()).abs().max() <= 2 * (u * out[0].abs().max() + (u + 2.0 ** -14) * pool[1].abs().max()).item()
