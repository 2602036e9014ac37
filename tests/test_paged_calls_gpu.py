"""Calls of the operators over cache pages that are refused, or taken, beside those of test_paged_gpu."""
import pytest
import torch

import turbotransformers_b200 as tt
from turbotransformers_b200 import _capi
from turbotransformers_b200._cxx import cxx

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)
DEV = torch.device("cuda:0")


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEV)


@pytest.fixture
def pool():
    """(keys, values, table, cu_seqlens, past_lens) of one sequence of one new token behind 10, heads of 64, and q of 4 heads over k, v of 2."""
    both = torch.randn(2, 3, 2, 16, 64, device=DEV, dtype=torch.float16)
    return (both[0], both[1], ints([[2, -1]]), ints([0, 1]), ints([10])), torch.randn(1, 4, 64, device=DEV, dtype=torch.float16)


def test_rotary_positions_without_frequencies_are_refused(pool):
    """(The address of an empty tensor is null, which is how the runtime is told that nothing is to be turned.)"""
    args, q = pool
    k, none, before = q[:, :2], torch.empty(0, dtype=torch.float64, device=DEV), args[0].clone()
    with pytest.raises(ValueError):
        tt.paged_append(k, k, *args, q=q, freqs=none)
    with pytest.raises(ValueError):
        tt.paged_append(k, k, *args, freqs=none)
    with pytest.raises(ValueError):
        tt.rotary(q, k, torch.zeros(1, dtype=torch.int64, device=DEV), none)
    assert torch.equal(args[0], before) and cxx.device_status(0) == _capi.OK


def attended(q, k, v, past, causal):
    """Attention of q [n, heads, d] over k, v [past + n, key heads, d] in 64 bits, and how far off a kernel's may be: half a step of the output, half a step of every probability
    (fp16: 2^-25 of the largest at least), 2^-14 for what is fp32."""
    n, heads, d = q.shape
    u = torch.finfo(q.dtype).eps / 2
    k, v = (x.double().repeat_interleave(heads // k.shape[1], 1) for x in (k, v))
    s = torch.einsum("ihd,jhd->hij", q.double(), k) * d ** -0.5
    if causal:
        s.masked_fill_(torch.arange(past + n, device=DEV) > past + torch.arange(n, device=DEV)[:, None], -float("inf"))
    w = (s - s.amax(-1, keepdim=True)).exp()
    total = w.sum(-1, keepdim=True)
    want, mean = (torch.einsum("hij,jhd->ihd", w / total, x) for x in (v, v.abs()))
    off = u * want.abs() + (u + 2.0 ** -14) * mean
    if q.dtype == torch.float16:
        off += 2.0 ** -25 * torch.einsum("hij,jhd->ihd", (s > -float("inf")).double() / total, v.abs())
    return want, off


@pytest.mark.parametrize("new", [1, 200])
def test_pools_beyond_32_bits(new):
    """Pages 2^24 elements apart, so that the last lie 5 * 10^9 elements behind the first: filed, read and copied where they are."""
    pages, kv, heads, page, d, past = 300, 2, 4, 16, 64, 20
    g = torch.Generator(DEV).manual_seed(new)
    wide = torch.empty(pages, 1 << 24, device=DEV, dtype=torch.float16)
    size = kv * page * d
    keys, values = (wide[:, at:at + size].view(pages, kv, page, d) for at in (64, (1 << 24) - size))
    keys.zero_(), values.zero_()
    n, rows = past + new, -(-(past + new) // page)
    table = torch.tensor([[pages - 1 - 3 * c for c in range(rows)]], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(n, kv, d, generator=g, device=DEV, dtype=torch.float16) for _ in range(2))
    q = torch.randn(new, heads, d, generator=g, device=DEV, dtype=torch.float16)
    tt.paged_append(k[:past], v[:past], keys, values, table, ints([0, past]), ints([0]))
    tt.paged_append(k[past:], v[past:], keys, values, table, ints([0, new]), ints([past]))
    at = torch.arange(n, device=DEV)
    held = table[0].long()[at // page]
    assert torch.equal(keys[held, :, at % page], k) and torch.equal(values[held, :, at % page], v)
    got = tt.paged_attention(q, keys, values, table, ints([0, new]), ints([past]))
    want, off = attended(q, k, v, past, True)
    assert ((got.double() - want).abs() <= off).all()
    tt.paged_copy(wide[None, :, 64:64 + size], ints([[pages - 1, 1], [pages - 4, 0]]))
    assert torch.equal(keys[1], keys[pages - 1]) and torch.equal(keys[0], keys[pages - 4]) and (values[:2] == 0).all()
    assert cxx.device_status(0) == _capi.OK


@pytest.mark.parametrize("new", [[1] * 6, [2, 0, 40, 1, 200, 0]])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_over_pages_that_rows_share(new, causal):
    """Beams: the same first pages in every row, a last one of each row's own; lengths that end in a page that others go on in."""
    page, kv, heads, d, dtype = 32, 2, 8, 128, torch.bfloat16
    g = torch.Generator(DEV).manual_seed(sum(new))
    shared = torch.randperm(40, generator=g, device=DEV)[:12].tolist()
    table, past, next_page = [], [380, 300, 383, 0, 384, 130], 40
    for b, n in enumerate(new):
        full, last = past[b] // page, -(-(past[b] + n) // page)
        table.append(shared[:full] + list(range(next_page, next_page + last - full)) + [-1] * (20 - last))
        next_page += last - full
    pool = torch.randn(2, next_page, kv, page, d, generator=g, device=DEV, dtype=dtype)
    q = torch.randn(sum(new), heads, d, generator=g, device=DEV, dtype=dtype)
    cu = ints([sum(new[:b]) for b in range(len(new) + 1)])
    got, t = tt.paged_attention(q, pool[0], pool[1], ints(table), cu, ints(past), causal=causal), 0
    for b, n in enumerate(new):
        at = torch.arange(past[b] + n, device=DEV)
        held = torch.tensor(table[b], device=DEV)[at // page]
        want, off = attended(q[t:t + n], pool[0][held, :, at % page], pool[1][held, :, at % page], past[b], causal)
        assert ((got[t:t + n].double() - want).abs() <= off).all()
        t += n
    assert cxx.device_status(0) == _capi.OK


def test_advance_takes_what_can_be_added_to_the_lengths():
    for counts, want in (([1, 2, 3], [1, 0, 3]), (ints([1, 2, 3]), [1, 0, 3]), (torch.tensor([1, 2, 3], device=DEV), [1, 0, 3]), (4, [4, 0, 4]), (torch.tensor(2), [2, 0, 2]),
                         (torch.tensor([True, True, False], device=DEV), [1, 0, 0]), (ints([-0]), [0, 0, 0])):
        cache = tt.PagedKVCache(1, 4, 3, 64, 2, 64, device=DEV)
        cache.room[1] = 0
        cache.advance(counts)
        assert cache.lens.tolist() == want and cache.lens.dtype == torch.int32


def test_a_step_captured_without_an_arena():
    """Workspaces that the graph allocates and frees by itself: replays beside the eager run, a second graph of the same step alive."""
    B, dtype = 3, torch.float16
    q, k, v = (torch.randn(B, 2, 64, device=DEV, dtype=dtype) for _ in range(3))
    cu, ones = ints(range(B + 1)), ints([1] * B)

    def step(c, out):
        c.reserve(ones)
        c.append(0, k, v, cu)
        c.attend(0, q, cu, out=out)
        c.advance(ones)

    caches, outs, graphs = [tt.PagedKVCache(1, 30, B, 160, 2, 64, 16, dtype, DEV) for _ in range(3)], [torch.zeros_like(q) for _ in range(3)], []
    step(tt.PagedKVCache(1, 30, B, 160, 2, 64, 16, dtype, DEV), torch.zeros_like(q))  # (a first run loads the kernels)
    torch.cuda.synchronize()
    for c, out in list(zip(caches, outs))[1:]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step(c, out)
    cxx.set_stream(0, torch.cuda.current_stream().cuda_stream)
    for _ in range(40):
        step(caches[0], outs[0])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for c, out in zip(caches[1:], outs[1:]):
            assert torch.equal(outs[0], out) and torch.equal(caches[0].lens, c.lens) and torch.equal(caches[0].table, c.table)
    assert cxx.device_status(0) == _capi.OK
