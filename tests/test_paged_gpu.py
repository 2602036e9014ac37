"""Serving over a pool of cache pages: rotary positions, appending, attention and page maintenance against plain implementations in 64 bits.

Tolerances. A stored value is off by at most u = eps / 2 of itself, or by half the step between subnormal numbers (fp16: 2^-25) where that is more: a value below
2^-14, the smallest normal one, has fewer bits, so that u of itself is less than half a step. A rotated element is a sum of two products: beside u, each of its two terms carries the sine's or
cosine's error (fp32, below 2^-21 with the angle's own rounding) and two fp32 roundings. An attention output is rounded once (u |out|); its probabilities are rounded
to 16 bits before they are multiplied with the values (u of each, u * mean |v| under the same weights; in fp16 a probability below 2^-14 of the largest is off by
2^-25 of it instead); exponents (2^-22), fp32 sums and the scores' own rounding together stay below 2^-14 of mean |v| for scores up to some tens.
"""
import random

import pytest
import torch

import turbotransformers_b200 as tt
from turbotransformers_b200 import _capi
from turbotransformers_b200._cxx import cxx

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)
DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def stored(want, dtype):
    """How far rounding to dtype may take a value."""
    return (unit(dtype) * want.abs()).clamp(min=torch.finfo(dtype).smallest_normal * unit(dtype))


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def cumulative(new):
    return ints([sum(new[:i]) for i in range(len(new) + 1)])


def turned(x, positions, freqs, interleaved, scale):
    """(the rotation in 64 bits, how far off a kernel's may be)."""
    x, n = x.double(), freqs.numel()
    angle = positions.double()[:, None, None] * freqs
    want, most = x.clone(), x.abs().clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    want[..., first], want[..., second] = scale * (a * angle.cos() - b * angle.sin()), scale * (b * angle.cos() + a * angle.sin())
    most[..., first] = most[..., second] = scale * (a.abs() + b.abs())
    return want, most * 2.0 ** -20


def status():
    return cxx.device_status(0)


# ---------------------------------------------------------------------------------------------------
# rotary
# ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,heads,kv,d,dim,interleaved", [
    (1, 4, 2, 64, 64, False), (1, 1, 1, 8, 2, True), (5, 3, 1, 128, 128, True), (33, 12, 12, 64, 32, False), (700, 8, 2, 128, 64, True),
    (3, 2, 2, 72, 20, False), (3, 2, 2, 72, 20, True), (2, 2, 1, 512, 512, False), (9, 5, 5, 96, 24, True), (9, 5, 5, 96, 48, False),
    (5001, 3, 2, 24, 16, False), (4800, 1, 0, 16, 16, False), (2500, 7, 1, 40, 6, True), (1300, 5, 3, 64, 64, False), (2, 2000, 1000, 128, 128, False),
    (7203, 21, 11, 64, 32, True), (7301, 30, 2, 128, 128, False), (8001, 2, 126, 32, 32, False), (7600, 33, 0, 64, 64, True)])
def test_rotary(dt, T, heads, kv, d, dim, interleaved):
    g, dtype = gen(T + d + dim), DT[dt]
    q, k = randn(g, T, heads, d, dtype=dtype), randn(g, T, kv, d, dtype=dtype)
    positions = torch.randint(0, 2000000, (T,), generator=g, device=DEV)
    freqs = 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64, device=DEV) / (dim // 2))
    got = tt.rotary(q, k, positions, freqs, interleaved=interleaved, scale=1.25)
    for x, y in zip((q, k), got):
        want, off = turned(x, positions, freqs, interleaved, 1.25)
        assert ((y.double() - want).abs() <= off + stored(want, dtype)).all()
        assert torch.equal(y[..., dim:], x[..., dim:])


@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_rotary_in_place_in_packed_rows_of_any_stride(dt):
    g, T, heads, kv, d, dtype = gen(3), 50, 6, 2, 64, DT[dt]
    freqs = 10000.0 ** (-torch.arange(16, dtype=torch.float64, device=DEV) / 16)
    positions = torch.arange(T, device=DEV)
    for extra, shift in ((0, 0), (8, 0), (3, 0), (8, 1)):  # the last two are on no 16-byte boundary
        rows = randn(g, T, (heads + 2 * kv) * d + extra + shift, dtype=dtype)
        before = rows.clone()
        q, k = rows[:, shift:shift + heads * d].view(T, heads, d), rows[:, shift + heads * d:shift + (heads + kv) * d].view(T, kv, d)
        wants = [turned(x.clone(), positions, freqs, False, 1.0) for x in (q, k)]
        tt.rotary(q, k, positions, freqs, out=(q, k))
        for x, (want, off) in zip((q, k), wants):
            assert ((x.double() - want).abs() <= off + stored(want, dtype)).all()
        assert torch.equal(rows[:, shift + (heads + kv) * d:], before[:, shift + (heads + kv) * d:]) and torch.equal(rows[:, :shift], before[:, :shift])
    alone, none = tt.rotary(q, None, positions, freqs)
    assert none is None and alone.shape == q.shape
    assert tt.rotary(q[:0], k[:0], positions[:0], freqs)[0].shape == (0, heads, d)


def test_rotary_turns_back():
    """A turn by the opposite frequencies undoes it, whatever the position."""
    g = gen(1)
    q, freqs = randn(g, 40, 4, 64, dtype=torch.float32), 3.0 ** -torch.arange(32, dtype=torch.float64, device=DEV)
    positions = torch.randint(0, 1 << 40, (40,), generator=g, device=DEV) >> 9
    back = tt.rotary(tt.rotary(q, None, positions, freqs)[0], None, positions, -freqs)[0]
    assert (back - q).abs().max() < 2 ** -18  # two turns, each 2^-20 of |a| + |b| < 8 at most: rms far below


def test_rotary_embedding_stretches():
    base = tt.RotaryEmbedding(64, device=DEV)
    assert torch.allclose(base.freqs, 10000.0 ** (-torch.arange(32, dtype=torch.float64, device=DEV) / 32), rtol=1e-14) and base.scale == 1.0
    assert torch.equal(tt.RotaryEmbedding(64, stretch="linear", factor=4.0, device=DEV).freqs, base.freqs / 4)
    ntk = tt.RotaryEmbedding(64, stretch="ntk", factor=4.0, device=DEV).freqs
    assert torch.allclose(ntk[[0, -1]], torch.stack((base.freqs[0], base.freqs[-1] / 4)), rtol=1e-12)
    yarn = tt.RotaryEmbedding(64, stretch="yarn", factor=4.0, trained=4096, device=DEV)
    ratio = base.freqs / yarn.freqs
    assert abs(yarn.scale - 1.1386294361) < 1e-9 and ratio[0] == 1 and abs(ratio[-1] - 4) < 1e-9 and (ratio.diff() >= -1e-12).all()
    g = gen(2)
    q, positions = randn(g, 7, 2, 64, dtype=torch.float32), torch.arange(7, device=DEV)
    want, off = turned(q, positions, yarn.freqs, False, yarn.scale)
    assert ((yarn(q, None, positions)[0].double() - want).abs() <= off + stored(want, torch.float32)).all()


# ---------------------------------------------------------------------------------------------------
# a pool with ragged sequences
# ---------------------------------------------------------------------------------------------------
class Pool:
    """Sequences over scattered pages. What belongs to no token is NaN; unused table entries are nonsense."""

    def __init__(self, seed, dtype, past, new, kv, d, page, together=False, stray=5):
        self.past, self.new, self.page = list(past), list(new), page
        g = self.g = gen(seed)
        counts = [-(-(p + n) // page) for p, n in zip(past, new)]
        pages, width = sum(counts) + 2, max(counts + [1]) + 1
        both = torch.full((pages, 2, kv, page, d), float("nan"), dtype=dtype, device=DEV)
        if not together:
            both = both.transpose(0, 1).contiguous().transpose(0, 1)
        self.keys, self.values = both[:, 0], both[:, 1]
        order = torch.randperm(pages, generator=g, device=DEV).tolist()
        self.rows, at = [], 0
        for c in counts:
            self.rows.append(order[at:at + c] + [2 ** 30] * (width - c))
            at += c
        self.table = ints(self.rows).view(len(past), width)
        self.cu, self.past_lens = cumulative(new), ints(self.past).view(len(past))
        for b, p in enumerate(past):
            self.fill(b, 0, randn(g, p, kv, d, dtype=dtype), randn(g, p, kv, d, dtype=dtype))

    def fill(self, b, start, k, v):
        for j in range(start, start + k.shape[0]):
            page, slot = self.rows[b][j // self.page], j % self.page
            self.keys[page, :, slot], self.values[page, :, slot] = k[j - start], v[j - start]

    def held(self, b, n):
        """Keys and values of sequence b's first n tokens, [n, kv, d]."""
        at = torch.arange(n, device=DEV)
        page = self.table[b].long()[at // self.page]
        return self.keys[page, :, at % self.page], self.values[page, :, at % self.page]

    def fill_new(self, dtype, kv, d):
        for b, n in enumerate(self.new):
            self.fill(b, self.past[b], randn(self.g, n, kv, d, dtype=dtype), randn(self.g, n, kv, d, dtype=dtype))

    def args(self):
        return self.keys, self.values, self.table, self.cu, self.past_lens


def attended(q, pool, causal, scale):
    """(attention in 64 bits, how far off a kernel's may be), rows as q's."""
    want, off = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    u, t = unit(q.dtype), 0
    for b, (p, n) in enumerate(zip(pool.past, pool.new)):
        if n == 0:
            continue
        k, v = (x.double() for x in pool.held(b, p + n))
        group = q.shape[1] // k.shape[1]
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        s = torch.einsum("ihd,jhd->hij", q[t:t + n].double(), k) * scale
        if causal:
            s.masked_fill_(torch.arange(p + n, device=DEV) > p + torch.arange(n, device=DEV)[:, None], -float("inf"))
        w = (s - s.amax(-1, keepdim=True)).exp()
        total = w.sum(-1, keepdim=True)
        mean = torch.einsum("hij,jhd->ihd", w / total, v.abs())
        want[t:t + n] = torch.einsum("hij,jhd->ihd", w / total, v)
        off[t:t + n] = u * want[t:t + n].abs() + (u + 2.0 ** -14) * mean
        if q.dtype == torch.float16:
            off[t:t + n] += 2.0 ** -25 * torch.einsum("hij,jhd->ihd", (s > -float("inf")).double() / total, v.abs())
        t += n
    return want, off


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page,past,new,heads,kv,d,dim,interleaved,together", [
    (16, [0], [1], 4, 2, 64, 64, False, False), (16, [15, 16, 0, 31], [1, 1, 0, 2], 4, 1, 128, 64, True, False), (64, [0, 100], [130, 65], 6, 6, 64, 64, False, True),
    (256, [255, 1], [3, 300], 8, 2, 128, 128, True, False), (32, [7] * 200, [1] * 200, 2, 2, 64, 16, False, True), (128, [0, 0, 5], [0, 7, 0], 3, 3, 64, 20, True, False),
    (64, [0, 100, 5], [3000, 4300, 1], 16, 8, 64, 32, True, False), (16, [7, 0, 0, 130], [1500, 0, 4000, 1800], 15, 9, 128, 128, False, True)])
def test_append(dt, page, past, new, heads, kv, d, dim, interleaved, together):
    dtype = DT[dt]
    pool = Pool(sum(new) + page, dtype, past, new, kv, d, page, together)
    T, g = sum(new) + 3, pool.g  # three rows behind the last sequence
    rows = randn(g, T, (heads + 2 * kv) * d, dtype=dtype)
    q, k, v = rows[:, :heads * d].view(T, heads, d), rows[:, heads * d:(heads + kv) * d].view(T, kv, d), rows[:, (heads + kv) * d:].view(T, kv, d)
    freqs = 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64, device=DEV) / (dim // 2))
    before = [x.clone() for x in (pool.keys, pool.values)]
    out = torch.full((T, heads, d), 7.0, dtype=dtype, device=DEV)
    got = tt.paged_append(k, v, *pool.args(), q=q, freqs=freqs, interleaved=interleaved, scale=0.75, out=out)
    assert got is out and status() == _capi.OK
    position = torch.tensor([p + i for p, n in zip(past, new) for i in range(n)], device=DEV, dtype=torch.int64)
    wq, oq = turned(q[:sum(new)], position, freqs, interleaved, 0.75)
    wk, ok = turned(k[:sum(new)], position, freqs, interleaved, 0.75)
    assert ((out[:sum(new)].double() - wq).abs() <= oq + stored(wq, dtype)).all() and (out[sum(new):] == 7.0).all()
    t = 0
    for b, (p, n) in enumerate(zip(past, new)):
        hk, hv = pool.held(b, p + n)
        assert ((hk[p:].double() - wk[t:t + n]).abs() <= ok[t:t + n] + stored(wk[t:t + n], dtype)).all() and torch.equal(hv[p:], v[t:t + n])
        t += n
    # without frequencies: the rows as they are. Everything else in the pool is as it was.
    assert tt.paged_append(k, v, *pool.args()) is None
    pool.keys, pool.values, had = pool.keys.clone(), pool.values.clone(), before
    t = 0
    for b, (p, n) in enumerate(zip(past, new)):
        hk, hv = pool.held(b, p + n)
        assert torch.equal(hk[p:], k[t:t + n]) and torch.equal(hv[p:], v[t:t + n])
        for j in range(p, p + n):
            at = pool.rows[b][j // page], slice(None), j % page
            pool.keys[at], pool.values[at] = had[0][at], had[1][at]
        t += n
    assert torch.equal(pool.keys.nan_to_num(9.0), had[0].nan_to_num(9.0)) and torch.equal(pool.values.nan_to_num(9.0), had[1].nan_to_num(9.0))


ATTEND = [
    # page, past, new, heads, kv heads, head size, causal
    (16, [0], [1], 1, 1, 64, True), (16, [0], [1], 4, 1, 128, True), (16, [15], [1], 2, 2, 128, True), (16, [16], [1], 2, 2, 128, True),
    (16, [127, 128, 0, 129, 0, 500], [1, 1, 1, 1, 0, 1], 12, 12, 64, True), (32, [31, 32, 33, 1000], [1, 1, 1, 1], 32, 8, 128, True),
    (64, [3000], [1], 8, 1, 64, True), (16, [5000], [1], 16, 2, 128, True), (16, [9000], [1], 4, 4, 64, True), (256, [700, 3], [1, 2], 40, 2, 64, True),
    (128, [100, 0, 50], [5, 3, 1], 64, 8, 128, True), (16, [1000, 2000], [6, 4], 7, 1, 128, True), (16, [0, 10], [17, 40], 6, 6, 64, True),
    (64, [0, 200, 0], [300, 129, 64], 4, 2, 128, True), (16, [0], [257], 3, 1, 64, True), (16, [130], [128], 2, 2, 64, True), (32, [64], [900], 10, 5, 64, True),
    (16, [33, 0], [20, 200], 8, 8, 128, False), (16, [500], [1], 4, 4, 64, False), (64, [0, 70], [130, 1], 24, 2, 128, False), (16, [100], [2], 150, 1, 64, True),
    (16, [40], [130], 150, 1, 128, True), (16, [3] * 300, [1] * 300, 2, 1, 64, True), (16, [2, 300] * 12, [100, 1] * 12, 8, 2, 128, True),
    (256, [0, 1000], [1500, 700], 2, 1, 128, True), (16, [20000], [140], 4, 2, 64, True), (16, [6000], [300], 4, 1, 128, True),
]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page,past,new,heads,kv,d,causal", ATTEND)
def test_attention(dt, page, past, new, heads, kv, d, causal):
    dtype = DT[dt]
    pool = Pool(sum(past) + heads, dtype, past, new, kv, d, page, together=heads % 3 == 0)
    pool.fill_new(dtype, kv, d)
    T = sum(new) + 2
    rows = randn(pool.g, T, (heads + 2) * d, dtype=dtype)
    rows[sum(new):] = float("nan")  # rows that belong to no sequence
    q = rows[:, d:(heads + 1) * d].view(T, heads, d)
    out = torch.full((T, heads + 1, d), 5.0, dtype=dtype, device=DEV)
    got = tt.paged_attention(q, *pool.args(), causal=causal, scale=0.2, out=out[:, :heads])
    assert status() == _capi.OK
    want, off = attended(q[:sum(new)], pool, causal, 0.2)
    far = (got[:sum(new)].double() - want).abs()
    assert (far <= off).all(), f"{(far / off).max().item():.3g} times the tolerance"
    assert (out[sum(new):] == 5.0).all() and (out[:, heads] == 5.0).all()
    again = tt.paged_attention(q, *pool.args(), causal=causal, scale=0.2)
    assert torch.equal(again[:sum(new)], got[:sum(new)])  # the same on every run


# No more tokens than sequences: tiles of 8, 16 and 32 rows, and heads that need more, for all of them; then one sequence of a tile's rows, or some more.
STEPS = [
    # page, past, new, heads, kv heads, head size, causal
    (16, [0, 1, 127, 128, 700], [1, 1, 1, 1, 1], 5, 1, 64, True), (16, [40, 3000, 0], [1, 1, 1], 9, 1, 128, True), (32, [127, 0, 1300], [1, 1, 1], 32, 2, 64, True),
    (16, [2000, 15, 16], [1, 1, 1], 16, 1, 128, False), (64, [129, 0, 5000], [1, 1, 1], 17, 1, 64, True), (16, [31, 6000], [1, 1], 64, 2, 128, True),
    (16, [255, 10], [1, 1], 32, 1, 64, False), (16, [300, 0, 77], [1, 1, 1], 33, 1, 64, True), (16, [90, 5, 300, 0, 0, 2], [0, 6, 0, 0, 0, 0], 24, 2, 64, True),
    (32, [90, 5, 300, 40], [1, 0, 3, 0], 40, 2, 128, True), (16, [10] * 40, [0] * 39 + [40], 4, 4, 64, True), (16, [7000], [7], 16, 1, 64, True), (16, [7000], [8], 32, 2, 64, False),
    (256, [4000], [2], 32, 2, 128, True), (16, [1000], [4], 4, 2, 128, True), (128, [999], [9], 4, 4, 64, True),
    (16, [1000, 3000], [3, 2], 7, 1, 128, True), (32, [700, 10, 0, 5000], [8, 6, 7, 7], 4, 1, 64, True), (16, [2000, 127, 129], [6, 1, 2], 16, 2, 128, False),
]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page,past,new,heads,kv,d,causal", STEPS)
def test_attention_of_a_step(dt, page, past, new, heads, kv, d, causal):
    dtype = DT[dt]
    pool = Pool(sum(past) + heads, dtype, past, new, kv, d, page)
    pool.fill_new(dtype, kv, d)
    q = randn(pool.g, sum(new), heads, d, dtype=dtype)
    got = tt.paged_attention(q, *pool.args(), causal=causal, scale=0.2)
    assert status() == _capi.OK
    want, off = attended(q, pool, causal, 0.2)
    far = (got.double() - want).abs()
    assert (far <= off).all(), f"{(far / off).max().item():.3g} times the tolerance"
    assert torch.equal(tt.paged_attention(q, *pool.args(), causal=causal, scale=0.2), got)


@pytest.mark.parametrize("heads", [8, 16, 32])
def test_attention_of_a_step_with_scores_far_apart(heads):
    """As below, for tiles of each number of rows, every row with a course of its own."""
    past, d = 1500, 64
    pool = Pool(4, torch.float16, [past, past], [1, 1], 1, d, 16)
    pool.fill_new(torch.float16, 1, d)
    for b in range(2):
        for j in range(past + 1):
            page, slot = pool.rows[b][j // 16], j % 16
            pool.keys[page, :, slot] = pool.keys[page, :, slot] * 0.01 + (j % 700) / 64.0 * (1 if j < 1100 else 0.3)
    q = torch.ones(2, heads, d, dtype=torch.float16, device=DEV) + randn(pool.g, 2, heads, d, dtype=torch.float16) * 0.01
    q *= (1 - torch.arange(heads, device=DEV) % 3 * 0.75)[:, None].half()  # rising, rising slowly, falling
    got = tt.paged_attention(q, *pool.args(), scale=1.0)
    want, off = attended(q, pool, True, 1.0)
    # scores of up to 700: their fp32 sums are off by 64 roundings of up to 700 * 2^-24 at most, 2^-9 in the exponent
    assert ((got.double() - want).abs() <= off + 2.0 ** -8 * want.abs().amax()).all()


@pytest.mark.parametrize("new", [1, 200])
def test_attention_with_scores_far_apart(new):
    """A running maximum that rises by hundreds from key to key, and falls again: nothing overflows, and only the largest counts."""
    past, heads, d = 1500, 2, 64
    pool = Pool(4, torch.float16, [past], [new], heads, d, 16)
    pool.fill_new(torch.float16, heads, d)
    for j in range(past + new):
        page, slot = pool.rows[0][j // 16], j % 16
        pool.keys[page, :, slot] = pool.keys[page, :, slot] * 0.01 + (j % 700) / 64.0 * (1 if j < 1100 else 0.3)
    q = torch.ones(new, heads, d, dtype=torch.float16, device=DEV) + randn(pool.g, new, heads, d, dtype=torch.float16) * 0.01
    got = tt.paged_attention(q, *pool.args(), scale=1.0)
    want, off = attended(q, pool, True, 1.0)
    # scores of up to 700: their fp32 sums are off by 64 roundings of up to 700 * 2^-24 at most, 2^-9 in the exponent
    assert ((got.double() - want).abs() <= off + 2.0 ** -8 * want.abs().amax()).all()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("page,past,new,heads,kv,d,causal", [
    (64, [0], [314], 12, 3, 64, True), (16, [616], [336], 33, 1, 128, False), (128, [0, 1054], [667, 20], 8, 2, 128, False), (16, [0, 4000], [1, 300], 40, 1, 64, True),
    (16, [300, 2000, 77], [1, 1, 1], 24, 1, 128, True)])
def test_attention_with_few_keys_that_count(page, past, new, heads, kv, d, causal, dt):
    """Scores spread by some 60: the reference is raised time and again, with no more than one rounding of a probability."""
    dtype, scale = DT[dt], 0.3
    pool = Pool(sum(new) + d, dtype, past, new, kv, d, page)
    pool.fill_new(dtype, kv, d)
    q = randn(pool.g, sum(new), heads, d, dtype=dtype) * 4
    got = tt.paged_attention(q, *pool.args(), causal=causal, scale=scale)
    assert status() == _capi.OK
    want, off = attended(q, pool, causal, scale)
    # A score is off by d / 16 + 1 roundings (of a step at most: the products are summed 16 at a time) of a sum that the moduli bound, and two roundings of the scaled one: a
    # probability by that much of itself, and their sum as well.
    t = 0
    for b, (p, n) in enumerate(zip(past, new)):
        k, v = (x.double().repeat_interleave(heads // kv, 1) for x in pool.held(b, p + n))
        most = torch.einsum("ihd,jhd->hij", q[t:t + n].double().abs(), k.abs()).amax() * scale
        score = torch.einsum("ihd,jhd->hij", q[t:t + n].double(), k) * scale
        if causal:
            score.masked_fill_(torch.arange(p + n, device=DEV) > p + torch.arange(n, device=DEV)[:, None], -float("inf"))
        off[t:t + n] += 2 * (d // 16 + 3) * 2.0 ** -23 * most * torch.einsum("hij,jhd->ihd", score.softmax(-1), v.abs())
        t += n
    far = (got.double() - want).abs()
    assert (far <= off).all(), f"{(far / off).max().item():.3g} times the tolerance"


def test_attention_of_nothing_and_of_padded_calls():
    pool = Pool(5, torch.float16, [10, 0, 4], [0, 0, 0], 2, 64, 16)
    q = torch.full((4, 2, 64), float("nan"), dtype=torch.float16, device=DEV)
    out = torch.full_like(q, 3.0)
    assert (tt.paged_attention(q, *pool.args(), out=out) == 3.0).all() and status() == _capi.OK
    assert tt.paged_attention(q[:0], *pool.args()).shape == (0, 2, 64)
    none = (pool.keys, pool.values, pool.table[:0], ints([0]), ints([]))
    assert (tt.paged_attention(q, *none, out=out) == 3.0).all()
    # rows before the first sequence and behind the last are left alone
    pool = Pool(6, torch.float16, [10, 20], [1, 1], 2, 64, 16)
    pool.fill_new(torch.float16, 2, 64)
    q = randn(pool.g, 5, 2, 64, dtype=torch.float16)
    pool.cu = pool.cu + 2
    out = torch.full_like(q, 3.0)
    tt.paged_attention(q, *pool.args(), out=out)
    want, off = attended(q[2:4], pool, True, 0.125)
    assert ((out[2:4].double() - want).abs() <= off).all() and (out[:2] == 3.0).all() and (out[4:] == 3.0).all()


@pytest.mark.parametrize("new", [1, 150])
def test_bad_pages_lengths_and_offsets_are_reported_and_never_used(new):
    """Kernels read and write inside the pool whatever the tables say (the arithmetic is checked on the CPU in test_paged_rules_cpu); other sequences are not touched."""
    pool = Pool(7, torch.float16, [100, 50, 60], [new, new, new], 2, 64, 16)
    pool.fill_new(torch.float16, 2, 64)
    q = randn(pool.g, 3 * new, 2, 64, dtype=torch.float16)
    want, off = attended(q, pool, True, 0.125)
    good = slice(new, 2 * new)
    keys, values = pool.keys.clone(), pool.values.clone()

    def check():
        got = tt.paged_attention(q, *pool.args())
        assert status() == _capi.ERR_BAD_INDEX
        assert ((got[good].double() - want[good]).abs() <= off[good]).all()
        tt.paged_append(q, q, *pool.args())
        assert status() == _capi.ERR_BAD_INDEX
        pool.keys.copy_(keys), pool.values.copy_(values)

    for bad in (-1, pool.keys.shape[0], 2 ** 31 - 1, -2 ** 31):
        table = pool.table.clone()
        pool.table[0, 0:20] = bad
        check()
        pool.table.copy_(table)
    for at, value in ((0, -5), (2, 2 ** 31 - 1), (2, 10 ** 6)):
        past = pool.past_lens.clone()
        pool.past_lens[at] = value
        check()
        pool.past_lens.copy_(past)
    for value in (10 ** 6, -3):
        cu = pool.cu.clone()
        pool.cu[3] = value
        check()
        pool.cu.copy_(cu)


# ---------------------------------------------------------------------------------------------------
# page maintenance
# ---------------------------------------------------------------------------------------------------
class Book:
    """Page tables kept by the rules, one row after the other."""

    def __init__(self, rng, B, width, pages, page, shared=True):
        self.page, self.B, self.width = page, B, width
        free = list(range(pages))
        rng.shuffle(free)
        self.lens, self.table = [], []
        for _ in range(B):
            n = rng.choice([0, rng.randint(1, width * page)])
            c = -(-n // page)
            if c > len(free):
                n = c = 0
            self.lens.append(n)
            self.table.append([free.pop() for _ in range(c)] + [-1] * (width - c))
        self.refs = [0] * pages
        self.count()
        if shared:
            self.fork([rng.choice([-1, b, rng.randrange(B), rng.randrange(B)]) for b in range(B)])

    def count(self):
        self.refs = [0] * len(self.refs)
        for p in (p for row in self.table for p in row if p >= 0):
            self.refs[p] += 1

    def fork(self, parents):
        self.table = [list(self.table[p]) if p >= 0 else [-1] * self.width for p in parents]
        self.lens = [self.lens[p] if p >= 0 else 0 for p in parents]
        self.count()

    def reserve(self, new):
        granted, copies, stopped = [], [], False
        free = [p for p, r in enumerate(self.refs) if r == 0]
        for b, n in enumerate(new):
            if n == 0:
                granted.append(1)
                continue
            if self.lens[b] + n > self.width * self.page:
                granted.append(0)
                continue
            have, want = -(-self.lens[b] // self.page), -(-(self.lens[b] + n) // self.page)
            last = self.table[b][have - 1]
            own = self.lens[b] % self.page != 0 and self.refs[last] > 1
            stopped |= want - have + own > len(free)
            granted.append(0 if stopped else 1)
            if stopped:
                continue
            if own:
                self.table[b][have - 1] = free.pop(0)
                copies.append([last, self.table[b][have - 1]])
                self.refs[last] -= 1
            for c in range(have, want):
                self.table[b][c] = free.pop(0)
            for c in range(have - own, want):
                self.refs[self.table[b][c]] += 1
        return granted, copies + [[-1, -1]] * (self.B - len(copies))

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if self.refs[p] == 0]
        to = dict(zip([p for p in range(used, len(self.refs)) if self.refs[p] > 0], holes))
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        self.count()
        return used, to

    def tensors(self):
        wide = torch.full((max(self.B, 1), self.width + 3), -7, dtype=torch.int32, device=DEV)
        table = wide[:self.B, :self.width]
        table.copy_(ints(self.table).view(self.B, self.width))
        return table, ints(self.lens).view(self.B), ints(self.refs)

    def same(self, table, lens, refs):
        return table.tolist() == self.table and lens.tolist() == self.lens and refs.tolist() == self.refs


@pytest.mark.parametrize("B,width,pages,page", [(1, 1, 1, 16), (1, 4, 3, 16), (3, 5, 20, 16), (8, 17, 60, 32), (40, 9, 200, 64), (100, 40, 5000, 16), (1024, 3, 1500, 256),
                                                (64, 300, 40000, 16)])
def test_reserve_fork_and_compact_follow_the_rules(B, width, pages, page):
    rng = random.Random(B * width + pages)
    for round_ in range(6):
        book = Book(rng, B, width, pages, page)
        t = book.tensors()
        for step in range(4):
            new = [rng.choice([0, 1, 1, rng.randint(1, 2 * page)]) for _ in range(B)]
            granted, copies = tt.paged_reserve(*t, ints(new).view(B), page)
            want, pairs = book.reserve(new)
            assert granted.tolist() == want and copies.tolist() == pairs and book.same(*t)
            t[1].add_(ints(new).view(B) * granted)
            book.lens = [n + a * g for n, a, g in zip(book.lens, new, want)]
            parents = [rng.choice([-1, b, b, b, rng.randrange(B)]) for b in range(B)]
            tt.paged_fork(*t, ints(parents).view(B))
            book.fork(parents)
            assert book.same(*t)
        pool = torch.arange(2 * pages * 8, device=DEV, dtype=torch.float32).view(2, pages, 8)
        before = pool.clone()
        used, to = book.compact()
        assert tt.paged_compact(t[0], t[2], pool).tolist() == [used] and book.same(*t)
        for a, b in to.items():
            before[:, b] = before[:, a]
        assert torch.equal(pool, before)
    assert status() == _capi.OK


def test_a_full_pool_grants_in_the_rows_order():
    book = Book(random.Random(0), 0, 4, 6, 16)
    book.B, book.lens, book.table = 5, [16, 20, 0, 8, 0], [[0, -1, -1, -1], [1, 2, -1, -1], [-1] * 4, [3, -1, -1, -1], [-1] * 4]
    book.count()
    t = book.tensors()
    new = [1, 44, 1, 8, 0]  # row 1 wants two pages where one is left; row 3 needs none, but comes behind it
    want, pairs = book.reserve(new)
    granted, copies = tt.paged_reserve(*t, ints(new), 16)
    assert want == [1, 0, 0, 0, 1] and granted.tolist() == want and copies.tolist() == pairs and book.same(*t)


def test_bad_entries_of_the_tables_are_reported():
    table, lens, refs = ints([[3, 9], [-1, -1]]), ints([20, 0]), ints([0, 0, 0, 1])
    tt.paged_fork(table, lens, refs, ints([0, 0]))
    assert status() == _capi.ERR_BAD_INDEX and refs.tolist() == [0, 0, 0, 2]
    tt.paged_fork(table, lens, refs, ints([5, -2]))
    assert status() == _capi.ERR_BAD_INDEX and table.tolist() == [[3, 9], [3, 9]] and lens.tolist() == [20, 20]
    granted, copies = tt.paged_reserve(table, ints([20, -4]), refs, ints([1, 1]), 16)
    assert status() == _capi.ERR_BAD_INDEX and granted.tolist()[1] == 0 and refs.tolist() == [0, 0, 0, 2]
    pool = torch.arange(8.0, device=DEV).view(1, 2, 4)
    tt.paged_copy(pool, ints([[0, 2], [7, 1], [-1, 0], [0, -5]]))
    assert status() == _capi.ERR_BAD_INDEX and torch.equal(pool, torch.arange(8.0, device=DEV).view(1, 2, 4))
    tt.paged_compact(table, ints([0, 0, 0, 2]), torch.zeros(1, 4, 4, device=DEV))
    assert status() == _capi.ERR_BAD_INDEX and table.tolist() == [[0, 9], [0, 9]]


@pytest.mark.parametrize("planes,pages,n,shape,dtype", [(1, 2, 1, (8,), torch.float16), (3, 50, 20, (2, 16, 64), torch.bfloat16), (5, 700, 300, (1, 16, 64), torch.float16),
                                                        (2, 9, 4, (8, 256, 128), torch.float16), (48, 6, 3, (4100,), torch.float32)])
def test_copy(planes, pages, n, shape, dtype):
    g = gen(pages)
    pool = randn(g, planes, pages, *shape, dtype=dtype)
    pairs = torch.randperm(pages, generator=g, device=DEV)[:2 * n].view(n, 2).to(torch.int32)
    if n > 2:
        pairs[1] = -1
    want = pool.clone()
    for a, b in pairs.tolist():
        if a >= 0:
            want[:, b] = want[:, a]
    tt.paged_copy(pool, pairs)
    assert torch.equal(pool, want) and status() == _capi.OK
    tt.paged_copy(pool, pairs[:0])
    # a pool whose planes and pages are parts of a wider one
    wide = randn(g, planes + 1, pages, 2, *shape, dtype=dtype)
    part, want = wide[1:, :, 1], wide.clone()
    for a, b in pairs.tolist():
        if a >= 0:
            want[1:, b, 1] = want[1:, a, 1]
    tt.paged_copy(part, pairs)
    assert torch.equal(wide, want)


# ---------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------
def play(cache, rotary, layers, heads, kv, d, steps, seed):
    """Prompts, steps and forks of a beam search over the cache; yields (sequence's history per layer, its queries, what came out)."""
    g, rng = gen(seed), random.Random(seed)
    B = cache.table.shape[0]
    history = [[(torch.empty(0, kv, d, device=DEV, dtype=cache.pool.dtype),) * 2 for _ in range(layers)] for _ in range(B)]
    for step in range(steps):
        new = [rng.choice([0, 1, 1, 3, 40 if step < 3 else 1]) for _ in range(B)]
        granted = cache.reserve(new)
        assert granted.tolist() == [1] * B
        T, cu = sum(new), cumulative(new)
        for layer in range(layers):
            q, k, v = (randn(g, T, h, d, dtype=cache.pool.dtype) for h in (heads, kv, kv))
            turned_q = cache.append(layer, k, v, cu, q=q, rotary=rotary)
            out = cache.attend(layer, turned_q, cu)
            t = 0
            for b, n in enumerate(new):
                hk, hv = history[b][layer]
                past = hk.shape[0]
                positions = torch.arange(past, past + n, device=DEV)
                kk = tt.rotary(k[t:t + n], None, positions, rotary.freqs, interleaved=rotary.interleaved, scale=rotary.scale)[0]
                history[b][layer] = torch.cat((hk, kk)), torch.cat((hv, v[t:t + n]))
                if n:
                    yield history[b][layer], turned_q[t:t + n], out[t:t + n]
                t += n
        cache.advance(new)
        parents = [rng.choice([b, b, rng.randrange(B), -1 if step % 3 == 2 else b]) for b in range(B)]
        cache.fork(parents)
        history = [list(history[p]) if p >= 0 else [(torch.empty(0, kv, d, device=DEV, dtype=cache.pool.dtype),) * 2 for _ in range(layers)] for p in parents]
        if step % 4 == 3:
            used = cache.compact().item()
            assert (cache.refs[:used] > 0).all() and (cache.refs[used:] == 0).all()


@pytest.mark.parametrize("dt,page,heads,kv,d,interleaved", [("f16", 16, 4, 4, 64, False), ("bf16", 32, 6, 2, 128, True)])
def test_a_beam_search_over_the_cache(dt, page, heads, kv, d, interleaved):
    """Every answer of a run of prompts, steps, forks, frees and compactions is the attention over the sequence's own history."""
    layers, B = 2, 7
    cache = tt.PagedKVCache(layers, 400, B, 600, kv, d, page, DT[dt], DEV)
    rotary = tt.RotaryEmbedding(d // 2, interleaved=interleaved, device=DEV)
    for (k, v), q, out in play(cache, rotary, layers, heads, kv, d, 12, 1):
        class Held:
            past, new = [k.shape[0] - q.shape[0]], [q.shape[0]]
            held = staticmethod(lambda b, n, k=k, v=v: (k, v))
        want, off = attended(q, Held, True, d ** -0.5)
        assert ((out.double() - want).abs() <= off).all()
    assert status() == _capi.OK
    cache.release(range(B))
    assert (cache.refs == 0).all() and (cache.lens == 0).all() and (cache.table == -1).all()


def test_a_step_replayed_from_a_graph_and_on_other_streams():
    """One step, captured: fork, reserve, copy, append, attention, advance; replayed it goes on from where the tables on the device are. A second graph of the same
    context is alive, an eager call comes between, on a stream of its own: each is what the eager run gives."""
    B, heads, kv, d, steps = 5, 4, 2, 64, 40
    g = gen(9)
    q, k, v = (randn(g, steps, B, h, d, dtype=torch.float16) for h in (heads, kv, kv))
    cu, ones, parents = cumulative([1] * B), ints([1] * B), ints([0, 0, 2, 3, 1])
    rotary = tt.RotaryEmbedding(d, device=DEV)

    def fresh():
        c = tt.PagedKVCache(1, 64, B, 160, kv, d, 16, torch.float16, DEV)
        c.reserve([20] * B)
        rows = randn(gen(10), 20 * B, kv, d, dtype=torch.float16)
        c.append(0, rows, rows.flip(0), cumulative([20] * B))
        c.advance([20] * B)
        return c

    def step(c, q, k, v, out):
        c.fork(parents)
        c.reserve(ones)
        c.attend(0, c.append(0, k, v, cu, q=q, rotary=rotary), cu, out=out)
        c.advance(ones)

    eager = fresh()
    want = []
    for i in range(steps):
        out = torch.empty_like(q[0])
        step(eager, q[i], k[i], v[i], out)
        want.append(out)

    side = torch.cuda.Stream()
    caches, graphs, places = [fresh(), fresh()], [], []
    for c in caches:
        place = [x[0].clone() for x in (q, k, v)] + [torch.empty_like(q[0])]
        keep = [x.clone() for x in (c.table, c.lens, c.refs, c.pool)]
        with torch.cuda.stream(side):
            step(c, *place)  # warm
        side.synchronize()
        for x, y in zip((c.table, c.lens, c.refs, c.pool), keep):
            x.copy_(y)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        cxx.arena_begin(0, 32 << 20)
        with torch.cuda.graph(graph, stream=side):
            step(c, *place)
        graphs.append((graph, cxx.arena_end(0)[1]))
        places.append(place)
    cxx.set_stream(0, torch.cuda.current_stream().cuda_stream)
    third = fresh()
    for i in range(steps):
        for (graph, _), place in zip(graphs, places):
            for x, y in zip(place, (q[i], k[i], v[i])):
                x.copy_(y)
            graph.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            out = torch.empty_like(q[0])
            step(third, q[i], k[i], v[i], out)
        torch.cuda.synchronize()
        assert all(torch.equal(p[3], want[i]) for p in places) and torch.equal(out, want[i])
    assert all(torch.equal(c.table, eager.table) and torch.equal(c.lens, eager.lens) for c in caches + [third]) and status() == _capi.OK
    for graph, arena in graphs:
        del graph
    graphs.clear()
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------------
def test_calls_that_are_refused():
    pool = Pool(8, torch.float16, [10], [1], 2, 64, 16)
    q = randn(pool.g, 1, 4, 64, dtype=torch.float16)
    keys, values, table, cu, past = pool.args()
    freqs = torch.ones(32, dtype=torch.float64, device=DEV)
    at = torch.zeros(1, dtype=torch.int64, device=DEV)

    def refused(f, *a, error=ValueError, **k):
        with pytest.raises(error):
            f(*a, **k)

    refused(tt.paged_attention, q.cpu(), keys, values, table, cu, past, error=RuntimeError)
    refused(tt.paged_attention, q.float(), keys, values, table, cu, past)
    refused(tt.paged_attention, q[:, :3], keys, values, table, cu, past)
    refused(tt.paged_attention, q.bfloat16(), keys, values, table, cu, past)
    refused(tt.paged_attention, q, keys, values, table.long(), cu, past)
    refused(tt.paged_attention, q, keys, values, table, cu.long(), past)
    refused(tt.paged_attention, q, keys, values, table, cu, past.cpu())
    refused(tt.paged_attention, q, keys, values, table, cu[:1], past)
    refused(tt.paged_attention, q, keys.transpose(1, 2), values.transpose(1, 2), table, cu, past)
    refused(tt.paged_attention, q, keys, values[:, :1], table, cu, past)
    refused(tt.paged_attention, q.transpose(1, 2), keys, values, table, cu, past)
    refused(tt.paged_attention, q, keys, values, table, cu, past, out=torch.empty_like(q[:, :2]))
    refused(tt.paged_attention, q, keys, values, table, cu, past, scale=0.0, error=RuntimeError)
    refused(tt.paged_attention, q, keys, values, table, cu, past, scale=float("nan"), error=RuntimeError)
    refused(tt.paged_attention, q, keys[:, :, :8].contiguous(), values[:, :, :8].contiguous(), table, cu, past, error=RuntimeError)
    odd = torch.zeros(4 * 64 + 1, dtype=torch.float16, device=DEV)[1:].view(1, 4, 64)
    refused(tt.paged_attention, odd, keys, values, table, cu, past, error=RuntimeError)
    refused(tt.paged_attention, q[..., :32].contiguous(), keys[..., :32].contiguous(), values[..., :32].contiguous(), table, cu, past, error=RuntimeError)
    many = 1025
    refused(tt.paged_attention, q, keys, values, table.expand(many, -1).contiguous(), torch.zeros(many + 1, dtype=torch.int32, device=DEV),
            torch.zeros(many, dtype=torch.int32, device=DEV), error=RuntimeError)
    refused(tt.paged_append, q[:, :2], q[:, :2], keys, values, table, cu, past, q=q)
    refused(tt.paged_append, q, q, keys, values, table, cu, past)
    refused(tt.paged_append, q[:, :2], q[:, :1], keys, values, table, cu, past)
    refused(tt.paged_append, q[:, :2], q[:, :2], keys, values, table, cu, past, q=q, freqs=freqs.float())
    refused(tt.paged_append, q[:, :2], q[:, :2], keys, values, table, cu, past, q=q, freqs=torch.ones(33, dtype=torch.float64, device=DEV), error=RuntimeError)
    refused(tt.rotary, q, q, at.int(), freqs)
    refused(tt.rotary, q, q[:, :, :32], at, freqs)
    refused(tt.rotary, q, q, at, torch.ones(33, dtype=torch.float64, device=DEV), error=RuntimeError)
    refused(tt.rotary, q, None, at, freqs, out=(q, q))
    refused(tt.rotary, q[..., :60].contiguous(), None, at, freqs[:8], error=RuntimeError)
    refused(tt.paged_copy, torch.zeros(2, 3, 7, device=DEV, dtype=torch.float16), ints([[0, 1]]), error=RuntimeError)
    refused(tt.paged_copy, torch.zeros(2, 3, 8, device=DEV), ints([0, 1]))
    refused(tt.paged_reserve, table, past, ints([0] * 5), ints([1]), 0, error=RuntimeError)
    refused(tt.paged_fork, table, past, ints([0] * 5), ints([1, 2]))
    refused(tt.paged_compact, table, ints([0] * 5), torch.zeros(1, 4, 8, device=DEV), error=RuntimeError)
    refused(tt.RotaryEmbedding, 63)
    refused(tt.RotaryEmbedding, 64, stretch="other")
    refused(tt.PagedKVCache, 1, 4, 1, 64, 2, 64, dtype=torch.float32, error=NotImplementedError)
    assert status() == _capi.OK


def test_the_c_interface(ctx):
    """The same through the C ABI, and its null pointers."""
    pool = Pool(11, torch.bfloat16, [40, 9], [2, 1], 2, 128, 16)
    g = pool.g
    q, k, v = (randn(g, 3, h, 128, dtype=torch.bfloat16) for h in (4, 2, 2))
    out, turned_q = torch.empty_like(q), torch.empty_like(q)
    freqs = 10000.0 ** (-torch.arange(64, dtype=torch.float64, device=DEV) / 64)
    kv = dict(keys=pool.keys, values=pool.values, page_stride=pool.keys.stride(0), pages=pool.keys.shape[0], kv_heads=2, page_tokens=16, d=128, table=pool.table,
              table_stride=pool.table.stride(0), table_width=pool.table.shape[1], cu_seqlens=pool.cu, past_lens=pool.past_lens, B=2)
    ctx.paged_append(_capi.BF16, kv, 3, k, 256, v, 256, dict(freqs=freqs, rotary_dim=128, interleaved=0, scale=1.0, q=q, q_out=turned_q, ldq=512, ldq_out=512, heads=4))
    ctx.paged_attention(_capi.BF16, kv, turned_q, 512, 3, 4, 1, 0.1, out, 512)
    assert ctx.device_status() == _capi.OK
    want, off = attended(turned_q, pool, True, 0.1)
    assert ((out.double() - want).abs() <= off).all()
    lib, h = _capi.lib(), ctx.h
    for bad in (dict(keys=None), dict(table=None), dict(cu_seqlens=None), dict(past_lens=None), dict(page_tokens=24), dict(page_stride=8), dict(page_stride=4097), dict(d=96),
                dict(kv_heads=0), dict(pages=0), dict(B=-1), dict(B=2000), dict(table_width=0), dict(table_stride=1)):
        with pytest.raises(_capi.TTBError):
            ctx.paged_attention(_capi.BF16, {**kv, **bad}, turned_q, 512, 3, 4, 1, 0.1, out, 512)
    for f in ("ttb_rotary", "ttb_paged_fork", "ttb_paged_copy"):
        assert getattr(lib, f)(h, *([None] * (len(_capi.SIGNATURES[f][1]) - 2)), *([None] if f == "ttb_rotary" else [0] if f == "ttb_paged_copy" else [None])) == _capi.ERR_INVALID
    assert lib.ttb_paged_attention(None, 1, None, None, 0, 0, 0, 0, 1.0, None, 0) == _capi.ERR_INVALID
    with pytest.raises(_capi.TTBError):
        ctx.paged_attention(_capi.F32, kv, turned_q, 512, 3, 4, 1, 0.1, out, 512)
