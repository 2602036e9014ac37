"""Attention over cache pages where the key that a row sees first outweighs each of thousands of others, as the first tokens of a text do: what is left for those is theirs."""
import math

import pytest
import torch

import turbotransformers_b200 as tt
from turbotransformers_b200 import _capi
from turbotransformers_b200._cxx import cxx

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,heads,above", [(1, 1, 17.0), (1, 8, 12.0), (1, 16, 17.0), (3, 8, 15.0), (40, 4, 17.0), (200, 1, 17.0), (130, 2, 10.0)])
def test_one_key_far_above_all_others(new, heads, above, d, dt):
    """The first key's values are zero, so that an output is the others' share alone. All sequences list the same pages, and there are so many that a row's keys are not dealt out
    to many CTAs.

    A probability is rounded to 16 bits: off by u of itself, or, of a normal number's range, by half a step between subnormal ones, in fp16 2^-25 where the largest
    is 2^6 and more (the reference lies that far below the first maximum): 2^-31 of the largest. exp2, sums and scores are fp32: 2^-14 of the mean of the values. The output is rounded once."""
    N, B, page = 6000, 300, 256
    g = torch.Generator(DEV).manual_seed(new * heads + d)
    pages = -(-(N + new) // page)
    keys = torch.zeros(pages, 1, page, d, device=DEV, dtype=dt)
    keys[..., 0] = (0.3 + 0.05 * torch.randn(pages, 1, page, generator=g, device=DEV)).to(dt)
    keys[0, 0, 0, 0] = above
    values = torch.rand(pages, 1, page, d, generator=g, device=DEV).add_(0.5).to(dt)
    values[0, 0, 0] = 0
    q = torch.zeros(B * new, heads, d, device=DEV, dtype=dt)
    q[..., 0] = 1 + torch.arange(heads, device=DEV) / 64
    table = torch.arange(pages, device=DEV, dtype=torch.int32).expand(B, -1).contiguous()
    cu, past = torch.arange(B + 1, device=DEV, dtype=torch.int32) * new, torch.full((B,), N, device=DEV, dtype=torch.int32)
    got = tt.paged_attention(q, keys, values, table, cu, past, scale=1.0).view(B, new, heads, d).double()
    assert cxx.device_status(0) == _capi.OK
    k, v = keys.view(-1, d)[:N + new, 0].double(), values.view(-1, d)[:N + new].double()
    u, fi = torch.finfo(dt).eps / 2, torch.finfo(dt)
    for h in range(heads):
        score = q[0, h, 0].double() * k
        w = (score - score.max()).exp()
        total, sums = w.cumsum(0)[N:, None], (w[:, None] * v).cumsum(0)[N:]
        want, mean = sums / total, sums / total  # (no value is negative)
        off = (u * want).clamp(min=fi.smallest_normal * u) + (u + 2.0 ** -14) * mean
        if dt == torch.float16:
            off += 2.0 ** -31 * v.cumsum(0)[N:] / total
        far = (got[:, :, h] - want).abs()
        assert (far <= off).all(), f"{(far / off).max().item():.3g} times the tolerance, {(far / want).max().item():.3g} of the output"


def test_an_even_cache_keeps_its_reference():
    """Scores that are all alike, and first ones that are lower than the rest by more and more: equal weights, whatever the reference."""
    N, d = 5000, 64
    for dt in (torch.float16, torch.bfloat16):
        for rise in (0.0, 2.0, 5.0, 6.5, 9.0, 20.0):
            for new in (1, 150):
                pages = -(-(N + new) // 64)
                keys = torch.zeros(pages, 1, 64, d, device=DEV, dtype=dt)
                keys[..., 0] = rise
                keys[0, 0, :32, 0] = 0
                values = torch.ones(pages, 1, 64, d, device=DEV, dtype=dt)
                values[0, 0, :32] = 0
                q = torch.zeros(new, 2, d, device=DEV, dtype=dt)
                q[..., 0] = 1
                table = torch.arange(pages, device=DEV, dtype=torch.int32)[None].contiguous()
                got = tt.paged_attention(q, keys, values, table, torch.tensor([0, new], device=DEV, dtype=torch.int32), torch.tensor([N], device=DEV, dtype=torch.int32),
                                         scale=1.0).double()
                n = N + 1 + torch.arange(new, device=DEV).double()[:, None, None]
                want = (n - 32) / (n - 32 + 32 * math.exp(-rise))
                u = torch.finfo(dt).eps / 2
                assert ((got - want).abs() <= (2 * u + 2.0 ** -14) * want).all()
    assert cxx.device_status(0) == _capi.OK
