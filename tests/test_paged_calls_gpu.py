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
    return torch.tensor(values, dtype=torch.int32, device=DEV)


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
