"""CPU: what PagedKVCache works out on the host."""
import pytest
import torch

import turbotransformers_b200 as tt


@pytest.mark.parametrize("gone", [[1, 3], (3, 1, 1), range(1, 4, 2), {1, 3}, torch.tensor([1, 3]), torch.tensor([3, 1], dtype=torch.int32)])
def test_release_frees_the_sequences_that_it_is_given(gone, monkeypatch):
    """Whatever they are given as: a tensor's elements are tensors of their own, equal to no number as keys of a set."""
    cache, forks = tt.PagedKVCache(1, 4, 5, 64, 2, 64, device="cpu"), []
    monkeypatch.setattr(cache, "fork", lambda parents: forks.append(list(parents)))
    cache.release(gone)
    assert forks == [[0, -1, 2, -1, 4]]


def test_advance_counts_what_had_room():
    cache = tt.PagedKVCache(1, 4, 3, 64, 2, 64, device="cpu")
    cache.advance([1, 2, 3])
    cache.room[1] = 0
    cache.advance(torch.tensor([10, 10, 10]))
    cache.advance(torch.tensor([5, 5, 5], dtype=torch.int32))
    assert cache.lens.tolist() == [16, 2, 18] and cache.lens.dtype == torch.int32
