"""Arguments of the eviction calls that numbers of 32 bits or a program's
defaults would change, on the host."""
from __future__ import annotations

import pytest
import torch

from strict_topk_overlap_b200 import _lib, paged_eviction
from test_paged_hosts import _cache, _on_device


class Refuses:
    def __getattr__(self, name):
        raise AssertionError(f"{name} must not be called")


@pytest.mark.parametrize("keep", [2 ** 31, 2 ** 32 + 1, 2 ** 40])
def test_more_tokens_than_32_bits_hold(monkeypatch, keep):
    """keep = 2^32 + 1 is not keep = 1."""
    monkeypatch.setattr(_lib, "load", lambda path=None: Refuses())
    weights, lengths = _on_device(torch.zeros(2, 4, 32)), _on_device(torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="keep"):
        paged_eviction.evict(_cache(_on_device), weights, lengths, keep)
    with pytest.raises(ValueError, match="keep"):
        paged_eviction.evict_workspace(_cache(_on_device), keep)


@pytest.mark.parametrize("kind", [torch.float64, torch.bfloat16])
def test_weights_are_fp32_whatever_the_default(kind):
    before = torch.get_default_dtype()
    torch.set_default_dtype(kind)
    try:
        weights = paged_eviction.empty_weights(_cache())
    finally:
        torch.set_default_dtype(before)
    assert weights.dtype is torch.float32 and weights.shape == (2, 4, 32)
