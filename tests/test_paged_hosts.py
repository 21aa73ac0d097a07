"""Tensors in host memory, or laid out otherwise than the kernels read them, are
refused before any call of the library: here with a library that must not be
called, so that no GPU is needed."""
from __future__ import annotations

import dataclasses

import pytest
import torch

from strict_topk_overlap_b200 import _lib, metadata, paged_append, paged_attention


class Untouched:
    """Stands for the loaded library: workspace sizes may be asked for, nothing else."""

    def stk_paged_attention_workspace_bytes(self, *args):
        return 0

    def __getattr__(self, name):
        def call(*args):
            raise AssertionError(f"{name} was called")
        return call


@pytest.fixture(autouse=True)
def library(monkeypatch):
    monkeypatch.setattr(_lib, "load", lambda path=None: Untouched())


class OnDevice(torch.Tensor):
    """A host tensor that says it is on device 0."""

    def get_device(self):
        return 0


def _on_device(x):
    return x.as_subclass(OnDevice)


def _cache(on=lambda x: x):
    cache = paged_append.empty_paged_cache([64, 64], 2, 64, 32, 16, device="cpu")
    return dataclasses.replace(cache, **{f: on(getattr(cache, f)) for f in
                                         ("k_pages", "v_pages", "page_table", "block_offsets", "lo", "hi")})


def _calls(cache, on):
    x = on(torch.zeros((2, 4, 64), dtype=torch.bfloat16))
    at = on(torch.ones(2, dtype=torch.int32))
    return (lambda: paged_append.append_tokens(cache, on(x[:, :2]), on(x[:, 2:]), at),
            lambda: paged_attention.attention(x, cache, at),
            lambda: paged_attention.shared_prefix_attention(x, cache, at, 16))


def test_host_tensors_are_refused():
    for call in _calls(_cache(), lambda x: x):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("name", ["v_pages", "page_table", "block_offsets", "lo", "hi"])
def test_one_host_tensor_of_the_cache_is_refused(name):
    cache = _cache(_on_device)
    setattr(cache, name, getattr(cache, name).as_subclass(torch.Tensor))
    calls = _calls(cache, _on_device)
    for call in calls[:1] if name in ("lo", "hi") else calls:
        with pytest.raises(ValueError, match="device"):
            call()


@pytest.mark.parametrize("change", [
    dict(k_pages=lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)), dict(v_pages=lambda x: x[::2]),
    dict(v_pages=lambda x: x.float()), dict(page_table=lambda x: x.long()), dict(page_table=lambda x: x[::2]),
    dict(block_offsets=lambda x: x.long())])
def test_other_layouts_of_the_cache_are_refused(change):
    cache = _cache(_on_device)
    for name, f in change.items():
        setattr(cache, name, _on_device(f(getattr(cache, name).as_subclass(torch.Tensor))))
    for call in _calls(cache, _on_device):
        with pytest.raises(ValueError):
            call()


def test_host_workspace_is_refused():
    cache = _cache(_on_device)
    x, at = _on_device(torch.zeros((2, 4, 64), dtype=torch.bfloat16)), _on_device(torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="workspace"):
        paged_attention.attention(x, cache, at, workspace=torch.empty(1 << 20, dtype=torch.uint8))


def test_streams_of_host_tensors_are_refused():
    """The older calls have no other check of the device than this."""
    with pytest.raises(ValueError, match="CUDA"):
        _lib.stream_of(torch.zeros(1))
    k, lo = torch.zeros((2, 3, 8, 16)), torch.zeros((2, 3, 16))
    with pytest.raises(ValueError, match="CUDA"):
        metadata.append_token(k, k.clone(), lo, lo.clone(), k[:, 0, 0], k[:, 0, 0], 4)


@pytest.mark.parametrize("current", [0, 1])
def test_launches_happen_on_the_tensors_device(monkeypatch, current):
    """Two devices in one process: the library launches on the current one, which has to be the tensors'."""
    state, seen = {"device": current}, []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, state["device"] = state["device"], self.index

        def __exit__(self, *error):
            state["device"] = self.before

    class Launches(Untouched):
        def __getattr__(self, name):
            def call(*args):
                seen.append(state["device"])
                return 0
            return call

    monkeypatch.setattr(_lib, "load", lambda path=None: Launches())
    monkeypatch.setattr(_lib, "raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "current_device", lambda: state["device"])
    for call in _calls(_cache(_on_device), _on_device):
        call()
    assert seen == [0, 0, 0] and state["device"] == current


@pytest.mark.parametrize("d,scale", [(64, 1.0), (128, 60.0), (1024, 65504.0)])
def test_bounds_of_empty_blocks_score_in_fp32(d, scale):
    """A block without tokens scores far below all others, in sums that stay finite (infinite ones would have every
    such block rescored exactly)."""
    cache = paged_append.empty_paged_cache([64], 2, d, 32, 16, device="cpu")
    q = scale * torch.randn((16, d), generator=torch.Generator().manual_seed(1))
    for h in range(2):
        top = (q.clamp(min=0) @ cache.hi[h].T + q.clamp(max=0) @ cache.lo[h].T)
        assert bool(top.isfinite().all()) and bool((top < -1e28).all())
