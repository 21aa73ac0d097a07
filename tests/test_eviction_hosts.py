"""Refusals of the eviction and sampling calls on the host, without a GPU: by
the Python entry points with a library that must not be called, and by the
library itself."""
from __future__ import annotations

import pytest
import torch

from strict_topk_overlap_b200 import _lib, paged_eviction, sampling
from test_paged_hosts import Untouched, _cache, _on_device


@pytest.fixture
def untouched(monkeypatch):
    class Sizes(Untouched):
        def stk_accumulate_weights_workspace_bytes(self, *args):
            return 0

        def stk_evict_tokens_workspace_bytes(self, *args):
            return 0

    class Device:
        def __init__(self, index):
            pass

        def __enter__(self):
            pass

        def __exit__(self, *error):
            pass

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "load", lambda path=None: Sizes())


def _args(on=_on_device):
    return dict(weights=on(torch.zeros(2, 4, 32)), q=on(torch.zeros((2, 4, 64), dtype=torch.bfloat16)),
                lengths=on(torch.ones(2, dtype=torch.int32)), lse=on(torch.zeros(2, 4)))


def _weigh(cache, weights, q, lengths, lse, **more):
    return paged_eviction.accumulate_weights(weights, q, cache, lengths, lse, **more)


def _evict(cache, weights, lengths, keep=8, **more):
    return paged_eviction.evict(cache, weights, lengths, keep, **more)


def test_host_tensors(untouched):
    a = _args(lambda x: x)
    with pytest.raises(ValueError, match="CUDA"):
        _weigh(_cache(), **a)
    with pytest.raises(ValueError, match="CUDA"):
        _evict(_cache(), a["weights"], a["lengths"])
    with pytest.raises(ValueError, match="CUDA"):
        sampling.sample(torch.zeros(2, 5), torch.zeros(2))


@pytest.mark.parametrize("name", ["weights", "q", "lengths", "lse"])
def test_one_host_tensor(untouched, name):
    a = _args()
    a[name] = a[name].as_subclass(torch.Tensor)
    with pytest.raises(ValueError, match="device"):
        _weigh(_cache(_on_device), **a)
    if name in ("weights", "lengths"):
        with pytest.raises(ValueError, match="device"):
            _evict(_cache(_on_device), a["weights"], a["lengths"])


@pytest.mark.parametrize("change", [
    dict(weights=torch.zeros(2, 4, 16)), dict(weights=torch.zeros((2, 4, 32), dtype=torch.float64)),
    dict(weights=torch.zeros(2, 4, 64)[..., ::2]), dict(q=torch.zeros(2, 3, 64)), dict(q=torch.zeros(2, 4, 64)),
    dict(q=torch.zeros((2, 4, 128), dtype=torch.bfloat16)[..., ::2]), dict(lse=torch.zeros(2, 3)), dict(lse=torch.zeros(4, 2).T),
    dict(lse=torch.zeros((2, 4), dtype=torch.bfloat16)), dict(lengths=torch.ones(3, dtype=torch.int32)), dict(lengths=torch.ones(2)),
    dict(slopes=torch.zeros(3)), dict(kv_lo=torch.zeros(2)), dict(kv_hi=torch.zeros(1, dtype=torch.int32)), dict(softcap=-1.0),
    dict(scale=0.0), dict(token_offsets=torch.zeros(2, dtype=torch.int32)), dict(max_tokens=0, token_offsets=torch.zeros(3, dtype=torch.int32))])
def test_arguments_of_weights(untouched, change):
    a = _args() | {n: _on_device(x) if isinstance(x, torch.Tensor) else x for n, x in change.items()}
    with pytest.raises(ValueError):
        _weigh(_cache(_on_device), **a)


@pytest.mark.parametrize("change", [
    dict(keep=0), dict(keep=-3), dict(first=5, last=4), dict(first=-1), dict(last=-1), dict(weights_out=torch.zeros(2, 4, 16)),
    dict(workspace=torch.zeros(100, dtype=torch.uint8))])
def test_arguments_of_eviction(untouched, change):
    a = _args()
    more = {n: _on_device(x) if isinstance(x, torch.Tensor) and n != "workspace" else x for n, x in change.items()}
    with pytest.raises(ValueError):
        _evict(_cache(_on_device), a["weights"], a["lengths"], **more)


def test_workspaces_without_memory_of_their_own(untouched):
    a, spread = _args(), _on_device(torch.zeros(1, dtype=torch.uint8).expand(1 << 20))
    with pytest.raises(ValueError, match="workspace"):
        _weigh(_cache(_on_device), **a, workspace=spread)
    with pytest.raises(ValueError, match="workspace"):
        _evict(_cache(_on_device), a["weights"], a["lengths"], workspace=spread)


def test_bounds_of_eviction(untouched):
    a, cache = _args(), _cache(_on_device)
    cache.hi = _on_device(torch.zeros(2, 4, 32))
    with pytest.raises(ValueError, match="hi"):
        _evict(cache, a["weights"], a["lengths"])


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(5)), dict(logits=torch.zeros(2, 0)), dict(logits=torch.zeros(5, 2).T), dict(logits=torch.zeros(2, 5, dtype=torch.int32)),
    dict(uniforms=torch.zeros(3)), dict(uniforms=torch.zeros(2, dtype=torch.float64)), dict(temperature=-1.0), dict(top_k=-1), dict(top_p=-0.5),
    dict(min_p=float("nan")), dict(top_k=torch.zeros(2)), dict(top_p=torch.zeros(3)), dict(temperature=torch.zeros(2, dtype=torch.float64)),
    dict(out=torch.zeros(2)), dict(out=torch.zeros(3, dtype=torch.int32))])
def test_arguments_of_sampling(untouched, change):
    a = dict(logits=torch.zeros(2, 5), uniforms=torch.zeros(2)) | change
    a = {n: _on_device(x) if isinstance(x, torch.Tensor) else x for n, x in a.items()}
    with pytest.raises(ValueError):
        sampling.sample(a.pop("logits"), a.pop("uniforms"), **a)


def test_launches_happen_on_the_tensors_device(monkeypatch):
    state, seen = {"device": 1}, []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, state["device"] = state["device"], self.index

        def __exit__(self, *error):
            state["device"] = self.before

    class Launches:
        def __getattr__(self, name):
            def call(*args):
                if not name.endswith("bytes"):
                    seen.append(state["device"])
                return 0
            return call

    monkeypatch.setattr(_lib, "load", lambda path=None: Launches())
    monkeypatch.setattr(_lib, "raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "current_device", lambda: state["device"])
    a = _args()
    _weigh(_cache(_on_device), **a)
    _evict(_cache(_on_device), a["weights"], a["lengths"])
    sampling.sample(_on_device(torch.zeros(2, 5)), _on_device(torch.zeros(2)))
    assert seen == [0, 0, 0] and state["device"] == 1


# ------------------------------------------------------------------ the library

@pytest.fixture(scope="module")
def lib():
    from strict_topk_overlap_b200.build import build_library
    build_library()
    return _lib.load()


def _kv(**more):
    f = dict(k=256, v=256, dtype=2, hkv=2, n=0, b=32, d=64, table=256, offsets=256, page=16, stride=0)
    f.update(more)
    return _lib.PACK_KV(*f.values())


def test_library_refusals_of_weights(lib):
    def call(kv=None, pages=8, q=256, R=1, T=1, hq=4, total=2, lengths=256, offsets=None, most=1, longest=64, options=None, lse=256,
             weights=256, ws=None, ws_bytes=0):
        return lib.stk_accumulate_weights(_kv() if kv is None else kv, pages, q, 256, 64, R, T, hq, total, lengths, offsets, most,
                                          longest, options, lse, weights, ws, ws_bytes, None, None)

    masked = _lib.PACK_OPTIONS(0.0, 0.0, 0, 256, 0)
    for bad, word in ((dict(q=None), b"null"), (dict(lse=None), b"null"), (dict(weights=None), b"null"), (dict(pages=0), b"empty pool"),
                      (dict(T=2), b"shape"), (dict(most=2), b"shape"), (dict(total=0), b"blocks"), (dict(hq=3), b"divisible"),
                      (dict(kv=_kv(table=0)), b"paged"), (dict(kv=_kv(dtype=9)), b"dtype"),
                      (dict(options=_lib.PACK_OPTIONS(0.0, -1.0, 0, 0, 0)), b"softcap"),
                      (dict(options=masked, ws=264, ws_bytes=1 << 20), b"boundary")):
        assert call(**bad) == -1 and word in lib.stk_last_error(), (bad, lib.stk_last_error())
    assert call(options=masked) == -4 and b"workspace" in lib.stk_last_error()
    assert call(T=0, offsets=256, most=0, q=None) == 0
    need = lib.stk_accumulate_weights_workspace_bytes
    assert need(_kv(), 1, 1, 4, 2, 0, 1, 64, 0) == 0 and need(_kv(), 1, 1, 4, 2, 0, 1, 64, 1) % 16 == 0
    assert need(_kv(), 1, 4000, 4, 128, 1, 4000, 4096, 0) > 0


def test_library_refusals_of_eviction(lib):
    def call(kv=None, pages=8, R=1, total=2, lengths=256, keep=8, first=0, last=0, longest=64, weights=256, out=256, lo=256, hi=256,
             kept=256, now=512, ws=256, ws_bytes=1 << 20):
        return lib.stk_evict_tokens(_kv() if kv is None else kv, pages, R, total, lengths, keep, first, last, longest, weights, out, lo,
                                    hi, kept, now, ws, ws_bytes, None, None)

    for bad, word in ((dict(lengths=None), b"null"), (dict(weights=None), b"null"), (dict(out=None), b"null"), (dict(kept=None), b"null"),
                      (dict(now=None), b"null"), (dict(pages=0), b"pool"), (dict(R=0), b"shape"), (dict(total=0), b"shape"),
                      (dict(longest=0), b"shape"), (dict(keep=0), b"kept"), (dict(first=5, last=4), b"kept"), (dict(first=-1), b"kept"),
                      (dict(first=2 ** 31 - 1, last=2 ** 31 - 1), b"kept"), (dict(hi=None), b"together"), (dict(now=256), b"lengths_out"),
                      (dict(out=256 + 4), b"apart"), (dict(weights=256 + 64 * 4), b"apart"),
                      (dict(kv=_kv(table=0)), b"paged"), (dict(ws=264), b"boundary"), (dict(pages=2 ** 31 - 1), b"rows")):
        assert call(**bad) == -1 and word in lib.stk_last_error(), (bad, lib.stk_last_error())
    assert call(longest=400000) == -2 and b"393216" in lib.stk_last_error()
    assert call(ws_bytes=16) == -4 and b"workspace" in lib.stk_last_error()


def test_library_refusals_of_sampling(lib):
    def call(logits=256, dtype=0, stride=5, R=2, V=5, u=256, t=1.0, k=0, p=1.0, m=0.0, out=256):
        return lib.stk_sample_tokens(logits, dtype, stride, R, V, u, None, t, None, k, None, p, None, m, out, None, None)

    for bad, word in ((dict(logits=None), b"null"), (dict(u=None), b"null"), (dict(out=None), b"null"), (dict(dtype=5), b"dtype"),
                      (dict(V=0), b"shape"), (dict(R=-1), b"shape"), (dict(stride=-5), b"shape"), (dict(t=-1.0), b"negative"),
                      (dict(t=float("nan")), b"negative"), (dict(k=-1), b"negative"), (dict(p=-0.1), b"negative"), (dict(m=-1.0), b"negative")):
        assert call(**bad) == -1 and word in lib.stk_last_error(), (bad, lib.stk_last_error())
    assert call(V=400000) == -2 and b"393216" in lib.stk_last_error()
    assert call(R=0, logits=None) == 0
