"""Host-side checks of the paged token entry points, without a GPU: bad
arguments are refused with a message before any device work, and sizes that
need no workspace ask for none."""
from __future__ import annotations

import pytest


@pytest.fixture(scope="module")
def lib():
    from strict_topk_overlap_b200 import _lib as L
    from strict_topk_overlap_b200.build import build_library
    build_library()
    return L.load()


def _kv(**more):
    from strict_topk_overlap_b200 import _lib as L
    f = dict(k=256, v=256, dtype=2, hkv=2, n=0, b=32, d=64, table=256, offsets=256, page=16, stride=0)
    f.update(more)
    return L.PACK_KV(*f.values())


def test_append_refusals(lib):
    from strict_topk_overlap_b200 import _lib as L

    def call(kv=None, pages=8, R=1, total=1, T=1, k=256, v=256, q=None, q_out=None, hq=0, lengths=256, offsets=None,
             positions=None, rotary=None, lo=256, hi=256):
        return lib.stk_append_tokens(_kv() if kv is None else kv, pages, R, total, T, k, 128, 64, v, 128, 64, q, 256, 64,
                                     hq, q_out, lengths, offsets, positions, rotary, lo, hi, None, None)

    table = dict(cos=256, sin=256, pairs=32, most=10, inter=0, axes=1, axis=0)
    for bad, word in ((dict(k=None), b"null"), (dict(lengths=None), b"null"), (dict(pages=0), b"shape"),
                      (dict(T=2), b"shape"), (dict(R=0), b"shape"), (dict(hi=None), b"together"),
                      (dict(q=256, hq=4), b"q_out"), (dict(q=256, q_out=256, hq=3), b"divisible"),
                      (dict(kv=_kv(table=0)), b"paged"), (dict(kv=_kv(page=12)), b"page size"),
                      (dict(kv=_kv(dtype=9)), b"dtype"),
                      (dict(rotary=L.PACK_ROTARY(*dict(table, pairs=33).values())), b"rotary"),
                      (dict(rotary=L.PACK_ROTARY(*dict(table, cos=0).values())), b"rotary"),
                      (dict(rotary=L.PACK_ROTARY(*dict(table, axis=256).values())), b"axes")):
        assert call(**bad) == -1 and word in lib.stk_last_error(), (bad, lib.stk_last_error())
    assert call(T=0, offsets=256, k=None, v=None) == 0


def test_attention_refusals(lib):
    from strict_topk_overlap_b200 import _lib as L

    def call(kv=None, pages=8, q=256, R=1, T=1, hq=4, lengths=256, offsets=None, most=1, longest=64, prefix=0,
             options=None, out=256, ws=None, ws_bytes=0):
        return lib.stk_paged_attention(_kv() if kv is None else kv, pages, q, 256, 64, R, T, hq, lengths, offsets, most,
                                       longest, prefix, options, out, None, ws, ws_bytes, None, None)

    for bad, word in ((dict(q=None), b"null"), (dict(out=None), b"null"), (dict(pages=0), b"empty pool"),
                      (dict(T=2), b"shape"), (dict(most=2), b"shape"), (dict(most=0), b"shape"),
                      (dict(longest=0), b"shape"), (dict(prefix=8), b"prefix"), (dict(prefix=-16), b"prefix"),
                      (dict(prefix=96), b"prefix"), (dict(hq=3), b"divisible"), (dict(kv=_kv(table=0)), b"paged"),
                      (dict(options=L.PACK_OPTIONS(0.0, -1.0, 0, 0, 0)), b"softcap"),
                      (dict(options=L.PACK_OPTIONS(float("nan"), 0.0, 0, 0, 0)), b"scale")):
        assert call(**bad) == -1 and word in lib.stk_last_error(), (bad, lib.stk_last_error())
    assert call() == -4 and b"workspace" in lib.stk_last_error()
    assert call(T=0, offsets=256, most=0, q=None, out=None) == 0


def test_workspace_bytes(lib):
    need = lib.stk_paged_attention_workspace_bytes
    assert need(_kv(), 1, 0, 4, 1, 0, 64, 0) == 0          # no tokens
    assert need(_kv(), 2, 1, 4, 0, 1, 64, 0) == 0          # refused shape
    assert need(_kv(), 1, 100000, 4, 1, 100000, 1 << 20, 0) == 0  # tiles for every SM: nothing to join
    assert need(_kv(), 1, 1, 4, 0, 1, 64, 0) % 16 == 0 and need(_kv(), 1, 1, 4, 0, 1, 64, 0) > 0
    assert need(_kv(), 4, 4, 4, 0, 1, 256, 64) > need(_kv(), 4, 4, 4, 0, 1, 256, 0)
