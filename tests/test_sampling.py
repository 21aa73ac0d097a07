"""Sampled tokens against the definition in 64 bits (oracle/eviction.py).

Masses are whole numbers of 2^-44 of the largest, each off by 2^-45 and by 2e-14
of itself (the largest is exact), so that a row's sums are off by at most those
of its smaller masses together, and their products with a share by 2^-50. A
decision of the definition that lies within four times that of its border, on
either side of two sums, is no test of the kernel (it is left out, and such rows
are few); every other one must be the same."""
from __future__ import annotations

import pytest
import torch

from oracle import eviction as E

gpu = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _rows(rows, v, dtype, seed, spread=2.5):
    g = torch.Generator(DEV).manual_seed(seed)
    x = (spread * torch.randn((rows, v), generator=g, device=DEV)).to(dtype)
    return x, torch.rand((rows,), generator=g, device=DEV)


def _check(x, u, *, most_left_out=0.05, **more):
    from strict_topk_overlap_b200 import sampling
    got = sampling.sample(x, u, **more).tolist()
    left_out = 0
    for r in range(x.shape[0]):
        one = {n: (more[n][r].item() if isinstance(more.get(n), torch.Tensor) else more.get(n, d))
               for n, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
        want, near, off = E.sample(x[r], u[r].item(), **one)
        if near < 4 * off:
            left_out += 1
        else:
            assert got[r] == want, (r, got[r], want, near, one)
    assert left_out <= max(1, most_left_out * x.shape[0])
    return got


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,v", [(1, 1), (3, 2), (2, 31), (5, 33), (7, 1000), (3, 4097), (2, 50257), (40, 5000), (1, 131072),
                                    (2, 262143)])
@pytest.mark.parametrize("more", [
    dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=20), dict(top_p=0.9), dict(top_p=0.0), dict(min_p=0.1),
    dict(temperature=0.6, top_k=50, top_p=0.8, min_p=0.02), dict(temperature=1.7, top_p=0.99)])
def test_sample(dtype, rows, v, more):
    x, u = _rows(rows, v, dtype, 1)
    _check(x, u, **more)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_parameters_of_each_row(dtype):
    x, u = _rows(64, 3001, dtype, 2)
    g = torch.Generator(DEV).manual_seed(3)
    pick = lambda values, kind: torch.tensor(values, dtype=kind, device=DEV)[  # noqa: E731
        torch.randint(0, len(values), (64,), generator=g, device=DEV)]
    _check(x, u, temperature=pick([0.0, 0.3, 1.0, 2.0], torch.float32), top_k=pick([0, 1, 7, 3000, 3001, 9999], torch.int32),
           top_p=pick([0.0, 0.5, 0.95, 1.0, 2.0], torch.float32), min_p=pick([0.0, 0.05, 1.0], torch.float32))


@gpu
@pytest.mark.parametrize("v", [40, 5000])
@pytest.mark.parametrize("more", [dict(), dict(top_k=13), dict(top_p=0.501), dict(top_k=13, top_p=0.501), dict(min_p=0.3)])
def test_equal_logits(v, more):
    """Ties go to the lower token: among all equal, and among few values."""
    g = torch.Generator(DEV).manual_seed(4)
    x = torch.cat((torch.zeros((4, v), device=DEV), -torch.zeros((4, v), device=DEV),
                   torch.randint(0, 3, (8, v), generator=g, device=DEV).float()))
    x[1, ::2] = -0.0
    u = torch.rand((16,), generator=g, device=DEV)
    _check(x, u, **more)


@gpu
@pytest.mark.parametrize("more", [dict(), dict(top_k=3), dict(top_p=0.7), dict(temperature=0.0)])
def test_odd_logits(more):
    """Infinities share the mass, NaN and -inf are never chosen, a row of them alone gives -1 and is reported."""
    from strict_topk_overlap_b200 import _lib as L
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[-inf, 1.0, nan, -inf, 2.0, 1.5], [inf, 1.0, inf, nan, inf, 0.0], [-inf] * 6, [nan] * 6,
                      [-inf, -inf, -inf, -3e38, -inf, nan], [3e38, 3.1e38, -3e38, 0.0, 1.0, 2.0]], device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    L.set_status_tensor(status)
    try:
        for u in (0.0, 0.4, 0.999):
            got = _check(x, torch.full((6,), u, device=DEV), most_left_out=1.0, **more)
            assert got[2] == got[3] == -1 and got[4] == 3
    finally:
        L.set_status_tensor(None)
    assert status.item() == 6


@gpu
@pytest.mark.parametrize("more", [dict(), dict(top_k=3), dict(top_p=0.9), dict(min_p=0.2)])
def test_distances_beyond_the_largest_number(more):
    """Logits whose difference FP32 cannot hold, at temperatures that make masses of it all the same."""
    x = torch.tensor([[3e38, -3e38, 1e38, 0.0, -2e38]], device=DEV).expand(64, 5)
    u = torch.arange(64, device=DEV).float() / 64 + 1 / 200
    _check(x, u, temperature=3e38, **more)


@gpu
def test_numbers_at_the_ends():
    """0, the last number below 1, and numbers outside [0, 1), which count as its ends."""
    x, _ = _rows(1, 700, torch.float32, 5)
    x = x.expand(6, 700)
    x[0, 699] = 1.0
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, float("nan")], device=DEV)
    from strict_topk_overlap_b200 import sampling
    first, last, one, more, below, none = sampling.sample(x, u).tolist()
    assert first == below == none == 0 and last == one == more == 699
    assert sampling.sample(x[:0], u[:0]).shape == (0,)


@gpu
def test_rows_of_any_stride():
    x, u = _rows(9, 3000, torch.bfloat16, 6)
    for part in (x[:, 1:2801], x[::2, :2999], x[:1].expand(5, 3000), x[:, 3:4]):
        _check(part, u[:part.shape[0]].contiguous(), top_p=0.9)


@gpu
def test_shares():
    """Many draws of one row follow its shares: each count lies within 5 standard deviations."""
    from strict_topk_overlap_b200 import sampling
    x = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5], device=DEV).expand(20000, 5)
    u = torch.rand((20000,), generator=torch.Generator(DEV).manual_seed(7), device=DEV)
    share = torch.softmax(x[0].double() / 0.8, 0)
    count = torch.bincount(sampling.sample(x, u, temperature=0.8).long(), minlength=5).double()
    assert bool(((count - 20000 * share).abs() <= 5 * (20000 * share * (1 - share)).sqrt()).all())
