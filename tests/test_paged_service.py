"""The example service runs its operators together: two attention forms of the
same tokens agree to the output's rounding (bf16, twice 2^-8 of values up to
about 1, and their weights' roundings of the same size)."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest


@pytest.mark.gpu
@pytest.mark.parametrize("requests,system,steps", [(8, 1024, 4), (3, 64, 2), (1, 320, 1)])
def test_service(requests, system, steps):
    path = Path(__file__).resolve().parent.parent / "examples" / "paged_service.py"
    spec = importlib.util.spec_from_file_location("paged_service", path)
    service = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(service)
    assert service.serve(requests, system, steps, say=lambda *_: None) <= 4 * 2.0 ** -8
