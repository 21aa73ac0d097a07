"""The next tokens from their logits and given uniform numbers.

``sample`` (stk_sample_tokens) applies temperature, top-k, top-p and min-p and
draws, in one launch, with the strict Top-K of this library: ties go to the
lower token, and masses are summed exactly, so that the same logits and numbers
give the same tokens on every run. New: the reference ends at the attention's
output.
"""
from __future__ import annotations

import torch

from . import _lib as L


def _parameter(x, name, rows, index, dtype):
    """Address of a parameter's values [R], or None, and its one value for all rows."""
    if isinstance(x, torch.Tensor):
        if x.dtype is not dtype or x.shape != (rows,) or x.get_device() != index or not x.is_contiguous():
            raise ValueError(f"{name} must be a number or contiguous {dtype} [R] on the logits' device")
        return x.data_ptr(), 0
    if not x >= 0:
        raise ValueError(f"{name} must not be negative")
    return None, x


def sample(logits, uniforms, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
    """One token for each row of ``logits`` [R, V] (f32, f16 or bf16, unit stride
    along V, at most 393,216 of them), drawn by ``uniforms`` FP32 [R] in [0, 1).
    Of the tokens in descending order of logits stay the first ``top_k`` (0:
    all), of those the ones before which less than ``top_p`` of their mass
    exp(logit / ``temperature``) lies, of those the ones of at least ``min_p``
    times the largest mass; the uniform number picks one of these in the
    vocabulary's order. ``temperature`` 0 takes the largest logit. Each parameter
    is a number or a tensor [R] (FP32; ``top_k`` int32). NaN logits are never
    chosen; a row without a logit above -inf gives -1. Returns int32 [R]
    (``out``)."""
    if logits.ndim != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be [R, V] with V > 0")
    rows, v = logits.shape
    index = logits.get_device()
    if index < 0:
        raise ValueError("logits must be on a CUDA device; there is no CPU fallback")
    stride, unit = logits.stride()
    if unit != 1 and v > 1:
        raise ValueError("logits must have unit stride along V")
    dtype = L.dtype_code(logits)
    if uniforms.dtype is not torch.float32 or uniforms.shape != (rows,) or uniforms.get_device() != index or \
            not uniforms.is_contiguous():
        raise ValueError("uniforms must be contiguous FP32 [R] on the logits' device")
    ts, t = _parameter(temperature, "temperature", rows, index, torch.float32)
    ks, k = _parameter(top_k, "top_k", rows, index, torch.int32)
    ps, p = _parameter(top_p, "top_p", rows, index, torch.float32)
    ms, m = _parameter(min_p, "min_p", rows, index, torch.float32)
    if out is None:
        out = uniforms.new_empty((rows,), dtype=torch.int32)
    elif out.dtype is not torch.int32 or out.shape != (rows,) or out.get_device() != index or not out.is_contiguous():
        raise ValueError("out must be contiguous int32 [R] on the logits' device")
    rc = L.on_device(index, L.load().stk_sample_tokens, logits.data_ptr(), dtype, stride, rows, v, uniforms.data_ptr(), ts,
                     t, ks, min(int(k), v), ps, p, ms, m, out.data_ptr(), L.status_ptr(), L.raw_stream(index))
    if rc:
        L.check(rc, "sample")
    return out
