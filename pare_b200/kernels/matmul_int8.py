"""W8A8 linear — Python face of the integer tensor-core kernels.

The reference rounds the activations of a SmoothQuant layer to 127 steps per token and then multiplies in floats
(``quantize_inputs``, ``pare/layers/linear.py:121-138``).  :func:`w8a8_forward` multiplies the steps themselves: int8 codes with a
scale per token, int8 weights with a scale per output channel, exact 32-bit sums, one rounding at the end.
"""

from __future__ import annotations

import functools

import torch
from torch import Tensor

from pare_b200.kernels import _lib

MAX_K = 65536


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(m: int, n: int, k: int, index: int) -> int:
    with torch.cuda.device(index):
        return _lib.lib().pare_w8a8_workspace_bytes(m, n, k)


def _vector(t: Tensor | None, n: int, device, what: str) -> int | None:
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous float32 tensor [{n}] on {device}, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def w8a8_forward(x: Tensor, q_weight: Tensor, scale: Tensor, zero: Tensor | None = None, *, bias: Tensor | None = None,
                 input_scale: Tensor | None = None, out: Tensor | None = None) -> Tensor:
    """``x [M, K] @ ((q_weight - zero) * scale).T (+ bias)`` in 8-bit integers.

    Each row of ``x`` (float16 / bfloat16) gets the step ``max(|x|, 1e-6) / 127`` and becomes int8 codes, rounded half to even.
    ``q_weight`` is int8 ``[N, K]`` (rows a multiple of 16 bytes apart and 16-byte aligned; others are copied), ``scale`` and the
    optional ``zero`` float32 ``[N]``, ``input_scale`` float32 ``[K]`` divides the activations first (the quotient rounded to
    their dtype), ``bias`` ``[N]``.  ``K`` is at most 65536.  The result has the dtype of ``x``; a row of ``x`` with an infinity or
    NaN gives NaN.  ``out``: where to put it (``[M, N]``, adjacent columns, not overlapping ``x``).  No gradients.
    """
    if not x.is_cuda:
        raise RuntimeError("w8a8_forward requires CUDA tensors.")
    dtype, dev = x.dtype, x.device
    if x.dim() != 2 or (dtype is not torch.float16 and dtype is not torch.bfloat16):
        raise ValueError(f"w8a8_forward: x must be float16 or bfloat16 [M, K], got {dtype} {list(x.shape)}")
    m, k = x.shape
    if q_weight.dtype is not torch.int8 or q_weight.dim() != 2 or q_weight.shape[1] != k or q_weight.device != dev:
        raise ValueError(f"w8a8_forward: q_weight must be int8 [N, {k}] on {dev}, got {q_weight.dtype} {list(q_weight.shape)} on {q_weight.device}")
    n = q_weight.shape[0]
    if not 0 < k <= MAX_K or n == 0:
        raise ValueError(f"w8a8_forward: 1 to {MAX_K} input and at least one output feature, got {k} and {n}")
    s, z, i = _vector(scale, n, dev, "scale"), _vector(zero, n, dev, "zero"), _vector(input_scale, k, dev, "input_scale")
    if bias is not None:
        if bias.shape != (n,) or bias.device != dev:
            raise ValueError(f"bias must be [{n}] on {dev}, got {list(bias.shape)} on {bias.device}")
        if bias.dtype is not dtype or not bias.is_contiguous():
            bias = bias.to(dtype).contiguous()
    if out is None:
        out = x.new_empty(m, n)
    elif out.shape != (m, n) or out.dtype is not dtype or out.device != dev or out.stride(1) != 1 or (m > 1 and out.stride(0) < n):
        raise ValueError(f"out must be {dtype} [{m}, {n}] on {dev} with adjacent columns")
    if m == 0:
        return out
    if x.stride(1) != 1 or (m > 1 and x.stride(0) < k):
        x = x.contiguous()
    if m <= 16 and k % 8 == 0 and (x.data_ptr() % 16 or (m > 1 and x.stride(0) % 8)):     # a few rows are read in 16-byte pieces
        x = x.clone(memory_format=torch.contiguous_format)
    ldw = q_weight.stride(0) if n > 1 else -(-k // 16) * 16
    if q_weight.stride(1) != 1 or ldw < k or ldw % 16 or q_weight.data_ptr() % 16:
        q_weight = aligned_rows(q_weight)
        ldw = q_weight.stride(0)
    if dev.index != _lib.current_device():
        with torch.cuda.device(dev):
            return w8a8_forward(x, q_weight, scale, zero, bias=bias, input_scale=input_scale, out=out)
    stream, nbytes = _lib.current_stream(dev), _workspace_bytes(m, n, k, dev.index)
    ws = _lib.scratch(dev, nbytes, stream).data_ptr() if nbytes else None
    status = _lib.lib().pare_w8a8_forward(
        x.data_ptr(), 0 if dtype is torch.float16 else 1, x.stride(0) if m > 1 else k, q_weight.data_ptr(), ldw, s, z, i, _lib.ptr(bias),
        out.data_ptr(), out.stride(0) if m > 1 else n, m, n, k, ws, nbytes, stream)
    if status:
        _lib.check(status, "pare_w8a8_forward")
    return out


def aligned_rows(q_weight: Tensor) -> Tensor:
    """``q_weight [N, K]`` with rows a multiple of 16 bytes apart: itself where they are, else a copy."""
    n, k = q_weight.shape
    pitch = -(-k // 16) * 16
    if q_weight.stride() == (pitch, 1) and q_weight.data_ptr() % 16 == 0:
        return q_weight
    rows = torch.zeros(n, pitch, dtype=torch.int8, device=q_weight.device)
    rows[:, :k] = q_weight
    return rows[:, :k]
