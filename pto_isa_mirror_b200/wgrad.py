"""The backward pass's use of activations kept in 8 bits: a linear layer's weight gradient."""
from __future__ import annotations

from typing import Optional

import torch

from . import _capi
from .gemm import _TORCH_TO_PTO, _device_of, _elsewhere, _raw_stream, _require_cuda_2d
from .nvfp4 import _FLOATS, _new, _ptr

_E8M0_BYTES = (torch.uint8,) + ((torch.float8_e8m0fnu,) if hasattr(torch, "float8_e8m0fnu") else ())


def _scratch_pays(t: int, n: int, k: int) -> bool:
    """Converting x once against converting it for every 256 columns of dy. Measured, us without / with scratch (T x N x K):
    16384x1024x8192 260 / 280, 16384x2048x2048 116 / 110, 2048x2048x2048 23.8 / 23.4, 1024x4096x4096 54 / 39,
    4096x4096x2048 64 / 55, 2048x8192x8192 325 / 208, 16384x8192x8192 1990 / 1720."""
    return n >= 2048 and t * n * k >= 1 << 34


def gemm_wgrad_mx(dy: torch.Tensor, data: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype = torch.float32,
                  addend: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, workspace=None,
                  stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """dW [N, K] = dy^T @ x (+ addend) for a layer y = x @ W^T whose input x [T, K] was kept as MXFP8: ``data`` [T, K] e4m3
    bytes and ``scales`` [T, K / 32] e8m0 bytes, as :func:`mx_quantize_e4m3` returns them (and :func:`gemm_mx` reads them
    in the forward pass). dy [T, N]: bfloat16 or float16, rows on 16-byte boundaries; K a multiple of 32.

    x enters as the numbers the bytes stand for, in dy's type - exact for bfloat16 down to 2^-126; float16 has its range. Sums are
    float32; dW is float32, bfloat16 or float16. ``addend`` [N, K], of dW's type, is added before the rounding; it may be
    ``out`` itself, which accumulates gradients in place.

    ``workspace``: None (default): where it makes the call faster, T x K values of dy's type are allocated through torch for
    the time of the call, into which x is converted once; False: none, x is converted tile by tile beside the products; or
    a uint8 CUDA tensor of at least 2 T K bytes, on a 32-byte boundary. The result is the same to the bit."""
    lib = _capi.load()
    for t, name in ((dy, "dy"), (data, "data"), (scales, "scales")):
        _require_cuda_2d(t, name)
    if dy.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("dy must be bfloat16 or float16")
    if data.dtype not in (torch.uint8, torch.float8_e4m3fn) or scales.dtype not in _E8M0_BYTES:
        raise ValueError("data must be e4m3 bytes (uint8 or float8_e4m3fn) and scales e8m0 bytes (uint8 or float8_e8m0fnu)")
    t, n = dy.shape
    k = data.shape[1]
    if data.shape[0] != t:
        raise ValueError("dy and data must have the same number of rows")
    if t == 0 or n == 0 or k == 0 or k % 32 != 0 or tuple(scales.shape) != (t, k // 32):
        raise ValueError("T, N and K must be positive, K a multiple of 32 and scales [T, K / 32]")
    if out is not None:
        _require_cuda_2d(out, "out")
        if out.dtype not in _FLOATS or tuple(out.shape) != (n, k):
            raise ValueError("out must be [N, K] float32, bfloat16 or float16")
        out_dtype = out.dtype
    elif out_dtype not in _FLOATS:
        raise ValueError("out_dtype must be float32, bfloat16 or float16")
    if addend is not None:
        _require_cuda_2d(addend, "addend")
        if addend.dtype != out_dtype or tuple(addend.shape) != (n, k):
            raise ValueError("addend must be [N, K] of dW's type")
    given = None
    if isinstance(workspace, torch.Tensor):
        given = workspace
        if not given.is_cuda or given.dtype != torch.uint8 or not given.is_contiguous():
            raise ValueError("workspace must be a contiguous uint8 CUDA tensor")
    elif workspace is not None and workspace is not False:
        raise ValueError("workspace must be None, False or a tensor")
    device = _device_of(dy, data, scales, addend, out, given)
    there = _elsewhere(device, stream)
    if there is not None:
        with there:
            return gemm_wgrad_mx(dy, data, scales, out_dtype, addend, out, workspace)
    if out is None:
        out = _new((n, k), (k, 1), out_dtype, dy)
    if workspace is None and _scratch_pays(t, n, k):
        given = _new((2 * t * k,), (1,), torch.uint8, dy)
    rc = lib.pto_b200_gemm_wgrad_mx(_raw_stream(device), out.data_ptr(), dy.data_ptr(), data.data_ptr(), scales.data_ptr(),
                                    _ptr(addend), _ptr(given), 0 if given is None else given.numel(), t, n, k,
                                    dy.stride()[0] if t > 1 else (n + 7) // 8 * 8,
                                    data.stride()[0] if t > 1 else (k + 15) // 16 * 16, scales.stride()[0] if t > 1 else k // 32,
                                    out.stride()[0] if n > 1 else k,
                                    0 if addend is None else addend.stride()[0] if n > 1 else k, _TORCH_TO_PTO[dy.dtype],
                                    _TORCH_TO_PTO[out_dtype])
    _capi.check(rc, "pto_b200_gemm_wgrad_mx")
    return out
