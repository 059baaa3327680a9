"""NVFP4 (two-level 4-bit floating point): quantise, back to numbers, multiply.

A tensor in NVFP4 is three buffers: packed e2m1 codes (two per byte, the even element low), one e4m3 scale per 16
elements of a row, and one fp32 scale for the whole tensor; an element stands for code * scale * tensor scale. The
scales are held in 512-byte tiles of 128 rows x 4 scales - ``[ceil(rows / 128), ceil(K / 64), 512]``, scale j of row r
of a tile at byte ``(r % 32) * 16 + r // 32 * 4 + j`` - which is how the tensor cores read them; bytes that only pad a
tile are zero. Row-major scales ``s [rows, K / 16]`` from elsewhere, padded with zeros to multiples of 128 and 4, become
tiles by ``s.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(rt, kt, 512)``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _capi
from .gemm import _TORCH_TO_PTO, _device_of, _elsewhere, _raw_stream, _require_cuda_2d

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
# what packed codes and scale bytes may come as
_CODES = (torch.uint8, torch.int8) + ((torch.float4_e2m1fn_x2,) if hasattr(torch, "float4_e2m1fn_x2") else ())
_E4M3_BYTES = (torch.uint8, torch.float8_e4m3fn)


def _require_float_scalar(t: Optional[torch.Tensor], name: str) -> None:
    if t is not None and (t.dtype is not torch.float32 or not t.is_cuda or t.numel() != 1):
        raise ValueError(f"{name} must be a CUDA float32 tensor with one element")


def _tiles(rows: int, k: int) -> Tuple[int, int, int]:
    return (rows + 127) // 128, (k + 63) // 64, 512


def _require_scales(t: torch.Tensor, rows: int, k: int, name: str) -> None:
    if not t.is_cuda or t.dtype not in _E4M3_BYTES or not t.is_contiguous() or t.shape != _tiles(rows, k):
        raise ValueError(f"{name} must be contiguous CUDA scale tiles of shape {_tiles(rows, k)}, uint8 or float8_e4m3fn")


def _new(size, stride, dtype: torch.dtype, like: torch.Tensor) -> torch.Tensor:
    """An uninitialised tensor on ``like``'s device (half the time of ``torch.empty``)."""
    return like.new_empty_strided(size, stride, dtype=dtype)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def nvfp4_quantize(src: torch.Tensor, amax: Optional[torch.Tensor] = None, transpose: bool = False,
                   data: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None,
                   tensor_scale: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
    """Quantise src [rows, K] (float32, bfloat16 or float16; any row pitch) to NVFP4. Returns (data [rows, K16 / 2] uint8,
    scales [ceil(rows / 128), ceil(K / 64), 512] uint8, tensor_scale [1] float32), K16 = K rounded up to 16 with zeros:
    the operands :func:`gemm_nvfp4` takes.

    tensor_scale: the smallest power of two >= amax / 2688 (1 for amax = 0). ``amax``: one float32 on the device, not
    negative, for a largest magnitude known from calibration (what exceeds it saturates; from an infinite or NaN one
    tensor_scale is NaN, and so is every number that uses it); without it the largest finite magnitude of src is found first: in the same launch for small sources, in a pass of its own for others. Block scale: the e4m3 value nearest to
    max|x| / (6 tensor_scale), at most 448; code: the e2m1 value nearest to x / (scale tensor_scale), ties to the even
    code, at most 6 in magnitude. A block with an infinity or a NaN gets the scale NaN.

    ``transpose``: quantise src's transpose instead, blocks running along src's rows: data [K, rows16 / 2] and so on, the
    form the products of a backward pass contract over. ``data`` / ``scales`` / ``tensor_scale``: the caller's output
    buffers (data's rows may be padded; a pitch that is a multiple of 16 bytes is what :func:`gemm_nvfp4` needs)."""
    lib = _capi.load()
    _require_cuda_2d(src, "src")
    if src.dtype not in _FLOATS:
        raise ValueError("src must be float32, bfloat16 or float16")
    _require_float_scalar(amax, "amax")
    _require_float_scalar(tensor_scale, "tensor_scale")
    if amax is not None and tensor_scale is not None and amax.data_ptr() == tensor_scale.data_ptr():
        raise ValueError("tensor_scale must not be amax itself")
    rows, k = src.shape
    if rows == 0 or k == 0:
        raise ValueError("src must not be empty")
    out_rows, length = (k, rows) if transpose else (rows, k)
    width = (length + 15) // 16 * 8
    if data is not None:
        _require_cuda_2d(data, "data")
        if data.dtype != torch.uint8 or tuple(data.shape) != (out_rows, width):
            raise ValueError(f"data must be uint8 of shape {(out_rows, width)}")
    if scales is not None:
        _require_scales(scales, out_rows, length, "scales")
    device = _device_of(src, amax, data, scales, tensor_scale)
    there = _elsewhere(device, stream)
    if there is not None:
        with there:
            return nvfp4_quantize(src, amax, transpose, data, scales, tensor_scale)
    sp = _raw_stream(device)
    pitch = (width + 15) // 16 * 16  # TMA rows start on 16-byte boundaries
    src_pitch = src.stride()[0] if rows > 1 else k
    dtype = _TORCH_TO_PTO[src.dtype]
    if data is None:
        data = _new((out_rows, width), (pitch, 1), torch.uint8, src)
    if scales is None:
        tiles = _tiles(out_rows, length)
        scales = _new(tiles, (tiles[1] * 512, 512, 1), torch.uint8, src)
    if tensor_scale is None:
        tensor_scale = _new((1,), (1,), torch.float32, src)
    out_pitch = data.stride()[0] if out_rows > 1 else pitch
    if amax is None:
        amax = _new((1,), (1,), torch.float32, src)
        rc = lib.pto_b200_nvfp4_quantize_dynamic(sp, data.data_ptr(), scales.data_ptr(), tensor_scale.data_ptr(),
                                                 amax.data_ptr(), src.data_ptr(), rows, k, src_pitch, out_pitch, dtype,
                                                 1 if transpose else 0)
        _capi.check(rc, "pto_b200_nvfp4_quantize_dynamic")
        return data, scales, tensor_scale
    rc = lib.pto_b200_nvfp4_quantize(sp, data.data_ptr(), scales.data_ptr(), tensor_scale.data_ptr(), src.data_ptr(),
                                     amax.data_ptr(), rows, k, src_pitch, out_pitch, dtype, 1 if transpose else 0)
    _capi.check(rc, "pto_b200_nvfp4_quantize")
    return data, scales, tensor_scale


def nvfp4_dequantize(data: torch.Tensor, scales: torch.Tensor, tensor_scale: Optional[torch.Tensor] = None,
                     out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None,
                     stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """The numbers [rows, K] that packed codes data [rows, K / 2] with their scale tiles stand for, K a multiple of 16: code *
    scale * tensor_scale (None: 1), float32, bfloat16 or float16. Exact before the output's own rounding when tensor_scale is a
    power of two. ``out`` may lack up to 15 of the last columns, those that filled up the last block."""
    lib = _capi.load()
    _require_cuda_2d(data, "data")
    if data.dtype not in _CODES:
        raise ValueError("data must be packed codes, uint8")
    rows, k = data.shape[0], data.shape[1] * 2
    if rows == 0 or k == 0 or k % 16 != 0:
        raise ValueError("data must hold whole blocks of 16 codes, 8 bytes each, and not be empty")
    _require_scales(scales, rows, k, "scales")
    _require_float_scalar(tensor_scale, "tensor_scale")
    if out is not None:
        _require_cuda_2d(out, "out")
        if out.dtype not in _FLOATS or out.shape[0] != rows or not k - 16 < out.shape[1] <= k:
            raise ValueError("out must be [rows, K] float32, bfloat16 or float16, K less at most the last 15 columns")
    elif out_dtype not in _FLOATS:
        raise ValueError("out_dtype must be float32, bfloat16 or float16")
    device = _device_of(data, scales, tensor_scale, out)
    there = _elsewhere(device, stream)
    if there is not None:
        with there:
            return nvfp4_dequantize(data, scales, tensor_scale, out_dtype, out)
    if out is None:
        out = _new((rows, k), (k, 1), out_dtype, data)
    cols = out.shape[1]
    rc = lib.pto_b200_nvfp4_dequantize(_raw_stream(device), out.data_ptr(), data.data_ptr(), scales.data_ptr(),
                                       _ptr(tensor_scale), rows, cols,
                                       data.stride()[0] if rows > 1 else k // 2,
                                       out.stride()[0] if rows > 1 else cols, _TORCH_TO_PTO[out.dtype])
    _capi.check(rc, "pto_b200_nvfp4_dequantize")
    return out


def gemm_nvfp4(a: torch.Tensor, b_dn: torch.Tensor, sfa: torch.Tensor, sfb: torch.Tensor, ga: Optional[torch.Tensor] = None,
               gb: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16,
               bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """C = ga gb (A @ B) (+ bias) of NVFP4 matrices: a [M, K / 2] and b_dn [N, K / 2] packed codes, sfa and sfb their scale
    tiles, ga and gb their tensor scales (one float32 each on the device; None: 1), as :func:`nvfp4_quantize` returns
    them. K is a multiple of 16; rows start on 16-byte boundaries. fp32 accumulation, then times ga gb, which is
    formed first, in fp32; C is float32, bfloat16 or float16.
    ``bias``: n float32 values added per column before the store's rounding. Any M: few rows take a kernel that reads B at
    memory speed, many rows one of 256 x 256 tiles on pairs of SMs."""
    lib = _capi.load()
    for t, name in ((a, "a"), (b_dn, "b_dn")):
        _require_cuda_2d(t, name)
        if t.dtype not in _CODES:
            raise ValueError(f"{name} must be packed codes, uint8")
    m, n, k = a.shape[0], b_dn.shape[0], a.shape[1] * 2
    if b_dn.shape[1] * 2 != k:
        raise ValueError("inner dimensions differ")
    if m == 0 or n == 0 or k == 0 or k % 16 != 0:
        raise ValueError("M, N and K must be positive and K a multiple of 16")
    _require_scales(sfa, m, k, "sfa")
    _require_scales(sfb, n, k, "sfb")
    _require_float_scalar(ga, "ga")
    _require_float_scalar(gb, "gb")
    if bias is not None and (bias.dtype != torch.float32 or not bias.is_cuda or bias.numel() != n or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous CUDA float32 tensor with {n} elements")
    if out is not None:
        _require_cuda_2d(out, "out")
        if out.dtype not in _FLOATS or tuple(out.shape) != (m, n):
            raise ValueError("out must be [M, N] float32, bfloat16 or float16")
    elif out_dtype not in _FLOATS:
        raise ValueError("out_dtype must be float32, bfloat16 or float16")
    device = _device_of(a, b_dn, sfa, sfb, ga, gb, bias, out)
    there = _elsewhere(device, stream)
    if there is not None:
        with there:
            return gemm_nvfp4(a, b_dn, sfa, sfb, ga, gb, out_dtype, bias, out)
    if out is None:
        out = _new((m, n), (n, 1), out_dtype, a)
    row = (k // 2 + 15) // 16 * 32  # a single row's pitch, in 4-bit elements
    rc = lib.pto_b200_gemm_nvfp4(_raw_stream(device), out.data_ptr(), a.data_ptr(), b_dn.data_ptr(), sfa.data_ptr(),
                                 sfb.data_ptr(), _ptr(ga), _ptr(gb), _ptr(bias), m, n, k,
                                 a.stride()[0] * 2 if m > 1 else row, b_dn.stride()[0] * 2 if n > 1 else row,
                                 out.stride()[0] if m > 1 else n, _TORCH_TO_PTO[out.dtype])
    _capi.check(rc, "pto_b200_gemm_nvfp4")
    return out
