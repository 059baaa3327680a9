"""Refusals of the NVFP4 operators, the 16-bit MX quantiser and the weight gradient: the C ABI answers with a code before it
touches a device, the Python entry points raise on what a pointer cannot say."""
import ctypes

import pytest
import torch

import pto_isa_mirror_b200 as pto
from pto_isa_mirror_b200 import _capi, build

EINVAL, EALIGN, EDTYPE = _capi.EINVAL, _capi.EALIGN, _capi.EDTYPE
F16, BF16, F32, S8, E4M3 = _capi.F16, _capi.BF16, _capi.F32, _capi.S8, _capi.E4M3


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_uint8 * 4096)()
    address = (ctypes.addressof(buf) + 63) & ~63
    yield address
    del buf


def refused(fn, good, changes):
    """`fn(**good)` with each change is refused with the code beside it."""
    for change, code in changes:
        args = dict(good)
        args.update(change)
        assert fn(*args.values()) == code, change


def test_quantize_refusals(lib, p):
    before = lib.pto_b200_launch_count()
    good = dict(stream=None, data=p, scales=p, tensor_scale=p, src=p, amax=p, rows=4, k=64, ld_src=64, ld_data=32, dtype=BF16,
                transpose=0)
    refused(lib.pto_b200_nvfp4_quantize, good, [
        (dict(data=None), EINVAL), (dict(scales=None), EINVAL), (dict(tensor_scale=None), EINVAL), (dict(src=None), EINVAL),
        (dict(amax=None), EINVAL), (dict(rows=0), EINVAL), (dict(k=0), EINVAL), (dict(ld_src=63), EINVAL),
        (dict(ld_data=24), EINVAL), (dict(k=0x7FFFFFFF, ld_src=1 << 32, ld_data=1 << 32), EINVAL),
        (dict(transpose=1, rows=65), EINVAL),              # five blocks of sixteen along the result's rows
        (dict(dtype=S8), EDTYPE), (dict(dtype=E4M3), EDTYPE),
        (dict(src=p + 1), EALIGN), (dict(data=p + 4), EALIGN), (dict(ld_data=36), EALIGN), (dict(scales=p + 2), EALIGN),
        (dict(tensor_scale=p + 2), EALIGN), (dict(amax=p + 1), EALIGN), (dict(dtype=F32, src=p + 2), EALIGN),
    ])
    good = dict(stream=None, data=p, scales=p, tensor_scale=p, amax=p, src=p, rows=4, k=64, ld_src=64, ld_data=32, dtype=BF16,
                transpose=0)
    refused(lib.pto_b200_nvfp4_quantize_dynamic, good, [
        (dict(data=None), EINVAL), (dict(scales=None), EINVAL), (dict(tensor_scale=None), EINVAL), (dict(src=None), EINVAL),
        (dict(amax=None), EINVAL), (dict(rows=0), EINVAL), (dict(k=-1), EINVAL), (dict(ld_src=63), EINVAL),
        (dict(ld_data=24), EINVAL), (dict(rows=1 << 20, ld_data=24), EINVAL), (dict(transpose=1, rows=65), EINVAL),
        (dict(dtype=S8), EDTYPE), (dict(src=p + 1), EALIGN), (dict(data=p + 4), EALIGN), (dict(scales=p + 2), EALIGN),
        (dict(tensor_scale=p + 2), EALIGN), (dict(amax=p + 1), EALIGN), (dict(rows=1 << 20, amax=p + 2), EALIGN)])
    good = dict(stream=None, amax=p, src=p, rows=4, k=64, ld_src=64, dtype=F32)
    refused(lib.pto_b200_amax, good, [(dict(amax=None), EINVAL), (dict(src=None), EINVAL), (dict(rows=-1), EINVAL),
                                      (dict(ld_src=8), EINVAL), (dict(dtype=S8), EDTYPE), (dict(src=p + 2), EALIGN),
                                      (dict(amax=p + 2), EALIGN)])
    good = dict(stream=None, out=p, data=p, scales=p, g=None, rows=4, k=64, ld_data=32, ld_out=64, dtype=F16)
    refused(lib.pto_b200_nvfp4_dequantize, good, [
        (dict(out=None), EINVAL), (dict(data=None), EINVAL), (dict(scales=None), EINVAL), (dict(rows=0), EINVAL),
        (dict(ld_data=28), EINVAL), (dict(ld_out=63), EINVAL), (dict(dtype=S8), EDTYPE), (dict(out=p + 1), EALIGN),
        (dict(data=p + 2), EALIGN), (dict(ld_data=34), EALIGN), (dict(g=p + 2), EALIGN)])
    assert lib.pto_b200_nvfp4_scale_bytes(0, 64) == 0 and lib.pto_b200_nvfp4_scale_bytes(129, 65) == 4 * 512
    assert lib.pto_b200_launch_count() == before


def test_product_refusals(lib, p):
    before = lib.pto_b200_launch_count()
    good = dict(stream=None, out=p, a=p, b=p, sfa=p, sfb=p, ga=None, gb=None, bias=None, m=16, n=16, k=64, lda=64, ldb=64, ldc=16,
                dtype=BF16)
    refused(lib.pto_b200_gemm_nvfp4, good, [
        (dict(out=None), EINVAL), (dict(a=None), EINVAL), (dict(b=None), EINVAL), (dict(sfa=None), EINVAL),
        (dict(sfb=None), EINVAL), (dict(m=0), EINVAL), (dict(n=0), EINVAL), (dict(k=0), EINVAL), (dict(k=56), EINVAL),
        (dict(lda=32), EINVAL), (dict(ldb=32), EINVAL), (dict(ldc=15), EINVAL), (dict(dtype=S8), EDTYPE),
        (dict(a=p + 8), EALIGN), (dict(b=p + 8), EALIGN), (dict(lda=80), EALIGN), (dict(ldb=80), EALIGN), (dict(sfa=p + 8), EALIGN),
        (dict(sfb=p + 8), EALIGN), (dict(out=p + 1), EALIGN), (dict(out=p + 2, dtype=F32), EALIGN), (dict(ga=p + 2), EALIGN),
        (dict(gb=p + 1), EALIGN), (dict(bias=p + 2), EALIGN)])
    assert lib.pto_b200_launch_count() == before


def test_checkpoint_refusals(lib, p):
    before = lib.pto_b200_launch_count()
    good = dict(stream=None, data=p, scales=p, src=p, rows=4, k=64, ld_src=64, ld_data=64, ld_scales=2, dtype=BF16, alg=0)
    refused(lib.pto_b200_mx_quantize_e4m3_src, good, [
        (dict(data=None), EINVAL), (dict(scales=None), EINVAL), (dict(src=None), EINVAL), (dict(rows=0), EINVAL),
        (dict(k=48), EINVAL), (dict(ld_src=32), EINVAL), (dict(ld_data=32), EINVAL), (dict(ld_scales=1), EINVAL),
        (dict(dtype=S8), EDTYPE), (dict(alg=2), EDTYPE), (dict(src=p + 8), EALIGN), (dict(ld_src=68), EALIGN),
        (dict(data=p + 4), EALIGN), (dict(ld_data=68), EALIGN), (dict(dtype=F32, src=p + 8), EALIGN)])
    good = dict(stream=None, out=p, dy=p, data=p, scales=p, addend=None, workspace=None, workspace_bytes=0, t=4, n=16, k=64, ld_dy=16, ld_data=64, ld_scales=2,
                ld_out=64, ld_addend=0, dy_dtype=BF16, out_dtype=F32)
    refused(lib.pto_b200_gemm_wgrad_mx, good, [
        (dict(out=None), EINVAL), (dict(dy=None), EINVAL), (dict(data=None), EINVAL), (dict(scales=None), EINVAL),
        (dict(t=0), EINVAL), (dict(n=0), EINVAL), (dict(k=0), EINVAL), (dict(k=48), EINVAL), (dict(ld_dy=8), EINVAL),
        (dict(ld_data=48), EINVAL), (dict(ld_scales=1), EINVAL), (dict(ld_scales=1 << 26), EINVAL), (dict(ld_out=63), EINVAL),
        (dict(addend=p, ld_addend=32), EINVAL), (dict(dy_dtype=F32), EDTYPE), (dict(dy_dtype=E4M3), EDTYPE),
        (dict(out_dtype=S8), EDTYPE), (dict(dy=p + 8), EALIGN), (dict(ld_dy=20), EALIGN), (dict(data=p + 8), EALIGN),
        (dict(ld_data=72), EALIGN), (dict(out=p + 2), EALIGN), (dict(addend=p + 2, ld_addend=64), EALIGN),
        (dict(workspace=p, workspace_bytes=511), _capi.EWORKSPACE), (dict(workspace=p + 16, workspace_bytes=4096), _capi.EWORKSPACE)])
    assert lib.pto_b200_launch_count() == before


@pytest.mark.parametrize("call", [
    lambda x, u, s: pto.nvfp4_quantize(x),
    lambda x, u, s: pto.nvfp4_dequantize(u, s),
    lambda x, u, s: pto.gemm_nvfp4(u, u, s, s),
    lambda x, u, s: pto.mx_quantize_e4m3(x),
    lambda x, u, s: pto.gemm_wgrad_mx(x, u, s),
])
def test_host_tensors_are_refused(lib, call):
    with pytest.raises(ValueError, match="CUDA"):
        call(torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((1, 1, 512), dtype=torch.uint8))
