"""Waits of the low-precision kernels that run out: the limit is lowered until ordinary waits exceed it, in some lanes of a
warp and not in others. The kernel returns and says so in the status word, and the next calls are right."""
import ctypes

import pytest
import torch

import pto_isa_mirror_b200 as pto
from pto_isa_mirror_b200 import _capi

pytestmark = pytest.mark.gpu
DEV = "cuda"


def product(m, n, k):
    g = torch.Generator(device=DEV).manual_seed(m)
    a, b = (pto.nvfp4_quantize(torch.randn((r, k), generator=g, device=DEV)) for r in (m, n))
    return lambda: pto.gemm_nvfp4(a[0], b[0], a[1], b[1], a[2], b[2])


def gradient(t, n, k, workspace):
    g = torch.Generator(device=DEV).manual_seed(t)
    dy = torch.randn((t, n), generator=g, device=DEV).to(torch.bfloat16)
    kept = pto.mx_quantize_e4m3(torch.randn((t, k), generator=g, device=DEV))
    scratch = torch.empty(2 * t * k, dtype=torch.uint8, device=DEV) if workspace else False
    return lambda: pto.gemm_wgrad_mx(dy, *kept, workspace=scratch)


@pytest.mark.parametrize("call,codes", [
    (lambda: product(8, 600, 16384), (21, 22, 23)),         # a cluster along K
    (lambda: product(100, 40000, 16384), (21, 22, 23)),     # without
    (lambda: product(2600, 2700, 16384), (21, 22, 23)),     # pairs, several tiles each
    (lambda: gradient(9000, 512, 512, False), (31, 32, 33)),  # a cluster along the tokens
    (lambda: gradient(9000, 2600, 2816, False), (31, 32, 33)),
    (lambda: gradient(9000, 2600, 2816, True), (31, 32, 33)),
])
def test_a_wait_that_runs_out_is_reported_and_passes(call, codes):
    lib = _capi.load()
    run = call()
    want = run()
    torch.cuda.synchronize()
    assert pto.device_status() == 0
    seen = ctypes.c_int(0)
    old = lib.pto_b200_set_wait_limit(1)
    try:
        for _ in range(20):
            run()
            rc = lib.pto_b200_device_status(ctypes.byref(seen))  # waits for the launch, reads the word and clears it
            assert (rc, seen.value) == (_capi.OK, 0) or (rc == _capi.ETIMEOUT and seen.value in codes)
    finally:
        lib.pto_b200_set_wait_limit(old)
    for _ in range(3):
        assert torch.equal(run(), want)
    assert pto.device_status() == 0
