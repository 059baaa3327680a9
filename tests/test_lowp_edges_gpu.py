"""Edges of the low-precision operators: maxima gone wrong, bits that depend on nobody's neighbours, sizes past a grid's
second axis, calls on other streams, every byte of a kept activation."""
import pytest
import torch

import nvfp4_reference as ref
import pto_isa_mirror_b200 as pto

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def status_word_stays_clear():
    yield
    assert pto.device_status() == 0, "a kernel gave up on a bounded wait"


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), -float("inf")])
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("rows,k", [(3, 64), (300, 208)])
def test_a_maximum_gone_wrong_stays_visible(rows, k, transpose, bad):
    x = torch.randn((rows, k), generator=gen(1)).to(DEV)
    data, scales, g = pto.nvfp4_quantize(x, amax=torch.tensor([bad], device=DEV), transpose=transpose)
    assert torch.isnan(g).all()
    assert torch.isnan(pto.nvfp4_dequantize(data, scales, g)).all()
    out = pto.gemm_nvfp4(data, data, scales, scales, g, g, out_dtype=torch.float32)
    assert torch.isnan(out).all()
    # the maximum found in the call is that of the numbers there are
    x[0, 5] = bad
    found = pto.nvfp4_quantize(x, transpose=transpose)[2]
    assert float(found) == ref.power_of_two_scale(float(x[torch.isfinite(x)].abs().max()))
