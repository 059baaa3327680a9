"""Low-precision launches beside one another: clusters whose CTAs share their SMs with another stream's work."""
import pytest
import torch

import pto_isa_mirror_b200 as pto

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def status_word_stays_clear():
    yield
    assert pto.device_status() == 0, "a kernel gave up on a bounded wait"


def test_clusters_beside_another_streams_work():
    # few-rows products cut along K (with columns past the last tile's end), one-launch quantisers over a cluster and a
    # weight gradient cut along tokens, on three streams at once: every result is that of the call alone
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((64, 4096), generator=g, device=DEV).to(torch.bfloat16)
    w = pto.nvfp4_quantize(torch.randn((1001, 4096), generator=g, device=DEV))
    dy = torch.randn((515, 1000), generator=g, device=DEV).to(torch.bfloat16)
    kept = pto.mx_quantize_e4m3(torch.randn((515, 1056), generator=g, device=DEV).to(torch.bfloat16))

    def step(stream):
        q = pto.nvfp4_quantize(x, stream=stream)
        y = pto.gemm_nvfp4(q[0][:40], w[0], q[1], w[1], q[2], w[2], stream=stream)
        one = pto.gemm_nvfp4(q[0][:1], w[0], q[1], w[1], q[2], w[2], out_dtype=torch.float32, stream=stream)
        return [*q, y, one, pto.gemm_wgrad_mx(dy, *kept, stream=stream)]

    alone = step(None)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    seen = [step(streams[i % 3]) for i in range(60)]
    torch.cuda.synchronize()
    for got in seen:
        assert all(torch.equal(a, b) for a, b in zip(alone, got))
