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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", ["fused", "scratch", "default"])
@pytest.mark.parametrize("e", [0, 1, 3, 7, 9, 12, 101, 102, 103, 110, 127, 134, 135, 142, 143, 180, 200])
@pytest.mark.parametrize("broken", [False, True])
def test_every_byte_with_every_neighbour(broken, e, form, dtype):
    # dy picks out one token a row, so dW is x as the product meets it: rounded once to dy's type, whatever stands beside it
    # (a NaN or another block's scale takes a warp, or a thread, to the conversion that holds for all bytes)
    t, k = 64, 256
    byte = (torch.arange(t)[:, None] * 37 + torch.arange(k)[None, :]) % 256
    byte[(byte & 0x7F) == 0x7F] = 0x7E
    scales = torch.full((t, k // 32), e, dtype=torch.uint8)
    if broken:
        byte[5, 3], byte[40, 200] = 0x7F, 0xFF
        scales[17, 4] = 254
    data = byte.to(torch.uint8)
    x = data.view(torch.float8_e4m3fn).double().view(t, -1, 32) * torch.exp2(scales.double() - 127)[:, :, None]
    x = x.view(t, k).float().to(dtype).double()  # exact as float: at most four bits, down to 2^-136
    up = 2.0 ** 60 if dtype == torch.bfloat16 and e < 64 else 1.0  # out of the range where fp32 sums have few bits
    dy = (torch.eye(t) * up).to(dtype).to(DEV)
    workspace = {"fused": False, "scratch": torch.empty(2 * t * k, dtype=torch.uint8, device=DEV), "default": None}[form]
    got = pto.gemm_wgrad_mx(dy, data.to(DEV), scales.to(DEV), workspace=workspace).double().cpu()
    clean = torch.isfinite(x).all(0)  # an infinity or a NaN times 0 is a NaN: its column is
    assert torch.equal(got[:, clean], (x[:, clean] * up).float().double())  # fp32 ends at 2^128, where 2^60 times x may not
    assert not torch.isfinite(got[:, ~clean]).all(0).any()
    assert int(clean.sum()) > 0 or (dtype == torch.float16 and e > 134)


def test_few_rows_of_more_columns_than_a_grids_second_axis_counts():
    m, n, k = 3, 65535 * 128 + 129, 16
    g = gen(3)
    codes = torch.randint(0, 256, (2048, k // 2), generator=g, dtype=torch.uint8)  # the columns repeat these
    a = torch.zeros((m, 16), dtype=torch.uint8)
    a[:, :8] = torch.randint(0, 256, (m, k // 2), generator=g, dtype=torch.uint8)
    sfa = ref.tile_scales(torch.randint(0x30, 0x40, (m, 1), generator=g))
    sfb_rows = torch.randint(0x30, 0x40, (2048, 1), generator=g)
    tiles = ref.tile_scales(sfb_rows)
    b = torch.zeros((n, 16), dtype=torch.uint8, device=DEV)
    b[:, :8] = codes.to(DEV).repeat((n + 2047) // 2048, 1)[:n]
    sfb = tiles.to(DEV).repeat(((n + 127) // 128 + 15) // 16, 1, 1)[: (n + 127) // 128].contiguous()
    out = pto.gemm_nvfp4(a.to(DEV)[:, :8], b[:, :8], sfa.to(DEV), sfb, out_dtype=torch.float32)
    want = (ref.values(a[:, :8].contiguous(), sfa) @ ref.values(codes, tiles).t()).float().to(DEV)  # sums of 16: exact in fp32
    assert torch.equal(out, want.repeat(1, (n + 2047) // 2048)[:, :n])


def test_outputs_of_another_stream_are_not_blocks_still_in_use():
    x = torch.randn((2048, 2048), generator=gen(6)).to(torch.bfloat16).to(DEV)
    want = pto.mx_quantize_e4m3(x)
    side = torch.cuda.Stream()
    for _ in range(4):
        torch.cuda.synchronize()
        blocks = [torch.empty_like(w) for w in want]
        torch.cuda._sleep(20_000_000)  # the current stream is busy for some ten milliseconds
        for b in blocks:
            b.fill_(0x55)  # and still to write these
        del blocks, b
        got = pto.mx_quantize_e4m3(x, stream=side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_of_maxima_and_widths():
    x = torch.randn((8, 64), generator=gen(7)).to(DEV)
    place = torch.ones(1, device=DEV)
    with pytest.raises(ValueError):
        pto.nvfp4_quantize(x, amax=place, tensor_scale=place)
    data, scales, g = pto.nvfp4_quantize(x[:1])
    for width in (1, 3, 12, 28):
        with pytest.raises(ValueError):
            pto.nvfp4_dequantize(data[:, :width], scales, g)
    assert torch.equal(pto.nvfp4_dequantize(data[:, :24], scales, g), pto.nvfp4_dequantize(data, scales, g)[:, :48])


@pytest.mark.parametrize("one_sign", [False, True])
@pytest.mark.parametrize("m,n,k", [(16, 256, 16384), (300, 520, 16400), (1500, 2700, 16384), (40, 384, 65552), (300, 2048, 65536)])
def test_products_over_as_many_tokens_as_a_batch_has(m, n, k, one_sign):
    # what a backward product contracts over; the tensor core's sums are off by at most two units (2^-22) a 64-element step
    g = gen(m + k)
    sides = []
    for rows in (m, n):
        codes = torch.randint(0, 256, (rows, k // 2), generator=g, dtype=torch.uint8)
        codes = codes & 0x77 if one_sign else codes
        tiles = ref.tile_scales(torch.randint(0x20, 0x58, (rows, k // 16), generator=g))
        rows16 = torch.zeros((rows, (k + 31) // 32 * 16), dtype=torch.uint8)  # rows on 16-byte boundaries
        rows16[:, :k // 2] = codes
        sides.append((rows16.to(DEV)[:, :k // 2], tiles.to(DEV), ref.values(codes, tiles).to(DEV)))
    (a, sfa, va), (b, sfb, vb) = sides
    got = pto.gemm_nvfp4(a, b, sfa, sfb, out_dtype=torch.float32).double()
    want, size = va @ vb.t(), va.abs() @ vb.abs().t()
    bound = size * (((k + 63) // 64) * 2.0 ** -22 + 4 * 2.0 ** -24)
    assert ((got - want).abs() <= bound).all()
