"""Activations kept in 8 bits: the MXFP8 quantiser from 16-bit rows, and the weight gradient computed from its output.

The 16-bit quantiser has to give the bytes of the fp32 one for the same numbers, which is checked against the reference
elsewhere. Weight gradients over small whole numbers are exact in fp32 and compared for equality; over real ones the
products are exact (8 + 4 significant bits), each 16-token step of the tensor core is off by at most two units (2^-22)
of the magnitudes summed in its 1024-token part, and each part's joining by half a unit of the whole."""
import pytest
import torch

import pto_isa_mirror_b200 as pto
from pto_isa_mirror_b200 import _capi

pytestmark = pytest.mark.gpu
DEV = "cuda"
FLOATS = (torch.float32, torch.bfloat16, torch.float16)
EPS = {t: torch.finfo(t).eps / 2 for t in FLOATS}
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in FLOATS}


@pytest.fixture(autouse=True)
def status_word_stays_clear():
    yield
    assert pto.device_status() == 0, "a kernel gave up on a bounded wait"


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ quantiser

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("alg", [_capi.SCALE_OCP, _capi.SCALE_NV])
@pytest.mark.parametrize("rows,k,pitch", [(1, 32, 32), (7, 96, 104), (333, 1056, 1056), (128, 4096, 4096), (1000, 64, 72)])
def test_16bit_source_gives_the_bytes_of_float32(rows, k, pitch, alg, dtype):
    x = torch.randn((rows, pitch), generator=gen(rows + k)) * torch.exp2(torch.randint(-14, 9, (rows, 1), generator=gen(k)).float())
    x[0, :32] = 0.0
    x[rows // 2, :32] = torch.arange(32) * -(2.0 ** -12)
    x = x.to(dtype).to(DEV)[:, :k]
    data, scales = pto.mx_quantize_e4m3(x, scale_alg=alg)
    want_data, want_scales = pto.mx_quantize_e4m3(x.float().contiguous(), scale_alg=alg)
    assert torch.equal(data, want_data) and torch.equal(scales, want_scales)


@pytest.mark.parametrize("dtype", FLOATS)
def test_one_row_of_any_pitch(dtype):
    column = torch.randn((96, 1), generator=gen(3)).to(dtype).to(DEV)
    row = column.t()  # one row whose stride says nothing
    assert row.stride() == (1, 1)
    got, want = pto.mx_quantize_e4m3(row), pto.mx_quantize_e4m3(column.reshape(1, 96))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for a, b in zip(pto.nvfp4_quantize(row), pto.nvfp4_quantize(column.reshape(1, 96))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_16bit_extremes(dtype):
    every = torch.arange(0, 65536, dtype=torch.int32).to(torch.int16).view(dtype)  # every pattern there is
    fine = every[torch.isfinite(every)]
    x = torch.sort(fine.float()).values.to(dtype)[: fine.numel() // 32 * 32].view(-1, 32).to(DEV)
    data, scales = pto.mx_quantize_e4m3(x)
    want_data, want_scales = pto.mx_quantize_e4m3(x.float())
    assert torch.equal(data, want_data) and torch.equal(scales, want_scales)
    bad = torch.zeros((3, 64), dtype=dtype)
    bad[0, 3], bad[1, 40], bad[2, 31] = float("nan"), float("inf"), float("-inf")
    bad[:, 50] = 1.0
    data, scales = pto.mx_quantize_e4m3(bad.to(DEV))
    assert scales.cpu().tolist() == [[255, 119], [0, 255], [255, 119]]
    assert (data.cpu()[0, :32] == 0).all() and (data.cpu()[1, 32:] == 0).all()


# ------------------------------------------------------------------ weight gradient

def kept(t, k, seed, whole, spread=0):
    """e4m3 bytes and e8m0 scales of an activation [t, k] in wider buffers, and its values in 64 bits."""
    if whole:
        v = torch.randint(-4, 5, (t, k), generator=gen(seed)).float()
        e = torch.randint(126, 129, (t, k // 32), generator=gen(seed + 1))
    else:
        v = torch.randn((t, k), generator=gen(seed)).clamp(-3, 3) * 100
        e = torch.randint(119 - spread, 122 + spread, (t, k // 32), generator=gen(seed + 1))
    data = torch.full((t, (k + 15) // 16 * 16 + 16), 0x7F, dtype=torch.uint8)  # NaN beyond the rows
    data[:, :k] = v.to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.full((t, k // 32 + 3), 255, dtype=torch.uint8)
    scales[:, : k // 32] = e.to(torch.uint8)
    value = data[:, :k].contiguous().view(torch.float8_e4m3fn).double().view(t, -1, 32) * torch.exp2(e.double() - 127)[:, :, None]
    return data.to(DEV)[:, :k], scales.to(DEV)[:, : k // 32], value.view(t, k).to(DEV)


def pitched(x, step, extra):
    buf = torch.full((x.shape[0], (x.shape[1] + step - 1) // step * step + extra), float("nan"), dtype=x.dtype)
    buf[:, : x.shape[1]] = x
    return buf.to(DEV)[:, : x.shape[1]]


SIZES = [(1, 8, 32), (3, 1, 32), (64, 256, 256), (65, 300, 288), (130, 257, 96), (515, 1000, 1056), (2048, 128, 512),
         (2113, 513, 64), (4500, 264, 160), (9000, 100, 32), (700, 2600, 2080), (640, 9000, 1056)]


@pytest.mark.parametrize("t,n,k", SIZES)
@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                             (torch.float16, torch.float16), (torch.float16, torch.bfloat16)])
def test_whole_numbers_are_exact(t, n, k, dtype, out_dtype):
    data, scales, x = kept(t, k, t + n, True)
    dy = torch.randint(-2, 3, (t, n), generator=gen(n)).to(dtype)
    got = pto.gemm_wgrad_mx(pitched(dy, 8, 8), data, scales, out_dtype=out_dtype)
    want = dy.to(DEV).double().t() @ x  # halves of whole numbers below 2^23: exact in fp32
    assert torch.equal(got, want.to(out_dtype))


@pytest.mark.parametrize("t,n,k", [(1, 8, 32), (515, 1000, 1056), (2500, 520, 320), (16390, 256, 256), (8192, 2304, 2304)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_gradient_against_the_formula(t, n, k, dtype, out_dtype):
    data, scales, x = kept(t, k, t + n, False, spread=4)
    dy = (torch.randn((t, n), generator=gen(n)) * 0.1).abs().to(dtype)  # one sign: cut-off sums would all fall short
    addend = torch.randn((n, k), generator=gen(k)).to(out_dtype).to(DEV)
    got = pto.gemm_wgrad_mx(pitched(dy, 8, 0), data, scales, out_dtype=out_dtype, addend=addend)
    d = dy.to(DEV).double()
    want = d.t() @ x + addend.double()
    size = d.abs().t() @ x.abs() + addend.double().abs()
    steps = min(t, 1024) / 16 + 1
    bound = size * (steps * 2.0 ** -22 + (t // 1024 + 6) * 2.0 ** -24) + torch.clamp(want.abs() * EPS[out_dtype], min=TINY[out_dtype])
    if dtype == torch.float16:  # x in fp16: half a step below 2^-14
        bound = bound + 2.0 ** -25 * d.abs().sum(0)[:, None]
    off = (got.double() - want).abs()
    assert (off <= bound).all(), f"{float((off / bound).max()):.2f} of the bound"


def test_long_sums_are_rounded_not_cut():
    # 32768 terms of one sign: a single tensor-core sum falls 1.8e-4 short here; parts of 1024 joined in fp32 lose what
    # 1024 terms lose, 64 steps of half a unit on average: 64 * 2^-24
    t = 32768
    data, scales, x = kept(t, 64, 5, False)
    data, x = torch.where(data >= 128, data - 128, data).contiguous(), x.abs()
    dy = torch.randn((t, 64), generator=gen(6)).abs().to(torch.bfloat16).to(DEV)
    got = pto.gemm_wgrad_mx(dy, data, scales).double()
    want = dy.double().t() @ x
    assert float((got - want).abs().max() / want.abs().max()) <= 64 * 2.0 ** -24


def test_accumulates_in_place():
    data, scales, x = kept(300, 96, 1, True)
    dy = torch.randint(-2, 3, (300, 40), generator=gen(2)).to(torch.bfloat16).to(DEV)
    once = dy.double().t() @ x
    buf = torch.zeros((41, 100), device=DEV)
    grad = buf[:40, :96]
    for i in range(1, 4):
        assert pto.gemm_wgrad_mx(dy, data, scales, addend=grad, out=grad) is grad
        assert torch.equal(grad.double(), once * i)
    assert (buf[40] == 0).all() and (buf[:, 96:] == 0).all()


def test_every_byte_and_scale():
    # one token per row of dy's identity: dW is x itself
    t = 256
    data = torch.arange(256, dtype=torch.int32).to(torch.uint8)[:, None].repeat(1, 32).to(DEV)
    for e in (0, 1, 7, 8, 100, 127, 134, 135, 180, 238, 255):
        scales = torch.full((t, 1), e, dtype=torch.uint8, device=DEV)
        for r in range(0, t, 64):  # a quarter of the tokens at a time: a NaN times 0 is a NaN
            got = pto.gemm_wgrad_mx(torch.eye(64, dtype=torch.bfloat16, device=DEV), data[r:r + 64].contiguous(),
                                    scales[r:r + 64].contiguous())
            v = data[r:r + 64].view(torch.float8_e4m3fn).double()
            if torch.isnan(v).any() or e == 255:
                assert torch.isnan(got).all()
                continue
            want = v * 2.0 ** (e - 127)
            # bf16 has no bits below 2^-133: what is cut off there is less than one of them
            assert torch.equal(got.double(), want) if e > 9 else ((got.double() - want).abs() <= 2.0 ** -133).all()


@pytest.mark.parametrize("t,n,k", [(1, 8, 32), (130, 257, 96), (515, 1000, 1056), (4500, 264, 160), (640, 9000, 1056), (3000, 2304, 2560)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scratch_memory_changes_no_bit(t, n, k, dtype):
    data, scales, _ = kept(t, k, t + n, False, spread=40)  # scales past what the short conversion holds for
    scales[:: 7] = torch.randint(100, 150, scales[:: 7].shape, generator=gen(1), dtype=torch.uint8).to(DEV)
    dy = pitched((torch.randn((t, n), generator=gen(n)) * 0.01).to(dtype), 8, 8)
    scratch = torch.full((2 * t * k + 64,), 0xFF, dtype=torch.uint8, device=DEV)
    without = pto.gemm_wgrad_mx(dy, data, scales, workspace=False)
    assert torch.equal(without.view(torch.int32), pto.gemm_wgrad_mx(dy, data, scales, workspace=scratch[:2 * t * k]).view(torch.int32))
    assert torch.equal(without.view(torch.int32), pto.gemm_wgrad_mx(dy, data, scales).view(torch.int32))
    assert (scratch[2 * t * k:] == 0xFF).all()


def test_scratch_memory_carries_nan_and_every_byte():
    data = torch.arange(256, dtype=torch.int32).to(torch.uint8)[:, None].repeat(1, 64).to(DEV)
    eye = torch.eye(256, device=DEV)
    for e in (0, 3, 102, 103, 127, 134, 135, 142, 143, 254, 255):
        scales = torch.full((256, 2), e, dtype=torch.uint8, device=DEV)
        for dtype in (torch.bfloat16, torch.float16):
            one = pto.gemm_wgrad_mx(eye.to(dtype), data, scales, workspace=False)
            two = pto.gemm_wgrad_mx(eye.to(dtype), data, scales, workspace=torch.empty(256 * 128, dtype=torch.uint8, device=DEV))
            assert torch.equal(torch.isnan(one), torch.isnan(two)) and torch.equal(torch.nan_to_num(one), torch.nan_to_num(two))


def test_splits_and_streams_agree_bit_for_bit():
    data, scales, _ = kept(3000, 512, 9, False)
    dy = torch.randn((3000, 512), generator=gen(8)).to(torch.bfloat16).to(DEV)
    first = pto.gemm_wgrad_mx(dy, data, scales)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [pto.gemm_wgrad_mx(dy, data, scales, stream=side if i % 2 else None) for i in range(6)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_captured_and_replayed():
    data, scales, x = kept(200, 64, 3, True)
    dy = torch.randint(-2, 3, (200, 48), generator=gen(4)).to(torch.bfloat16).to(DEV)
    out = torch.empty((48, 64), device=DEV)
    pto.gemm_wgrad_mx(dy, data, scales, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pto.gemm_wgrad_mx(dy, data, scales, out=out)
    dy.mul_(2)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.double(), dy.double().t() @ x)


def test_python_refusals():
    data, scales, _ = kept(64, 64, 3, True)
    dy = torch.zeros((64, 48), dtype=torch.bfloat16, device=DEV)
    out = torch.zeros((48, 64), device=DEV)
    bad = [
        lambda: pto.gemm_wgrad_mx(dy.float(), data, scales), lambda: pto.gemm_wgrad_mx(dy[:63], data, scales),
        lambda: pto.gemm_wgrad_mx(dy.t(), data, scales), lambda: pto.gemm_wgrad_mx(dy, data[:, :48], scales),
        lambda: pto.gemm_wgrad_mx(dy, data, scales[:, :1]), lambda: pto.gemm_wgrad_mx(dy, data.float(), scales),
        lambda: pto.gemm_wgrad_mx(dy, data.view(torch.float8_e5m2), scales), lambda: pto.gemm_wgrad_mx(dy[:, :0], data, scales),
        lambda: pto.gemm_wgrad_mx(dy, data, scales, out_dtype=torch.float64), lambda: pto.gemm_wgrad_mx(dy, data, scales, out=out.t()),
        lambda: pto.gemm_wgrad_mx(dy, data, scales, out=out[:, :32]), lambda: pto.gemm_wgrad_mx(dy, data, scales, addend=out.half()),
        lambda: pto.gemm_wgrad_mx(dy, data, scales, addend=out[:40]),
        lambda: pto.gemm_wgrad_mx(dy, data, scales, workspace=True), lambda: pto.gemm_wgrad_mx(dy, data, scales, workspace=out),
        lambda: pto.mx_quantize_e4m3(dy.double()), lambda: pto.mx_quantize_e4m3(dy[:, :40]),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call in (lambda: pto.gemm_wgrad_mx(dy[:, 1:], data, scales), lambda: pto.gemm_wgrad_mx(dy, data[:, :32].as_strided((64, 32), (72, 1)), scales[:, :1])):
        with pytest.raises(pto.PtoB200Error) as e:
            call()
        assert e.value.code == 2
    with pytest.raises(pto.PtoB200Error) as e:
        pto.gemm_wgrad_mx(dy, data, scales, workspace=torch.empty(2 * 64 * 64 - 1, dtype=torch.uint8, device=DEV))
    assert e.value.code == 4


def test_rows_of_nan_and_infinity_stay_theirs():
    data, scales, x = kept(700, 96, 4, True)
    dy = pitched(torch.randint(-2, 3, (700, 70), generator=gen(5)).to(torch.bfloat16), 8, 0)
    dy[100, 3] = float("nan")
    dy[650, 60] = float("inf")
    scales[:, :1][300] = 255
    got = pto.gemm_wgrad_mx(dy, data, scales).cpu()
    bad = torch.zeros((70, 96), dtype=torch.bool)
    bad[3] = bad[60] = True
    bad[:, :32] = True
    assert not torch.isfinite(got[3]).any() and not torch.isfinite(got[:, :32]).any()
    assert torch.isfinite(got[~bad].view(-1)).all()


def test_past_two_to_the_31_elements():
    t, k, n = 66000, 32768, 16
    data = torch.zeros((t, k), dtype=torch.uint8, device=DEV)
    scales = torch.full((t, k // 32), 127, dtype=torch.uint8, device=DEV)
    data[-3:] = torch.randint(0, 0x7F, (3, k), generator=gen(1), dtype=torch.uint8).to(DEV)
    scales[-1, -1] = 129
    dy = torch.zeros((t, n), dtype=torch.bfloat16, device=DEV)
    dy[-3:] = torch.randint(-2, 3, (3, n), generator=gen(2)).to(torch.bfloat16).to(DEV)
    got = pto.gemm_wgrad_mx(dy, data, scales)
    x = data[-3:].view(torch.float8_e4m3fn).double()
    x[-1, -32:] *= 4
    assert torch.equal(got.double(), dy[-3:].double().t() @ x)  # at most 3 * 2 * 1792 in steps of 2^-9: exact


# ------------------------------------------------------------------ together: one linear layer, forward and backward

@pytest.mark.parametrize("t,n,k", [(1, 48, 96), (37, 200, 160), (700, 520, 1056), (2500, 768, 512)])
def test_a_linear_layers_step(t, n, k):
    """y = x W^T in 4 bits, x kept in 8, dx in 4 bits from the transposed weight, dW from what was kept - each against
    64 bits on the numbers that were quantised, and dW against differences of the layer's own (linear) loss."""
    import nvfp4_reference as ref

    x = torch.randn((t, k), generator=gen(1)).to(torch.bfloat16).to(DEV)
    w = (torch.randn((n, k), generator=gen(2)) * 0.05).to(torch.bfloat16).to(DEV)
    dy = (torch.randn((t, n), generator=gen(3)) * 0.1).to(torch.bfloat16).to(DEV)

    xq, wq = pto.nvfp4_quantize(x), pto.nvfp4_quantize(w)
    y = pto.gemm_nvfp4(xq[0], wq[0], xq[1], wq[1], xq[2], wq[2], out_dtype=torch.float32)
    kept_data, kept_scales = pto.mx_quantize_e4m3(x)

    wtq, dyq = pto.nvfp4_quantize(w, transpose=True), pto.nvfp4_quantize(dy)
    dx = pto.gemm_nvfp4(dyq[0], wtq[0], dyq[1], wtq[1], dyq[2], wtq[2], out_dtype=torch.float32)
    dw = pto.gemm_wgrad_mx(dy, kept_data, kept_scales)

    def number(q):
        return ref.values(q[0].cpu(), q[1].cpu()).to(DEV) * q[2].double()

    def near(got, a, b, steps):
        size = a.abs() @ b.abs().t()
        assert ((got.double() - a @ b.t()).abs() <= size * ((steps + 4) * 2.0 ** -22)).all()

    near(y, number(xq), number(wq), (k + 63) // 64)
    near(dx, number(dyq), number(wtq), (n + 63) // 64)
    x8 = kept_data.view(torch.float8_e4m3fn).double().view(t, -1, 32) * torch.exp2(kept_scales.double() - 127)[:, :, None]
    x8 = x8.view(t, k)
    near(dw, dy.double().t(), x8.t(), min(t, 1024) // 16 + 1 + t // 1024)
    # the loss sum(dy * (x8 W^T)) is linear in W: its difference along any direction is dW's product with it
    direction = torch.randn((n, k), generator=gen(4)).double().to(DEV)
    wd = w.double()
    rise = ((dy.double() * (x8 @ (wd + direction).t())).sum() - (dy.double() * (x8 @ wd.t())).sum())
    spread = (dy.double().abs().t() @ x8.abs() * direction.abs()).sum()
    assert abs(float(rise - (dw.double() * direction).sum())) <= float(spread) * (min(t, 1024) / 16 + t // 1024 + 6) * 2.0 ** -22
    # the numbers themselves lie where four and eight bits put them: half a step of e2m1 (1/4 of a value's octave or a
    # sixth of the block's largest) and of e4m3
    assert float((number(xq) - x.double()).norm() / x.double().norm()) < 0.25
    assert float((x8 - x.double()).norm() / x.double().norm()) < 2.0 ** -4


@pytest.mark.parametrize("t,n,k", [(16, 256, 512), (300, 128, 64), (200, 2048, 640)])
def test_launches_that_overlap_keep_their_order(t, n, k):
    # the same buffers written and read by one call after the other, no waiting between them; every step's results have to
    # be those of the step computed alone
    g = torch.Generator(device=DEV).manual_seed(t)
    xs = [(torch.randn((t, k), generator=g, device=DEV) * 2.0 ** i).to(torch.bfloat16) for i in range(-6, 6)]
    dys = [(torch.randn((t, n), generator=g, device=DEV) * 2.0 ** -i).to(torch.bfloat16) for i in range(-6, 6)]
    w = pto.nvfp4_quantize(torch.randn((n, k), generator=g, device=DEV))

    def step(x, dy, buffers):
        q = pto.nvfp4_quantize(x, data=buffers[0], scales=buffers[1], tensor_scale=buffers[2])
        kept = pto.mx_quantize_e4m3(x, data=buffers[3], scales=buffers[4])
        y = pto.gemm_nvfp4(q[0], w[0], q[1], w[1], q[2], w[2], out=buffers[5], out_dtype=torch.float32)
        dw = pto.gemm_wgrad_mx(dy, *kept, out=buffers[6], workspace=buffers[7])
        back = pto.nvfp4_dequantize(*q, out=buffers[8], out_dtype=torch.float32)
        return [*q, *kept, y, dw, back]

    alone = []
    for x, dy in zip(xs, dys):
        alone.append(step(x, dy, [None] * 7 + [False, None]))
        torch.cuda.synchronize()
    buffers = [v.clone() for v in alone[0]]
    buffers = buffers[:7] + [torch.empty(2 * t * k, dtype=torch.uint8, device=DEV), buffers[7]]
    x, dy = torch.empty_like(xs[0]), torch.empty_like(dys[0])
    seen = []
    for i in range(len(xs)):
        x.copy_(xs[i])
        dy.copy_(dys[i])
        seen.append([v.clone() for v in step(x, dy, buffers)])
    torch.cuda.synchronize()
    for got, want in zip(seen, alone):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
