"""NVFP4 quantiser, dequantiser and product against their definition in 64 bits.

Quantised bytes and scales are those of exact arithmetic, so they are compared for equality. A product of two elements
and their scales is exact in fp32 (4 + 8 significant bits); the sums are not: one instruction adds 64 products to the
accumulator, each such step off by at most two units (2^-22) of the magnitudes added so far, then one rounding each for
the tensor scales and the bias, and half a step of the output's type."""
import numpy as np
import pytest
import torch

import nvfp4_reference as ref
import pto_isa_mirror_b200 as pto

pytestmark = pytest.mark.gpu
DEV = "cuda"
FLOATS = (torch.float32, torch.bfloat16, torch.float16)
EPS = {t: torch.finfo(t).eps / 2 for t in FLOATS}                              # half a step, relative to a normal value
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in FLOATS}  # half a step below those: f16 2^-25


@pytest.fixture(autouse=True)
def status_word_stays_clear():
    yield
    assert pto.device_status() == 0, "a kernel gave up on a bounded wait"


def wide(rows, cols, dtype, seed, pitch=None, offset=0):
    """Values over many binades with whole blocks of zeros and many ties, in rows of `pitch` elements."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * torch.exp2(torch.randint(-9, 5, (rows, (cols + 15) // 16), generator=g).float()
                                                            ).repeat_interleave(16, 1)[:, :cols]
    x[torch.rand((rows, cols), generator=g) < 0.1] = 0.0
    coarse = torch.rand((rows, cols), generator=g) < 0.3
    x = torch.where(coarse, torch.round(x * 4) / 4, x)
    if cols > 40:
        x[0, 16:32] = 0.0
    pitch = pitch or cols
    buf = torch.full((rows * pitch + offset + 64,), 7.0, dtype=dtype)
    view = buf[offset:offset + rows * pitch].view(rows, pitch)[:, :cols]
    view.copy_(x.to(dtype))
    dev = buf.to(DEV)
    return dev[offset:offset + rows * pitch].view(rows, pitch)[:, :cols], view.float()


def check_quantized(got, want_codes, want_scales, g, rows):
    data, scales, tensor_scale = got
    assert float(tensor_scale) == g
    assert torch.equal(ref.unpack(data.cpu()) & 7, want_codes & 7)
    signs = ref.unpack(data.cpu()) >> 3
    nonzero = (want_codes & 7) != 0
    assert torch.equal(signs[nonzero], (want_codes >> 3)[nonzero])
    assert torch.equal(scales.cpu(), ref.tile_scales(want_scales))  # padding included


SHAPES = [(1, 16, None, 0), (1, 1, None, 0), (3, 17, 19, 1), (130, 100, 104, 0), (128, 64, None, 0), (257, 1040, 1041, 3),
          (5, 4096, None, 0), (600, 200, 208, 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("rows,cols,pitch,offset", SHAPES)
def test_quantize_is_exact(rows, cols, pitch, offset, transpose, dtype):
    x, host = wide(rows, cols, dtype, 5 * rows + cols, pitch, offset)
    want = ref.quantize(host.t() if transpose else host)
    check_quantized(pto.nvfp4_quantize(x, transpose=transpose), *want, rows)


# blocks of 16 in one launch: within CTAs of 256 to 1024 threads, one to eight of them, once and twice over, and one more than fits
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(16, 1024), (17, 1024), (1, 20000), (33, 1009), (64, 4096), (3, 65536), (128, 2048), (1024, 255),
                                       (1025, 256), (1, 262144), (1, 262208), (4096, 3), (4097, 3)])
def test_one_launch_and_two_agree(rows, cols, dtype):
    x, host = wide(rows, cols, dtype, rows + cols)
    x[rows // 2, cols // 2] = float("inf")  # its block only
    x[rows - 1, cols - 1] = -100.0 if rows * cols > 3 else 1.0
    amax = x.float().abs()
    amax = amax[torch.isfinite(amax)].max().reshape(1)
    before = pto.launch_count()
    got = pto.nvfp4_quantize(x)
    assert pto.launch_count() - before == (1 if rows * ((cols + 63) // 64) * 4 <= 16384 else 2)
    for a, b in zip(got, pto.nvfp4_quantize(x, amax=amax)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("transpose", [False, True])
def test_quantize_ties_and_borders(transpose):
    # every border of the 4-bit grid and its fp32 neighbours, times scales of every significand
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    rows = []
    for s in range(8, 16):
        for near in (0.0, 1.0, -1.0):
            b = borders * s
            b = b if near == 0 else torch.nextafter(b, torch.full_like(b, near * 1e9))
            rows.append(torch.cat([torch.tensor([6.0 * s, -6.0 * s]), b, -b]))
    x = torch.stack(rows)
    x = torch.cat([x, x * 2.0 ** -11, torch.full_like(x, 6.0 * 448.0)], 0)
    amax = torch.tensor([2688.0], device=DEV)
    src = x.t().contiguous() if transpose else x
    check_quantized(pto.nvfp4_quantize(src.to(DEV), amax=amax, transpose=transpose), *ref.quantize(x, 2688.0), x.shape[0])


@pytest.mark.parametrize("amax", [0.0, 1.0, 2688.0, 2688.0 * 2.0 ** -20, 2689.0, 3.4e38, 1e-38])
def test_quantize_with_a_given_maximum(amax):
    x, host = wide(70, 96, torch.float32, 3)
    want = ref.quantize(host, float(np.float32(amax)))
    check_quantized(pto.nvfp4_quantize(x, amax=torch.tensor([amax], device=DEV)), *want, 70)


@pytest.mark.parametrize("scale", [0.0, 1e-38, 1e-30, 1e30])
def test_quantize_extreme_tensors(scale):
    host = torch.randn((40, 80), generator=torch.Generator().manual_seed(1)) * scale
    check_quantized(pto.nvfp4_quantize(host.to(DEV)), *ref.quantize(host), 40)


def test_non_finite_blocks_stay_visible():
    host = torch.randn((40, 160), generator=torch.Generator().manual_seed(2))
    host[1, 17], host[2, 40], host[39, 159] = float("inf"), float("nan"), float("-inf")
    for transpose in (False, True):
        src = host.t().contiguous() if transpose else host
        data, scales, g = pto.nvfp4_quantize(src.to(DEV), transpose=transpose)
        check_quantized((data, scales, g), *ref.quantize(host), 40)
    back = pto.nvfp4_dequantize(data, scales, g, out_dtype=torch.float32).cpu()
    assert torch.equal(torch.isnan(back).view(40, 10, 16).all(-1), ~torch.isfinite(host).view(40, 10, 16).all(-1))
    w = pto.nvfp4_quantize(torch.randn((8, 160), generator=torch.Generator().manual_seed(4)).to(DEV))
    out = pto.gemm_nvfp4(data, w[0], scales, w[1], g, w[2], out_dtype=torch.float32).cpu()
    assert torch.isnan(out[[1, 2, 39]]).all() and torch.isfinite(out[[0, 3, 38]]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,cols,offset", [(1, 16, 16, 0), (130, 112, 112, 0), (33, 64, 50, 1), (300, 1024, 1024, 8)])
def test_dequantize_is_exact(rows, k, cols, offset, dtype):
    g = torch.Generator().manual_seed(rows)
    data = torch.randint(0, 256, (rows, k // 2), generator=g, dtype=torch.uint8)
    scales = ref.tile_scales(torch.randint(0, 0x7F, (rows, k // 16), generator=g))
    want = (ref.values(data, scales) * 2.0 ** -3)[:, :cols].to(dtype)  # at most six significant bits: one rounding, if any
    buf = torch.full((rows, cols + offset), 9.0, dtype=dtype, device=DEV)
    out = buf[:, offset:] if offset % 8 else buf[:, :cols]
    pto.nvfp4_dequantize(data.to(DEV), scales.to(DEV), torch.tensor([0.125], device=DEV), out=out)
    assert torch.equal(out.cpu(), want)
    rest = buf[:, :offset] if offset % 8 else buf[:, cols:]
    assert (rest == 9.0).all()


def operand(rows, k, seed, extra=0):
    """Random codes and scales, the packed rows in a wider buffer of 0xFF."""
    g = torch.Generator().manual_seed(seed)
    width = k // 2
    pitch = (width + 15) // 16 * 16 + extra
    buf = torch.full((rows, pitch), 0xFF, dtype=torch.uint8)
    buf[:, :width] = torch.randint(0, 256, (rows, width), generator=g, dtype=torch.uint8)
    tiles = ref.tile_scales(torch.randint(0x20, 0x58, (rows, k // 16), generator=g))
    return buf.to(DEV)[:, :width], tiles.to(DEV), ref.values(buf[:, :width].contiguous(), tiles)


def check_product(m, n, k, out_dtype, bias, seed, out=None, extra=0):
    a, sfa, va = operand(m, k, seed, extra)
    b, sfb, vb = operand(n, k, seed + 1, extra)
    ga, gb = torch.tensor([0.037], device=DEV), torch.tensor([2.0 ** -5], device=DEV)
    bv = torch.randn((n,), generator=torch.Generator().manual_seed(seed + 2)).to(DEV) if bias else None
    got = pto.gemm_nvfp4(a, b, sfa, sfb, ga, gb, out_dtype=out_dtype, bias=bv, out=out)
    alpha = float(ga.double() * gb.double())
    va, vb = va.to(DEV), vb.to(DEV)
    want = va @ vb.t() * alpha
    size = va.abs() @ vb.abs().t() * abs(alpha)
    if bias:
        want, size = want + bv.double(), size + bv.double().abs()
    bound = size * ((k + 63) // 64 * 2.0 ** -22 + 4 * 2.0 ** -24) + torch.clamp(want.abs() * EPS[got.dtype], min=TINY[got.dtype])
    off = (got.double() - want).abs()
    assert (off <= bound).all(), f"{float((off / bound).max()):.2f} of the bound"
    return got


# up to 128 rows, and more of them where K is long beside few tiles; K cut over up to eight CTAs, or not at all
FEW = [(1, 16, 16), (1, 1, 16), (1, 8, 4096), (7, 130, 48), (16, 256, 64), (17, 100, 272), (32, 1000, 512), (33, 384, 1040),
       (64, 129, 4096), (65, 640, 336), (128, 128, 8192), (128, 1300, 6160), (129, 200, 2320), (300, 500, 4112), (1000, 300, 2576),
       (3, 20000, 256)]


@pytest.mark.parametrize("m,n,k", FEW)
@pytest.mark.parametrize("out_dtype,bias", [(torch.float32, True), (torch.bfloat16, False), (torch.float16, True)])
def test_product_few_rows(m, n, k, out_dtype, bias):
    check_product(m, n, k, out_dtype, bias, m + n + k)


# pairs of CTAs: less than one wave (halves of tiles), whole waves and ragged last ones, rows of C on 32, 16 and fewer bytes
MANY = [(129, 200, 256), (144, 512, 1024), (200, 1111, 768), (2304, 2304, 256), (2049, 2561, 272), (4000, 1801, 1040),
        (300, 20001, 80), (2560, 2312, 1808), (1000, 2004, 2320), (6000, 5000, 16)]


@pytest.mark.parametrize("m,n,k", MANY)
@pytest.mark.parametrize("out_dtype,bias", [(torch.float32, False), (torch.bfloat16, True), (torch.float16, False)])
def test_product_many_rows(m, n, k, out_dtype, bias):
    check_product(m, n, k, out_dtype, bias, m + n + k)


@pytest.mark.parametrize("m,n,k", [(5, 333, 304), (300, 333, 304), (2600, 2900, 304)])
@pytest.mark.parametrize("offset", [0, 1, 4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_product_into_a_part_of_a_buffer(m, n, k, offset, dtype):
    # operands with rows 48 bytes further apart than they need; C anywhere in a buffer whose rest stays as it was
    buf = torch.full((m + 2, n + 11), 5.0, dtype=dtype, device=DEV)
    out = buf[1:m + 1, offset:offset + n]
    assert check_product(m, n, k, dtype, True, m + offset, out=out, extra=48) is out
    assert (buf[0] == 5).all() and (buf[m + 1] == 5).all() and (buf[:, :offset] == 5).all() and (buf[:, offset + n:] == 5).all()


def test_quantize_into_given_buffers():
    x, host = wide(70, 90, torch.bfloat16, 1)
    data = torch.full((70, 64), 0xAB, dtype=torch.uint8, device=DEV)
    scales = torch.full((1, 2, 512), 0xCD, dtype=torch.uint8, device=DEV)
    g = torch.full((1,), -1.0, device=DEV)
    got = pto.nvfp4_quantize(x, data=data[:, :48], scales=scales, tensor_scale=g)
    assert got[1] is scales and got[2] is g
    check_quantized(got, *ref.quantize(host), 70)
    assert (data[:, 48:] == 0xAB).all()


def test_scales_of_zero_and_masked_rows():
    # a row of zeros beside others: its scales and codes are zero, and so is its row of the product
    host = torch.randn((20, 64), generator=torch.Generator().manual_seed(9))
    host[7] = 0.0
    a = pto.nvfp4_quantize(host.to(DEV))
    w = pto.nvfp4_quantize(torch.randn((33, 64), generator=torch.Generator().manual_seed(10)).to(DEV))
    out = pto.gemm_nvfp4(a[0], w[0], a[1], w[1], a[2], w[2], out_dtype=torch.float32)
    assert (out[7] == 0).all() and (out[[6, 8]] != 0).any(1).all()
    zero = pto.nvfp4_quantize(torch.zeros((3, 32), device=DEV))
    assert float(zero[2]) == 1.0 and (zero[0] == 0).all() and (zero[1] == 0).all()


def test_results_do_not_depend_on_the_stream_or_the_call():
    side = torch.cuda.Stream()
    for m, n, k in ((48, 700, 4096), (600, 3000, 1024)):
        x, w = torch.randn((m, k), device=DEV, dtype=torch.bfloat16), torch.randn((n, k), device=DEV, dtype=torch.bfloat16)
        side.wait_stream(torch.cuda.current_stream())
        outs = []
        for i in range(6):
            s = side if i % 2 else None
            a, b = pto.nvfp4_quantize(x, stream=s), pto.nvfp4_quantize(w, stream=s)
            outs.append(pto.gemm_nvfp4(a[0], b[0], a[1], b[1], a[2], b[2], stream=s))
        torch.cuda.synchronize()
        assert all(torch.equal(outs[0], o) for o in outs)


@pytest.mark.parametrize("m", [1, 40, 700])
def test_captured_and_replayed(m):
    k, n = 768, 900
    x = torch.randn((m, k), device=DEV, dtype=torch.bfloat16)
    w = pto.nvfp4_quantize(torch.randn((n, k), device=DEV))
    out, again = torch.empty((m, n), device=DEV), torch.empty((m, n), device=DEV)

    def step(into):
        a = pto.nvfp4_quantize(x)
        pto.gemm_nvfp4(a[0], w[0], a[1], w[1], a[2], w[2], out=into)

    step(out)  # warm: what is set up once per device
    graphs = []
    for into in (out, again):  # two graphs alive at once
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(into)
        graphs.append(g)
    x.mul_(-3.0)
    for _ in range(3):
        for g in graphs:
            g.replay()
    want = torch.empty((m, n), device=DEV)
    step(want)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(again, want)


def test_python_refusals():
    x = torch.randn((8, 64), device=DEV)
    data, scales, g = pto.nvfp4_quantize(x)
    bad = [
        lambda: pto.nvfp4_quantize(x.double()), lambda: pto.nvfp4_quantize(x[:, ::2]), lambda: pto.nvfp4_quantize(x[0]),
        lambda: pto.nvfp4_quantize(x[:0]), lambda: pto.nvfp4_quantize(x, amax=torch.ones(2, device=DEV)),
        lambda: pto.nvfp4_quantize(x, amax=torch.ones(1)), lambda: pto.nvfp4_quantize(x, data=data[:, :16]),
        lambda: pto.nvfp4_quantize(x, scales=scales[:, :, :256]), lambda: pto.nvfp4_quantize(x, tensor_scale=g.double()),
        lambda: pto.nvfp4_dequantize(data, scales[:, :0]), lambda: pto.nvfp4_dequantize(data, scales, out_dtype=torch.int32),
        lambda: pto.nvfp4_dequantize(data, scales, out=x[:, :40]), lambda: pto.nvfp4_dequantize(x, scales),
        lambda: pto.gemm_nvfp4(data, data[:, :24], scales, scales), lambda: pto.gemm_nvfp4(data, data, scales, scales.view(1, 512, 1)),
        lambda: pto.gemm_nvfp4(data.view(torch.float8_e4m3fn), data, scales, scales),
        lambda: pto.gemm_nvfp4(data[:, :4], data[:, :4], scales, scales),
        lambda: pto.gemm_nvfp4(data, data, scales, scales, ga=torch.ones(2, device=DEV)),
        lambda: pto.gemm_nvfp4(data, data, scales, scales, bias=torch.ones(7, device=DEV)),
        lambda: pto.gemm_nvfp4(data, data, scales, scales, bias=torch.ones(8, device=DEV).half()),
        lambda: pto.gemm_nvfp4(data, data, scales, scales, out=x), lambda: pto.gemm_nvfp4(data, data, scales, scales, out_dtype=torch.int8),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    shifted = torch.zeros(8 * 32 + 8, dtype=torch.uint8, device=DEV)[8:].view(8, 32)  # off the 16-byte boundary
    with pytest.raises(pto.PtoB200Error) as e:
        pto.gemm_nvfp4(shifted, data, scales, scales)
    assert e.value.code == 2


def test_past_two_to_the_31_elements():
    rows, k = 65664, 32832  # 2^31 + 8e6 elements
    x = torch.empty((rows, k), dtype=torch.bfloat16, device=DEV)
    for r in range(0, rows, 4104):
        x[r:r + 4104].normal_(generator=torch.Generator(DEV).manual_seed(r))
    amax = torch.tensor([6.0], device=DEV)
    data, scales, g = pto.nvfp4_quantize(x, amax=amax)
    tail = pto.nvfp4_quantize(x[-128:], amax=amax)
    assert torch.equal(data[-128:], tail[0]) and torch.equal(scales[-1], tail[1][0])
    back = pto.nvfp4_dequantize(data, scales, g)
    assert torch.equal(back[-128:], pto.nvfp4_dequantize(tail[0], tail[1], g))
    del back
    turned = pto.nvfp4_quantize(x, amax=amax, transpose=True)
    assert torch.equal(turned[0][:, -32:], pto.nvfp4_quantize(x[-64:], amax=amax, transpose=True)[0])
    del x, turned
    # a product with as many results
    a, b = (data[:, :32], scales[:, :1].contiguous()), (data[:k, 32:64], scales[:(k + 127) // 128, 1:2].contiguous())
    c = pto.gemm_nvfp4(a[0], b[0], a[1], b[1][:(k + 127) // 128])
    want = pto.gemm_nvfp4(a[0][-128:], b[0], a[1][-1:], b[1][:(k + 127) // 128])
    assert torch.equal(c[-128:], want)


@pytest.mark.parametrize("m,n,k", [(5, 256, 512), (300, 512, 4096)])
def test_captured_with_copies_and_two_streams(m, n, k):
    # launches that may overlap what comes before them, behind a copy, behind a memory set and where two streams join
    g = torch.Generator().manual_seed(m)
    x, w = torch.zeros((m, k), device=DEV), torch.zeros((n, k), device=DEV)
    source = torch.zeros((m, k), device=DEV)
    side = torch.cuda.Stream()
    out = torch.zeros((m, n), device=DEV)

    def step():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            qw = pto.nvfp4_quantize(w)
        x.copy_(source)
        qx = pto.nvfp4_quantize(x)
        main.wait_stream(side)
        pto.gemm_nvfp4(qx[0], qw[0], qx[1], qw[1], qx[2], qw[2], out=out)
        out.add_(0)
        back = pto.nvfp4_dequantize(*qx, out_dtype=torch.float32)
        x.zero_()
        return qx, qw, back

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qx, qw, back = step()
    for _ in range(3):
        source.copy_(torch.randn((m, k), generator=g))
        w.copy_(torch.randn((n, k), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        a, b = pto.nvfp4_quantize(source), pto.nvfp4_quantize(w)
        for got, want in zip((*qx, *qw, back), (*a, *b, pto.nvfp4_dequantize(*a, out_dtype=torch.float32))):
            assert torch.equal(got, want)
        assert torch.equal(out, pto.gemm_nvfp4(a[0], b[0], a[1], b[1], a[2], b[2], out_dtype=torch.float32))
