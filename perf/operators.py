"""The low-precision linear layer's operators on real sizes: two-level 4-bit floating point (NVFP4: e2m1 elements, one
e4m3 scale per 16 elements, one fp32 scale per tensor) quantised and multiplied, and activations kept in 8 bits (MXFP8:
e4m3 elements, one e8m0 scale per 32 elements) with the weight gradient computed from them.

``run`` computes one pass: in the plain form (elementary torch operations in 32 bits) where ``own`` is false, through
the package's entry points where it is true. Scales of 4-bit tensors are held in 512-byte tiles of 128 rows x 4 scales,
shape [ceil(rows / 128), ceil(K / 64), 512]: byte (row % 32) * 16 + (row % 128) // 32 * 4 + j holds scale j of the tile.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ES = {"f32": 4, "bf16": 2, "f16": 2}


def _up(v, m):
    return (v + m - 1) // m * m


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the activations of eight decoding sequences, the tensor's largest value known from calibration: latency
        {"name": "nvfp4_cast_decode", "op": "cast", "rows": 8, "k": 4096, "dtype": "bf16", "transpose": False, "static": True},
        # a training batch's activations, the largest value found in the call
        {"name": "nvfp4_cast_activations", "op": "cast", "rows": 16384, "k": 8192, "dtype": "bf16", "transpose": False, "static": False},
        # a gradient transposed for the weight gradient's product; odd token count, ragged width
        {"name": "nvfp4_cast_transposed", "op": "cast", "rows": 4093, "k": 2904, "dtype": "f32", "transpose": True, "static": False},
        # one token of one sequence against a square weight
        {"name": "gemm_nvfp4_one_token", "op": "gemm", "m": 1, "n": 4096, "k": 4096, "out": "bf16", "bias": False},
        # a few dozen decoding sequences against a wide weight
        {"name": "gemm_nvfp4_decode", "op": "gemm", "m": 48, "n": 14336, "k": 4096, "out": "f16", "bias": False},
        # a prompt of ragged length, odd width, bias
        {"name": "gemm_nvfp4_2040x8100x8192", "op": "gemm", "m": 2040, "n": 8100, "k": 8192, "out": "f32", "bias": True},
        # a training batch
        {"name": "gemm_nvfp4_16384x8192x8192", "op": "gemm", "m": 16384, "n": 8192, "k": 8192, "out": "bf16", "bias": False},
        # a batch's activations kept for the backward pass
        {"name": "mx_checkpoint_activations", "op": "checkpoint", "rows": 16384, "k": 8192, "dtype": "bf16"},
        # one short sequence's, half precision
        {"name": "mx_checkpoint_short", "op": "checkpoint", "rows": 333, "k": 1056, "dtype": "f16"},
        # the gradient of a small weight over a short ragged batch
        {"name": "wgrad_small", "op": "wgrad", "t": 515, "n": 1000, "k": 1056, "dtype": "f16", "out": "bf16", "addend": False},
        # an accumulation step: the new gradient joins the fp32 one that is there
        {"name": "wgrad_accumulate", "op": "wgrad", "t": 4096, "n": 4096, "k": 2048, "dtype": "bf16", "out": "f32", "addend": True},
        # a long batch's gradient of a large weight
        {"name": "wgrad_16384x8192x8192", "op": "wgrad", "t": 16384, "n": 8192, "k": 8192, "dtype": "bf16", "out": "f32", "addend": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cast", "gemm", "gemm", "checkpoint", "wgrad"])
    if op == "cast":
        return {"op": op, "rows": _log(rng, 1, 16384), "k": _log(rng, 2, 1024) * 8, "dtype": rng.choice(["f32", "bf16", "f16"]),
                "transpose": rng.random() < 0.4, "static": rng.random() < 0.4}
    if op == "gemm":
        return {"op": op, "m": _log(rng, 1, 16384), "n": _log(rng, 8, 8192), "k": _log(rng, 4, 512) * 16,
                "out": rng.choice(["f32", "bf16", "f16"]), "bias": rng.random() < 0.3}
    if op == "checkpoint":
        return {"op": op, "rows": _log(rng, 1, 16384), "k": _log(rng, 1, 256) * 32, "dtype": rng.choice(["bf16", "f16"])}
    return {"op": op, "t": _log(rng, 1, 16384), "n": _log(rng, 1, 1024) * 8, "k": _log(rng, 1, 256) * 32,
            "dtype": rng.choice(["bf16", "f16"]), "out": rng.choice(["f32", "bf16", "f16"]), "addend": rng.random() < 0.3}


def work(case):
    op = case["op"]
    if op == "cast":
        n = case["rows"] * case["k"]
        # read, write codes and scales; read them, write the values
        return {"bytes": n * (_ES[case["dtype"]] + 9 / 16 + 9 / 16 + 2), "flops": 0}
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k * 9 / 16 + m * n * _ES[case["out"]] + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if op == "checkpoint":
        return {"bytes": case["rows"] * case["k"] * (2 + 1 + 1 / 32), "flops": 0}
    t, n, k = case["t"], case["n"], case["k"]
    out = n * k * _ES[case["out"]]
    return {"bytes": t * n * 2 + t * k * (1 + 1 / 32) + out * (2 if case["addend"] else 1), "flops": 2 * t * n * k}


# ------------------------------------------------------------------------------------------------ inputs

def _exp2(e, dtype=torch.float32):
    """2^e exactly, e whole numbers from -127 to 127: put together from its bits."""
    if dtype == torch.float64:
        return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)
    bits = torch.where(e < -126, 0x00400000, (e.to(torch.int32) + 127) << 23)
    return bits.to(torch.int32).view(torch.float32)


def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 16 + salt)


def _activations(rows, k, dtype, seed, salt):
    """Normal values whose columns have widths of their own and a few of which are far out, as activations have."""
    g = _generator(seed, salt)
    x = torch.randn((rows, k), generator=g, device="cuda")
    width = torch.exp(torch.randn((k,), generator=g, device="cuda") * 0.7)
    far = (torch.rand((k,), generator=g, device="cuda") < 0.01) * 12.0 + 1.0
    return (x * (width * far)).to(_DT[dtype])


def _pitched(x):
    """x [rows, cols] in rows that start on 16-byte boundaries."""
    cols = x.shape[1]
    step = 16 // x.element_size()
    buf = torch.zeros((x.shape[0], _up(cols, step)), dtype=x.dtype, device=x.device)
    buf[:, :cols] = x
    return buf[:, :cols]


def _tile_scales(s):
    """[rows, K / 16] scale bytes in 512-byte tiles; what pads them is zero."""
    rows, ks = s.shape
    rt, kt = _up(rows, 128) // 128, _up(ks, 4) // 4
    full = torch.zeros((rt * 128, kt * 4), dtype=torch.uint8, device=s.device)
    full[:rows, :ks] = s
    return full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(rt, kt, 512)


def _untile_scales(tiles, rows, ks):
    rt, kt, _ = tiles.shape
    return tiles.view(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:rows, :ks]


def _operand(rows, k, seed, salt, width=1.0):
    """A tensor in NVFP4 as a program holds it: packed codes [rows, K / 2], tiled scales, the tensor's scale."""
    x = _activations(rows, k, "f32", seed, salt) * width
    codes, scales, g = _quantize_plain(x, None)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    return _pitched(packed), _tile_scales(scales), g


def _inputs(case, seed):
    op = case["op"]
    if op == "cast":
        x = _activations(case["rows"], case["k"], case["dtype"], seed, 0)
        # a calibrated largest value: a little below what this batch has
        amax = (x.float().abs().amax() * 0.9).reshape(1) if case["static"] else None
        return {"x": x, "amax": amax}
    if op == "gemm":
        a, sfa, ga = _operand(case["m"], case["k"], seed, 0)
        b, sfb, gb = _operand(case["n"], case["k"], seed, 1, width=0.02)  # a weight
        bias = torch.randn((case["n"],), generator=_generator(seed, 2), device="cuda") if case["bias"] else None
        return {"a": a, "sfa": sfa, "ga": ga, "b": b, "sfb": sfb, "gb": gb, "bias": bias}
    if op == "checkpoint":
        return {"x": _activations(case["rows"], case["k"], case["dtype"], seed, 0)}
    dy = (torch.randn((case["t"], case["n"]), generator=_generator(seed, 0), device="cuda") * 0.02).to(_DT[case["dtype"]])
    data, scales = _checkpoint_plain(_activations(case["t"], case["k"], "bf16", seed, 1))
    addend = None
    if case["addend"]:
        addend = torch.randn((case["n"], case["k"]), generator=_generator(seed, 2), device="cuda").to(_DT[case["out"]])
    return {"dy": dy, "data": data.view(torch.uint8), "scales": scales, "addend": addend}


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ------------------------------------------------------------------------------------------------ plain forms

def _power_of_two_scale(amax):
    """The smallest power of two that is at least amax / 2688 (= 6 * 448); 1 for 0."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1); 2688 = 0.65625 * 2^12
    e = torch.clamp(exponent - 12 + (mantissa > 0.65625), min=-126)
    return torch.where(amax == 0, torch.ones_like(amax), _exp2(e))


def _quantize_plain(x, amax):
    """(codes [rows, K16], scale bytes [rows, K16 / 16], tensor scale [1]) of x [rows, K], K16 = K rounded up to 16."""
    x = x.float()
    rows, k = x.shape
    if amax is None:
        amax = torch.where(torch.isfinite(x), x.abs(), 0.0).amax().reshape(1)
    g = _power_of_two_scale(amax)
    blocks = torch.nn.functional.pad(x, (0, _up(k, 16) - k)).view(rows, -1, 16)
    m = (blocks / g).abs().amax(-1, keepdim=True)
    # the quotient's rounding never crosses a border of the 8-bit format: 6 times a border has few bits
    s8 = torch.clamp(m / 6.0, max=448.0).to(torch.float8_e4m3fn)
    s = s8.float()
    q = torch.where(s > 0, blocks / (s * g), 0.0)
    a = q.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code | ((q < 0).to(torch.uint8) << 3)
    return code.view(rows, -1), s8.view(torch.uint8).view(rows, -1), g


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _values_of(codes, scales, dtype=torch.float32):
    """e2m1 codes [rows, K] times their e4m3 scales [rows, K / 16]."""
    v = torch.tensor(_E2M1, dtype=dtype, device=codes.device)[codes.int()]
    s = scales.view(torch.float8_e4m3fn).to(dtype)
    return (v.view(codes.shape[0], -1, 16) * s[:, :, None]).view(codes.shape[0], -1)


def _unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).view(packed.shape[0], -1)


def _operand_values(packed, tiles, dtype=torch.float32):
    return _values_of(_unpack(packed), _untile_scales(tiles, packed.shape[0], packed.shape[1] // 8).contiguous(), dtype)


def _checkpoint_plain(x):
    """e4m3 elements and e8m0 bytes of x [rows, K]: exponent of the block's largest value less 8, saturating, zeros positive."""
    rows, k = x.shape
    blocks = x.float().view(rows, k // 32, 32)
    _, exponent = torch.frexp(blocks.abs().amax(-1, keepdim=True))  # value in [2^(exponent - 1), 2^exponent)
    biased = torch.clamp(exponent.int() - 1 + 127, min=0)
    biased = torch.where(blocks.abs().amax(-1, keepdim=True) == 0, 0, biased)
    e = torch.clamp(biased - 8, min=0)
    y = blocks * _exp2(127 - e)
    data = torch.clamp(y, -448.0, 448.0).to(torch.float8_e4m3fn)
    data = torch.where(data.float() == 0, torch.zeros_like(y), data.float()).to(torch.float8_e4m3fn)
    return data.view(rows, k), e.view(rows, k // 32).to(torch.uint8)


def _checkpoint_values(data, scales, dtype=torch.float32):
    t, k = data.shape
    v = data.view(torch.float8_e4m3fn).to(dtype).view(t, k // 32, 32)
    return (v * _exp2(scales.int() - 127, dtype)[:, :, None]).view(t, k)


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "cast":
        x = s["x"].t() if case["transpose"] else s["x"]
        codes, scales, g = _quantize_plain(x, s["amax"])
        return {"values": (_values_of(codes, scales) * g).to(torch.bfloat16), "tensor_scale": g}
    if op == "gemm":
        out = _operand_values(s["a"], s["sfa"]) @ _operand_values(s["b"], s["sfb"]).t()
        out = out * (s["ga"] * s["gb"])
        if s["bias"] is not None:
            out = out + s["bias"]
        return out.to(_DT[case["out"]])
    if op == "checkpoint":
        data, scales = _checkpoint_plain(s["x"])
        return {"data": data, "scales": scales}
    dw = s["dy"].float().t() @ _checkpoint_values(s["data"], s["scales"])
    if s["addend"] is not None:
        dw = dw + s["addend"].float()
    return dw.to(_DT[case["out"]])


# ------------------------------------------------------------------------------------------------ the package's operators

def _run_own(s):
    import pto_isa_mirror_b200 as pto

    case = s["case"]
    op = case["op"]
    if op == "cast":
        data, scales, g = pto.nvfp4_quantize(s["x"], amax=s["amax"], transpose=case["transpose"])
        return {"values": pto.nvfp4_dequantize(data, scales, g, out_dtype=torch.bfloat16), "tensor_scale": g}
    if op == "gemm":
        return pto.gemm_nvfp4(s["a"], s["b"], s["sfa"], s["sfb"], s["ga"], s["gb"], out_dtype=_DT[case["out"]], bias=s["bias"])
    if op == "checkpoint":
        data, scales = pto.mx_quantize_e4m3(s["x"])
        return {"data": data.view(torch.float8_e4m3fn), "scales": scales}
    return pto.gemm_wgrad_mx(s["dy"], s["data"], s["scales"], out_dtype=_DT[case["out"]], addend=s["addend"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ in 64 bits

def _nearest(x, grid):
    """The values of an ascending grid (of non-negative numbers) nearest to x >= 0; between two, the one at an even place."""
    hi = torch.clamp(torch.searchsorted(grid, x), max=grid.numel() - 1)
    lo = torch.clamp(hi - 1, min=0)
    below, above = x - grid[lo], grid[hi] - x
    return grid[torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)]


def _e4m3_grid(device):
    v = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    return torch.tensor(v[:127], dtype=torch.float64, device=device)


def _e2m1_grid(device):
    return torch.tensor(_E2M1[:8], dtype=torch.float64, device=device)


def _exact_cast(x, amax):
    x = x.double()
    rows, k = x.shape
    top = float(x.abs().amax()) if amax is None else float(amax)
    g = 2.0 ** math.ceil(math.log2(top / 2688.0)) if top > 0 else 1.0
    while g / 2 >= top / 2688.0 and top > 0:  # the logarithm's rounding
        g /= 2
    while g < top / 2688.0:
        g *= 2
    e4m3, e2m1 = _e4m3_grid(x.device), _e2m1_grid(x.device)
    pad = torch.nn.functional.pad(x, (0, _up(k, 16) - k))
    out = torch.empty_like(pad, dtype=torch.bfloat16)
    for r in range(0, rows, 2048):
        b = pad[r:r + 2048].view(-1, pad.shape[1] // 16, 16)
        s = _nearest(torch.clamp(b.abs().amax(-1) / (6.0 * g), max=448.0), e4m3)[:, :, None]
        q = torch.where(s > 0, b.abs() / (s * g), 0.0)
        out[r:r + 2048] = (torch.sign(b) * _nearest(torch.clamp(q, max=6.0), e2m1) * s * g).view(b.shape[0], -1).to(torch.bfloat16)
    return {"values": out.double(), "tensor_scale": torch.tensor([g], dtype=torch.float64)}


def _exact_checkpoint(x):
    x = x.double()
    e4m3 = _e4m3_grid(x.device)
    rows, k = x.shape
    data = torch.empty_like(x)
    for r in range(0, rows, 2048):
        b = x[r:r + 2048].view(-1, k // 32, 32)
        m = b.abs().amax(-1, keepdim=True)
        e = torch.where(m > 0, torch.clamp(torch.frexp(m)[1] - 1, min=-119), -119)
        y = torch.clamp(b * _exp2(8 - e, torch.float64), -448.0, 448.0)
        data[r:r + 2048] = (torch.sign(y) * _nearest(y.abs(), e4m3)).view(-1, k)
    return {"data": data, "scales": None}


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "cast":
        return _exact_cast(s["x"].t() if case["transpose"] else s["x"], s["amax"])
    if op == "gemm":
        out = _operand_values(s["a"], s["sfa"], torch.float64) @ _operand_values(s["b"], s["sfb"], torch.float64).t()
        out = out * (s["ga"].double() * s["gb"].double())
        return out if s["bias"] is None else out + s["bias"].double()
    if op == "checkpoint":
        return _exact_checkpoint(s["x"])
    dw = s["dy"].double().t() @ _checkpoint_values(s["data"], s["scales"], torch.float64)
    return dw if s["addend"] is None else dw + s["addend"].double()
