"""NVFP4 from its definition in 64 bits, for the tests: quantiser, scale tiles, values."""
import math

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
E4M3 = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)],
                    dtype=torch.float64)[:127]


def nearest_code(x, grid):
    """Place of the value of an ascending grid nearest to x >= 0; between two the even place; past the end the last."""
    hi = torch.clamp(torch.searchsorted(grid, x.contiguous()), max=grid.numel() - 1)
    lo = torch.clamp(hi - 1, min=0)
    below, above = x - grid[lo], grid[hi] - x
    return torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)


def power_of_two_scale(amax):
    if amax == 0:
        return 1.0
    mantissa, exponent = math.frexp(amax / 2688.0)  # in 64 bits; 2688 * 2^j divides exactly
    return max(2.0 ** (exponent - 1 if mantissa == 0.5 else exponent), 2.0 ** -126)


def quantize(x, amax=None):
    """x [rows, K] on the CPU -> (codes [rows, K16], scale codes [rows, K16 / 16], g)."""
    x = x.double()
    rows, k = x.shape
    if amax is None:
        amax = float(torch.where(torch.isfinite(x), x.abs(), 0.0).max())
    g = power_of_two_scale(amax)
    b = torch.nn.functional.pad(x, (0, -k % 16)).view(rows, -1, 16)
    m = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    s = nearest_code(torch.where(bad, 0.0, torch.clamp(m / (6.0 * g), max=448.0)), E4M3)
    sv = E4M3[s][:, :, None]
    q = torch.where((sv > 0) & ~bad[:, :, None], b / (torch.where(sv > 0, sv, 1.0) * g), 0.0)
    codes = nearest_code(q.abs(), E2M1) | ((q < 0).long() << 3)
    return codes.view(rows, -1), torch.where(bad, 0x7F, s), g


def tile_scales(s):
    rows, ks = s.shape
    rt, kt = (rows + 127) // 128, (ks + 3) // 4
    full = torch.zeros((rt * 128, kt * 4), dtype=torch.uint8)
    full[:rows, :ks] = s.to(torch.uint8)
    return full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(rt, kt, 512)


def untile_scales(tiles, rows, ks):
    rt, kt, _ = tiles.shape
    return tiles.view(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:rows, :ks]


def unpack(data):
    return torch.stack((data & 15, data >> 4), -1).reshape(data.shape[0], -1).long()


def values(data, tiles):
    """code * scale in 64 bits of packed codes [rows, K / 2] and scale tiles, on the CPU."""
    codes = unpack(data)
    rows, k = codes.shape
    s = untile_scales(tiles, rows, k // 16).contiguous().view(torch.float8_e4m3fn).double()
    v = torch.where(codes >= 8, -1.0, 1.0) * E2M1[codes & 7]
    return (v.view(rows, -1, 16) * s[:, :, None]).view(rows, k)
