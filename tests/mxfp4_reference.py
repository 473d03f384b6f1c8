"""MXFP4 in 64 bits, from the format's definition: what the kernels are held to."""
import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize(x):
    """[rows, K] -> (codes [rows, K], scale bytes [rows, K / 32]) in 64 bits."""
    rows, k = x.shape
    b = x.double().reshape(rows, k // 32, 32)
    finite = torch.isfinite(b).all(-1)
    amax = torch.where(finite, b.abs().amax(-1), torch.ones_like(b[..., 0]))
    exponent = torch.frexp(amax)[1].double() - 1  # floor(log2), of a zero maximum something small
    code = torch.where(amax > 0, exponent - 2 + 127, torch.zeros_like(amax)).clamp(min=0)
    scaled = b / torch.exp2(code - 127).unsqueeze(-1)
    a = scaled.abs().clamp(max=6.0)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    above = torch.searchsorted(grid, a.contiguous()).clamp(1, 7)
    low, high = grid[above - 1], grid[above]
    up = (a - low > high - a) | ((a - low == high - a) & (above % 2 == 0))
    value = torch.where(up, above, above - 1) + 8 * torch.signbit(scaled)
    value = torch.where(finite.unsqueeze(-1), value, torch.zeros_like(value))
    return value.reshape(rows, k).to(torch.uint8), torch.where(finite, code, torch.full_like(code, 255.0)).to(torch.uint8)


def pack(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1)


def values(codes, scales):
    """Codes [..., K] and scale bytes [..., K / 32] -> 64-bit values, NaN where the scale is 255."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device=codes.device)
    s = torch.where(scales == 255, torch.full_like(scales, 0, dtype=torch.float64) / 0.0, torch.exp2(scales.double() - 127))
    return grid[codes.long()] * s.repeat_interleave(32, -1)


def untile(tiled, rows, k):
    """Tiled scale bytes -> ([rows, K / 32], whether all the padding is zero)."""
    blocks = k // 32
    t = tiled.reshape((rows + 127) // 128, (blocks + 3) // 4, 32, 4, 4)  # [row tile][block group][row % 32][row / 32 % 4][block % 4]
    full = t.permute(0, 3, 2, 1, 4).reshape((rows + 127) // 128 * 128, -1)
    padding = full.clone()
    padding[:rows, :blocks] = 0
    return full[:rows, :blocks], not bool(padding.any())


def weight(g, n, k, std=0.02, device="cuda"):
    """A random weight's (packed, scale bytes)."""
    codes, scales = quantize(torch.randn(n, k, generator=g, device=device) * std)
    return pack(codes), scales


def silu_mul(gate_up):
    gate, up = gate_up.chunk(2, -1)
    return gate * torch.sigmoid(gate) * up
