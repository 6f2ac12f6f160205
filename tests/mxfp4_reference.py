"""Microscaled 4-bit blocks in 64 bits on the host: the definition, element by element, for the tests."""
import torch

GRID = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def pitch(cols):
    return (cols + 127) // 128 * 64


def quantize(x):
    """x [rows, cols] -> (codes, scales) laid out as the library lays them out"""
    x = x.cpu().double()
    rows, cols = x.shape
    padded = torch.zeros(rows, pitch(cols) * 2, dtype=torch.float64)
    padded[:, :cols] = x
    blocks = padded.reshape(rows, -1, 32)
    top = blocks.abs().amax(-1)
    bad = ~torch.isfinite(blocks).all(-1)
    e = torch.frexp(torch.where(bad | (top == 0), 1.0, top))[1] - 3          # floor(log2 top) - 2
    e = torch.where(top == 0, -127, e).clamp(min=-127)
    v = torch.where(bad[..., None], 0.0, blocks) * torch.exp2(-e.double())[..., None]
    a = v.abs()
    code = torch.zeros_like(a, dtype=torch.int64)
    for i in range(7):   # past the midpoint to the next value: code i + 1; on it: to the even one of the two
        mid = (GRID[i] + GRID[i + 1]) / 2
        code += ((a > mid) | ((a == mid) & (i % 2 == 1))).long()
    code = code + 8 * torch.signbit(v).long()
    code = torch.where(bad[..., None], 0, code).reshape(rows, -1)
    codes = (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8)
    scales = torch.where(bad, 255, e + 127).to(torch.uint8)
    scales[:, (cols + 31) // 32:] = 0
    return codes, scales


def values(codes, scales, cols):
    """the values codes and scales stand for, in 64 bits"""
    codes, scales = codes.cpu(), scales.cpu()
    v = GRID[torch.stack([codes & 15, codes >> 4], -1).long().reshape(codes.shape[0], -1)]
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    return (v * s.repeat_interleave(32, 1))[:, :cols]


def random_codes(g, rows, cols, low=127, high=127):
    """random codes with scale bytes in [low, high]: padding as the library leaves it"""
    c = torch.randint(0, 16, (rows, pitch(cols) * 2), generator=g)
    c[:, cols:] = 0
    s = torch.randint(low, high + 1, (rows, pitch(cols) // 16), generator=g)
    s[:, (cols + 31) // 32:] = 0
    return (c[:, 0::2] + 16 * c[:, 1::2]).to(torch.uint8), s.to(torch.uint8)
