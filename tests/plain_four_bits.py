"""Microscaled 4-bit floating point in plain PyTorch, 64-bit: what fp4_quantize, fp4_dequantize and fp4_gemm are held to."""
import torch

BLOCK = {"nvfp4": 16, "mxfp4": 32}
KINDS = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def floor_power(v):
    """The largest power of two not above v > 0."""
    return (v.view(torch.int64) >> 52 << 52).view(torch.float64)


def to_e4m3(v):
    """v in [0, 448] to the nearest of three bits behind the first, steps of 2^-9 at the low end, halves to even."""
    step = torch.clamp(torch.where(v > 0, floor_power(v), 0.0), min=2.0 ** -6) / 8
    return torch.round(v / step) * step


def quantize(x, format):
    """(codes with a sign as values [rows, blocks, block], block scales [rows, blocks, 1], row scales [rows, 1]), all float64, of finite x."""
    rows, cols = x.shape
    b = BLOCK[format]
    v = torch.zeros(rows, -(-cols // b) * b, dtype=torch.float64)
    v[:, :cols] = x.double().cpu()
    v = v.reshape(rows, -1, b)
    top = v.abs().amax(2, keepdim=True)
    row = torch.ones(rows, 1, dtype=torch.float64)
    if format == "nvfp4":
        most = top.amax(1)
        row = torch.where(most > 0, torch.clamp(floor_power(most) / 1024, min=2.0 ** -126), 1.0)
        scale = torch.where(top > 0, torch.clamp(to_e4m3(top / row[:, :, None] / 6), min=2.0 ** -9), 0.0)
    else:
        scale = torch.clamp(torch.where(top > 0, floor_power(top) / 4, 0.0), min=2.0 ** -127)
    a = torch.where(scale > 0, v.abs() / row[:, :, None] / torch.where(scale > 0, scale, 1.0), 0.0)
    # the nearest of the eight; between two at the same distance the one with the even number
    far = (a.unsqueeze(-1) - KINDS).abs()
    odd = torch.arange(8) % 2
    code = (far == far.amin(-1, keepdim=True)).double().mul(2 - odd).argmax(-1)
    return torch.copysign(KINDS[code], v), scale, row


def values(x, format):
    """What x stands for in four bits, [rows, cols] float64."""
    rows, cols = x.shape
    code, scale, row = quantize(x, format)
    return (code * scale * row[:, :, None]).reshape(rows, -1)[:, :cols]
