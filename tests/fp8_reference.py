"""8-bit rows and their products in 64 bits, written from the definitions (test infrastructure)."""
import math

import torch


def power(e):
    """2^e in float64 for whole e (from its bits: a power function may be off by a rounding)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def blocks(v, fill=0.0):
    rows, cols = v.shape
    out = torch.full((rows, (cols + 127) // 128 * 128), fill, dtype=v.dtype, device=v.device)
    out[:, :cols] = v
    return out.view(rows, -1, 128)


def exponents(v64):
    """[rows, blocks] smallest whole e >= -127 with largest finite magnitude <= 448 * 2^e."""
    b = blocks(v64)
    a = torch.where(torch.isfinite(b), b.abs(), 0).amax(2)
    m, x = torch.frexp(a)                      # a = m * 2^x, 0.5 <= m < 1; 448 = 0.875 * 2^9
    return torch.where(a > 0, x - 9 + (m > 0.875).int(), -127).clamp(min=-127)


def quantize(v64):
    """-> (values of the padded rows as e4m3 numbers in float64, exponents); fp32 inputs only (the conversion goes through fp32, exactly)."""
    e = exponents(v64)
    z = blocks(v64) * power(-e)[:, :, None]
    z = torch.where(torch.isfinite(z), z, math.nan)
    return z.float().to(torch.float8_e4m3fn).double().view(v64.shape[0], -1), e


def pieces(bytes_):
    """[rows, blocks] scale bytes -> the layout of Fp8Rows.scales."""
    rows, n = bytes_.shape
    full = torch.zeros((rows + 127) // 128 * 128, (n + 3) // 4 * 4, dtype=torch.uint8, device=bytes_.device)
    full[:rows, :n] = bytes_
    out = torch.zeros(full.shape[0] // 128, full.shape[1] // 4, 32, 4, 4, dtype=torch.uint8, device=bytes_.device)
    for b in range(4):
        for j in range(4):
            out[:, :, :, b, j] = full[:, j::4].view(-1, 4, 32, full.shape[1] // 4)[:, b].permute(0, 2, 1)
    return out


def check_rows(got, v64, slack):
    """8-bit rows against values of which each is known to `slack`: padding as it should be, every block's scale the right power of two for a maximum that
    may be off by the slack, every value within half a step of the format (2^-4 of it, or 2^-10 of the scale among the smallest)."""
    rows, cols = v64.shape
    assert got.cols == cols and got.shape == (rows, cols)
    data, scales = got.data.double(), got.block_scales().double()
    assert data.shape == (rows, (cols + 127) // 128 * 128) and bool((data[:, cols:] == 0).all())
    raw = got.scales.view(torch.uint8)
    bytes_ = torch.frexp(scales)[1] - 1 + 127
    assert torch.equal(raw, pieces(bytes_.to(torch.uint8))), "bytes of rows or blocks that do not exist"
    bad = ~torch.isfinite(v64)
    assert torch.equal(torch.isnan(data[:, :cols]), bad)
    v, slack = torch.where(bad, 0.0, v64), torch.where(bad, 0.0, torch.broadcast_to(torch.as_tensor(slack, dtype=torch.float64, device=v64.device), v64.shape))
    top, off = blocks(v.abs()).amax(2), blocks(slack).amax(2)
    assert bool((top - off <= 448 * scales).all()), "a block's maximum does not fit its scale"
    assert bool(((top + off > 224 * scales) | (bytes_ == 0)).all()), "a block's scale is too large"
    s = scales.repeat_interleave(128, 1)[:, :cols]
    err = (torch.where(bad, 0.0, data[:, :cols]) * s - v).abs()
    # (a value right above 448 scales, by the slack, comes out as 448)
    lim = (v.abs() + slack) * 2.0 ** -4 + s * 2.0 ** -10 + slack
    assert bool((err <= lim).all()), f"off by {float((err - lim).max()):.3e} more than half a step"


def values(rows8):
    return rows8.data.double().view(rows8.data.shape[0], -1, 128).mul(rows8.block_scales().double()[:, :, None]).view(rows8.data.shape)[:, :rows8.cols]


def product(x, w):
    """-> (x w^T, what fp32 sums may be off): exact products; a chain adds the 32 of an instruction in one go, K / 32 instructions, blocks of 128 scaled apart;
    no partial sum is larger than the sum of magnitudes, and none is off by more than a rounding to 24 bits (twice that where it is cut off), so that
    K / 32 + K / 128 + the joining of 16 parts stay below (K / 16 + 32) 2^-23 of it."""
    a, b = values(x), values(w)
    return a @ b.T, (a.abs() @ b.abs().T) * ((x.cols / 16 + 32) * 2.0 ** -23)


def gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


def gate(x, w, w2):
    """-> (gelu_tanh(x w^T) * (x w2^T), what it may be off): |gelu'| <= 1.13; the function's own hardware exponential and division 2^-20."""
    (g, dg), (u, du) = product(x, w), product(x, w2)
    h = gelu(g) * u
    return h, 1.13 * dg * (u.abs() + du) + gelu(g).abs() * du + h.abs() * 2.0 ** -20
