"""Rings of 4 bits and attention over them, from the definitions, in 64 bits and one number after the other where that is clearest; how far a kernel's
result may be from them.  Runs where its tensors are."""
import math

import torch

FIFTEENTH = float(torch.tensor(1 / 15, dtype=torch.float32))


def bf16_toward(v, direction):
    """v, a finite number of fp32's, to one of bf16's: 8 bits, and steps of 2^-133 below 2^-126; zeros without a sign."""
    grid = torch.frexp(v).exponent.clamp(min=-125) - 8
    return torch.ldexp(direction(torch.ldexp(v, -grid)), grid) + 0.0


def f32(v):
    """A number of 64 bits rounded to fp32 (sums, products and quotients of two fp32 numbers come out as fp32's own: 53 bits are twice 24 and more)."""
    return v.float().double()


def numbers(x):
    """float64 [..., dims] of one piece -> (lowest, step, n)."""
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    x = torch.where(bad, 0.0, x)
    low = bf16_toward(x.amin(-1, keepdim=True), torch.floor)
    spread = f32(x.amax(-1, keepdim=True) - low)
    bad = bad | ~torch.isfinite(spread)
    step = bf16_toward(f32(torch.where(bad, 0.0, spread) * FIFTEENTH), torch.ceil)
    step = torch.where(step > 0, step.clamp(min=2.0 ** -126), step)
    bad = bad | ~torch.isfinite(step.float()) | ~torch.isfinite(low.float())
    inverse = torch.where(step > 0, f32(1 / step), 0.0)
    n = torch.round(f32(f32(x - low) * inverse)).clamp(0, 15)
    return torch.where(bad, math.nan, low), torch.where(bad, 0.0, step), torch.where(bad, 0.0, n)


def held(x):
    """What a key or value [..., hd] of fp32 numbers stands for in a ring, float64."""
    out = []
    for piece in x.double().split(64, -1):
        low, step, n = numbers(piece)
        out.append(low + step * n)
    return torch.cat(out, -1)


def width(hd):
    return 32 if hd <= 32 else 64 if hd <= 64 else 128


def ring_bytes(x):
    """x [..., slots, hd] of fp32 numbers -> the bytes of a ring [..., slots * row] whose every slot holds one."""
    lead, slots, hd = x.shape[:-2], x.shape[-2], x.shape[-1]
    pieces = list(x.double().split(64, -1))
    rows = torch.zeros(*lead, slots, width(hd) // 2, dtype=torch.int64, device=x.device)
    scales = torch.zeros(*lead, slots, len(pieces), 4, dtype=torch.int64, device=x.device)
    for p, piece in enumerate(pieces):
        low, step, n = numbers(piece)
        for c in range(piece.shape[-1]):
            byte = 4 * (c // 8 * len(pieces) + p) + c % 8 // 2
            rows[..., byte] += n[..., c].long() << 4 * (c & 1)
        for i, v in enumerate((low, step)):
            bits = v[..., 0].to(torch.bfloat16).view(torch.int16).long() & 0xffff
            bits = torch.where(v[..., 0].isnan(), 0x7fc0, bits)
            scales[..., p, 2 * i], scales[..., p, 2 * i + 1] = bits & 255, bits >> 8
    return torch.cat([rows.flatten(-2), scales.flatten(-3)], -1).to(torch.uint8)


def parts(ring, hd):
    """(rows [B, heads, slots, bytes], scales [B, heads, slots, bytes]) as views."""
    row, scale = width(hd) // 2, 8 if hd > 64 else 4
    slots = ring.shape[2] // (row + scale)
    return ring[:, :, :slots * row].unflatten(2, (slots, row)), ring[:, :, slots * row:].unflatten(2, (slots, scale))


def values(ring, hd):
    """What a ring stands for, float64 [B, heads, slots, hd]."""
    rows, scales = parts(ring, hd)
    pieces = 2 if hd > 64 else 1
    s = scales.contiguous().view(torch.bfloat16).double()
    out = []
    for c in range(hd):
        p = c // 64
        byte = rows[..., 4 * (c % 64 // 8 * pieces + p) + c % 8 // 2].long()
        out.append(s[..., 2 * p] + s[..., 2 * p + 1] * (byte >> 4 * (c & 1) & 15).double())
    return torch.stack(out, -1)


def attention(q, k, v, behind, seen, slope, cap, coarse=None):
    """q [n, hd], k, v [m, hd], behind, seen [n, m] -> (out [n, hd], tolerance ingredients).  coarse: (|k|, |v|) as large as the kernel's own terms get."""
    hd = q.shape[1]
    scale = hd ** -0.5
    z = q @ k.T * scale
    bent = cap * torch.tanh(z / cap) if cap else z
    s = torch.where(seen, bent - slope * behind, -math.inf)
    w = torch.softmax(s, 1)
    w = torch.where(seen, w, 0.0)
    v0 = torch.where(seen.any(0)[:, None], v, 0.0)   # (what nobody sees may be anything)
    ka, va = (k.abs(), v0.abs()) if coarse is None else coarse
    terms = (q.abs() @ torch.where(seen.any(0)[:, None], ka, 0.0).T * scale)
    big = lambda t: torch.where(seen, t, 0.0).amax(1, keepdim=True)  # noqa: E731
    spread = big((s.amax(1, keepdim=True) - s).nan_to_num(0.0, 0.0, 0.0))
    return w @ v0, dict(a=w @ v0.abs(), coarse=w @ torch.where(seen.any(0)[:, None], va, 0.0), terms=big(terms), score=big(bent.abs()), spread=spread,
                        far=big(slope * behind.abs().double()), hd=hd, keys=int(seen.sum(1).max()))


def tolerance(out, t, dtype, weights, tanh):
    """How far a kernel's row may be off.  weights: how far its rounding moves a weight (0: held in fp32); tanh: relative error of the soft cap it uses.
      scores    sums of hd products in fp32, in chains of at most hd (2^-24 each of their terms, and as much for what a scale or its rounding adds: x 2);
                the cap moves one by its own error, ALiBi's product and difference by 2^-23 of it
      weights   twice what moves a score (numerator and denominator); exp2's own error and that of its argument, 2^-22 (spread + 4); their rounding
      sums      chains of a 64th of the keys, and 32 to join them, 2^-23 each, of terms as large as the kernel's own
      result    half a step of its type"""
    moved = t["terms"] * (t["hd"] + 8) * 2.0 ** -23 + t["score"] * tanh + (t["far"] + t["score"]) * 2.0 ** -23
    return (out.abs() * torch.finfo(dtype).eps / 2 + t["a"] * (2 * moved + (t["spread"] + 4) * 2.0 ** -22 + weights)
            + t["coarse"] * (t["keys"] / 64 + 32) * 2.0 ** -23)


# tanh: the hardware's, relative error 2^-11 (bf16); the library's, 2 units in the last place (fp32).  weights: rounded to bf16 (packed prompts in bf16), or
# in two bf16 parts, 2^-17 (a step in bf16), or in three, 2^-25 (in fp32; where they are held in fp32 there is none).
TANH = {torch.bfloat16: 2.0 ** -11, torch.float32: 2.0 ** -22}
WEIGHTS_PACKED = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
WEIGHTS_STEP = {torch.bfloat16: 2.0 ** -16, torch.float32: 2.0 ** -24}


def packed(qkv, lengths, first, slopes, H, kv, window, cap, dtype):
    """(out [N, H hd] float64 with NaN where no sequence is, tolerance of the same shape)"""
    x = qkv.double().view(qkv.shape[0], H + 2 * kv, -1)
    hd = x.shape[2]
    out = torch.full((qkv.shape[0], H, hd), math.nan, dtype=torch.float64, device=qkv.device)
    tol = torch.zeros_like(out)
    at = first
    for n in lengths:
        if n:
            p = torch.arange(n, device=qkv.device)
            behind = p[:, None] - p
            seen = (behind >= 0) if window is None else (behind >= 0) & (behind <= window)
            for h in range(H):
                g = h * kv // H
                o, t = attention(x[at:at + n, h], x[at:at + n, H + g], x[at:at + n, H + kv + g], behind, seen, float(slopes[h]) if slopes is not None else 0.0,
                                 cap)
                out[at:at + n, h], tol[at:at + n, h] = o, tolerance(o, t, dtype, WEIGHTS_PACKED[dtype], TANH[dtype])
        at += n
    return out.flatten(1), tol.flatten(1)


def step(qkv, k4, v4, pos, slopes, H, window, cap, dtype):
    """(out [B, 1, H hd] float64, tolerance) of one token per sequence."""
    B, kv = k4.shape[:2]
    x = qkv.double().view(B, H + 2 * kv, -1)
    hd = x.shape[2]
    out = torch.empty(B, 1, H, hd, dtype=torch.float64, device=qkv.device)
    tol = torch.empty_like(out)
    # (in bf16 a number n enters the products as 128 + n, and what that adds is taken off the sum)
    top = 143 if dtype == torch.bfloat16 else 15
    for b in range(B):
        t = int(pos[b, 0])
        both, coarse = [], []
        for i, ring in enumerate((k4, v4)):
            slots = parts(ring, hd)[0].shape[2]
            j = torch.arange(max(0, t - window), t, device=qkv.device)
            both.append(torch.cat([values(ring[b:b + 1], hd)[0][:, j % slots], x[b, H + i * kv:H + (i + 1) * kv, None]], 1))
            s = parts(ring[b:b + 1], hd)[1][0].contiguous().view(torch.bfloat16).double()[:, j % slots]
            large = torch.cat([(s[..., 2 * (c // 64)].abs() + top * s[..., 2 * (c // 64) + 1])[..., None] for c in range(hd)], -1)
            coarse.append(torch.cat([large, both[-1][:, -1:].abs()], 1))
        behind = torch.cat([t - j, j.new_zeros(1)])[None]
        for h in range(H):
            g = h * kv // H
            o, tt = attention(x[b, h][None], both[0][g], both[1][g], behind, torch.ones_like(behind, dtype=torch.bool),
                              float(slopes[h]) if slopes is not None else 0.0, cap, (coarse[0][g], coarse[1][g]))
            out[b, 0, h], tol[b, 0, h] = o[0], tolerance(o, tt, dtype, WEIGHTS_STEP[dtype], TANH[dtype])[0]
    return out.flatten(2), tol.flatten(2)


def check(got, want, tol):
    """Within the tolerance, NaN where the reference is."""
    assert got.shape == want.shape
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    off = ((got - want).abs() - tol).nan_to_num(0.0)
    assert bool((off <= 0).all()), f"{float((off > 0).double().mean()):.2g} of the values are off by up to {float(((got - want).abs() / tol).nan_to_num(0).max()):.3g} x the tolerance"
