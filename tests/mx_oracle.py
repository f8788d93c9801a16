"""The microscaled operators in 64 bits, from their definition: rounding by a search in the table of an element's values."""
import math

import torch

BLOCK, PAD = 32, 256
LARGEST = {"fp4": 6.0, "fp8": 448.0}


def table(fmt):
    """The non-negative values of an element, by code."""
    if fmt == "fp4":
        return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    v = [m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)]
    return torch.tensor(v[:127], dtype=torch.float64)


def scale_exponent(amax, fmt):
    """The smallest e >= -127 with amax <= largest 2^e; 0 for 0."""
    if amax == 0:
        return 0
    e = math.floor(math.log2(amax / LARGEST[fmt])) - 1
    while amax > LARGEST[fmt] * 2.0 ** e:
        e += 1
    return max(e, -127)


def quantize(x, fmt, noise=None):
    """(codes, scales) of x (R x K, any dtype), as MxTensor stores them."""
    t = table(fmt)
    r, k = x.shape
    wide = -(-k // PAD) * PAD
    v = torch.zeros(r, wide, dtype=torch.float64)
    v[:, :k] = x.double()
    v = v.view(r, -1, BLOCK)
    u = torch.zeros(r, wide, dtype=torch.float64)
    if noise is not None:
        u[:, :k] = noise.double()
    u = u.view_as(v)
    amax = v.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    uniq, inverse = torch.unique(torch.where(bad, 0.0, amax), return_inverse=True)
    e = torch.tensor([scale_exponent(a, fmt) for a in uniq.tolist()], dtype=torch.float64)[inverse].view_as(amax)
    a = torch.where(bad[..., None], 0.0, v.abs()) / torch.exp2(e)[..., None]
    if noise is None:
        mids = (t[1:] + t[:-1]) / 2
        code = torch.bucketize(a, mids)
        tie = (code < len(mids)) & (mids[code.clamp(max=len(mids) - 1)] == a)
        code = code + (tie & (code % 2 == 1))
    else:
        code = (torch.bucketize(a, t, right=True) - 1)
        up = (code + 1).clamp(max=len(t) - 1)
        gap = torch.where(up > code, t[up] - t[code], 1.0)
        code = torch.where((a - t[code]) / gap + (u + 0.5) / 256 >= 1, up, code)
    sign = torch.signbit(v) & ~bad[..., None]
    code = code.reshape(r, wide) + sign.reshape(r, wide) * (8 if fmt == "fp4" else 128)
    scales = torch.where(bad, 255.0, e + 127).to(torch.uint8)
    if fmt == "fp4":
        code = code[:, 0::2] + 16 * code[:, 1::2]
    return code.to(torch.uint8), scales


def dequantize(codes, scales, k, fmt):
    t = table(fmt)
    t = torch.cat((t, -t)) if fmt == "fp4" else torch.cat((t, torch.tensor([math.nan], dtype=torch.float64), -t, torch.tensor([math.nan], dtype=torch.float64)))
    c = codes.long()
    if fmt == "fp4":
        c = torch.stack((c % 16, c // 16), -1).reshape(codes.shape[0], -1)
    s = torch.where(scales == 255, math.nan, torch.exp2(scales.double() - 127))
    return (t[c] * s.repeat_interleave(BLOCK, 1))[:, :k]


def rounded(x, fmt, noise=None):
    return dequantize(*quantize(x, fmt, noise), x.shape[1], fmt)


def norm(x, gain, residual, eps):
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    inv = 1 / torch.sqrt(s.double().square().mean(-1) + eps)
    return s, inv, s.double() * inv[:, None] * gain.double()


def norm_backward(dy, s, gain, inv, ds=None):
    s, dy, inv = s.double(), dy.double(), inv.double()[:, None]
    u, dg = s * inv, dy * gain.double()
    dx = inv * (dg - u * (dg * u).mean(-1, keepdim=True))
    return dx if ds is None else dx + ds.double(), (dy * u).sum(0)
