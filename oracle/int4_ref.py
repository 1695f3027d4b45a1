"""Products with 4-bit packed weights in 64 bits, on the deploy layouts' words
(module_utils.py:929-955 vLLM, :1097-1158 AutoAWQ), with a bound on what fp32 sums may lose."""
from __future__ import annotations

import torch

AWQ_COLUMN = (0, 2, 4, 6, 1, 3, 5, 7)   # column of nibble i


def _nibbles(words: torch.Tensor) -> torch.Tensor:
    """[rows, w] int32 -> [rows, w, 8] codes, nibble order."""
    w = words.cpu().to(torch.int64) & 0xffffffff
    return torch.stack([(w >> (4 * i)) & 15 for i in range(8)], -1)


def _awq_columns(words: torch.Tensor) -> torch.Tensor:
    nib = _nibbles(words)
    out = torch.empty_like(nib)
    for i, c in enumerate(AWQ_COLUMN):
        out[..., c] = nib[..., i]
    return out.reshape(out.shape[0], -1)


def unpack(qweight, scales, qzeros=None):
    """(codes, zeros, scales) [n, k] float64 of a packed weight (zero point 8 without qzeros)."""
    s = scales.cpu().double()
    if qzeros is None:
        c = _nibbles(qweight).reshape(qweight.shape[0], -1)
        g = c.shape[1] // s.shape[1]
        return c.double(), torch.full(c.shape, 8., dtype=torch.float64), s.repeat_interleave(g, 1)
    c, z = _awq_columns(qweight), _awq_columns(qzeros)
    g = c.shape[0] // s.shape[0]
    return (c.t().double(), z.t().double().repeat_interleave(g, 1),
            s.t().repeat_interleave(g, 1))


def linear(x, qweight, scales, qzeros=None, bias=None):
    """(y, tol) float64: the product, and how far an fp32-accumulated one may be from it before
    its rounding to the output type.

    A kernel may form s (sum x u - (16 + z) sum x) with u = 16 + code. Products are exact in fp32.
    A sum runs over at most K / 32 steps of 32 products; a step's error is at most 2^-22 of the
    sum of magnitudes so far, so the group sums lose at most (g / 32 + 1) 2^-22 sum |x| (u + 16 +
    z) s, and the sum over groups and partial sums (K / g + 16 terms) as many 2^-23 of
    sum |x| |w|."""
    c, z, s = unpack(qweight, scales, qzeros)
    xd = x.cpu().double()
    w = (c - z) * s
    g = w.shape[1] // (scales.shape[1] if qzeros is None else scales.shape[0])
    y = xd @ w.t()
    ax = xd.abs()
    tol = ((g / 32 + 1) * 2. ** -22 * (ax @ ((c + 16 + 16 + z) * s.abs()).t())
           + (w.shape[1] / g + 16) * 2. ** -23 * (ax @ w.abs().t()))
    if bias is not None:
        y = y + bias.cpu().double()
        tol = tol + 2. ** -23 * y.abs()
    return y, tol


def silu_mul(g, u):
    """silu(g) u of two (value, tol) pairs: |silu'| <= 1.1; the fp32 exp, divide and products
    within 2^-20 of the value."""
    (gv, gt), (uv, ut) = g, u
    h = gv * torch.sigmoid(gv)
    y = h * uv
    return y, 1.1 * gt * (uv.abs() + ut) + (h.abs() + 1.1 * gt) * ut + 2. ** -20 * y.abs()


def close(got, y, tol) -> bool:
    """got within tol of y plus half a step of got's type (and its smallest subnormal)."""
    fi = torch.finfo(got.dtype)
    room = tol + (y.abs() + tol) * fi.eps / 2 + fi.tiny * fi.eps
    return bool(((got.cpu().double() - y).abs() <= room).all())
