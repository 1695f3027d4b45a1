"""Latent attention in 64 bits, expanded and absorbed, with a bound on what a flash kernel (fp32
scores and sums, P rounded to the input type before P V) may differ by before its own rounding."""
from __future__ import annotations

import torch


def _attend(q, k, v, see, scale, dt):
    """One head: q [n, d], k [m, d], v [m, e] float64, see [n, m] bool -> (out, tol) [n, e]; rows
    that see nothing are zero.

    Scores: sums of d exact products in fp32, at most d / 16 + 1 steps each off by 2^-22 of the
    magnitudes: ds. Each weight is then off by 2 ds (its own and the maximum's) + 2^-20 (exp2,
    rescales) relative, and by half a step of dt from the rounding of P; the sums over the keys by
    m / 16 steps of 2^-22. Everything scales sum_j p_j |v_j|; the normaliser's error does too. In
    fp16 a weight below 2^-14 is off by up to 2^-25 of the largest one instead."""
    s = q @ k.t() * scale
    mag = (q.abs() @ k.abs().t() * scale).masked_fill(~see, 0).amax(-1, keepdim=True)
    s = s.masked_fill(~see, float('-inf'))
    any_ = see.any(-1, keepdim=True)
    p = torch.where(any_, torch.softmax(s, -1), torch.zeros_like(s))
    out = p @ v
    ds = (q.shape[1] / 16 + 1) * 2. ** -22 * mag
    rel = 2 * (2 * ds + 2. ** -20) + torch.finfo(dt).eps / 2 + k.shape[0] / 16 * 2. ** -22
    tol = rel * (p @ v.abs())
    if dt == torch.float16:
        tol = tol + 2. ** -25 * (see.double() @ v.abs())
    return out, torch.where(any_, tol, torch.zeros_like(tol))


def fwd_causal(q_nope, q_rope, k_nope, k_rope, v, scale, q_start=None, kv_lens=None):
    """q [B, H, Sq, *], k_nope / v [B, H, Skv, 128], k_rope [B, Skv, 64] -> (out, tol)
    [B, Sq, H, 128]."""
    dt = q_nope.dtype
    qn, qr, kn, kr, vv = (t.cpu().double() for t in (q_nope, q_rope, k_nope, k_rope, v))
    B, H, Sq, _ = qn.shape
    Skv = kn.shape[2]
    out = torch.zeros(B, Sq, H, vv.shape[-1], dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = Skv if kv_lens is None else max(0, min(Skv, int(kv_lens[b])))
        first = Skv - Sq if q_start is None else int(q_start[b])
        if n == 0:
            continue
        see = torch.arange(n)[None] <= first + torch.arange(Sq)[:, None]
        for h in range(H):
            out[b, :, h], tol[b, :, h] = _attend(
                torch.cat([qn[b, h], qr[b, h]], -1), torch.cat([kn[b, h, :n], kr[b, :n]], -1),
                vv[b, h, :n], see, scale, dt)
    return out, tol


def decode(q_latent, q_rope, ckv, k_rope, block_table, kv_lens, scale):
    """q_latent [B, Sq, H, 512], pages ckv [P, ps, 512] / k_rope [P, ps, 64]; keys on a page number
    outside the pool are not attended -> (out, tol) [B, Sq, H, 512]."""
    dt = q_latent.dtype
    ql, qr = q_latent.cpu().double(), q_rope.cpu().double()
    c, kr, tab = ckv.cpu().double(), k_rope.cpu().double(), block_table.cpu().long()
    B, Sq, H, _ = ql.shape
    P, ps = c.shape[:2]
    out = torch.zeros(B, Sq, H, c.shape[-1], dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = max(0, min(int(kv_lens[b]), tab.shape[1] * ps))
        if n == 0:
            continue
        j = torch.arange(n)
        page = tab[b, j // ps]
        ok = (page >= 0) & (page < P)
        kc, kk = c[page.clamp(0, P - 1), j % ps], kr[page.clamp(0, P - 1), j % ps]
        kc, kk = kc.masked_fill(~ok[:, None], 0), kk.masked_fill(~ok[:, None], 0)
        for i in range(Sq):
            see = (ok & (j <= n - Sq + i))[None].expand(H, n)
            out[b, i], tol[b, i] = _attend(torch.cat([ql[b, i], qr[b, i]], -1),
                                           torch.cat([kc, kk], -1), kc, see, scale, dt)
    return out, tol


def close(got, y, tol) -> bool:
    """got within tol of y plus half a step of got's type (and its smallest subnormal)."""
    fi = torch.finfo(got.dtype)
    room = tol + (y.abs() + tol) * fi.eps / 2 + fi.tiny * fi.eps
    return bool(((got.cpu().double() - y).abs() <= room).all())
