"""Plain 64-bit forms of the paged cache's operators, for the tests: rotation,
the 4-bit format, and attention over whole sequences, with the error bounds
that the tests hold the kernels to."""
import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def unit(rows):
    """Half a rounding step of the type, relative to the value."""
    return torch.finfo(TYPES[rows]).eps / 2


def rotate(x, pos, freq, scale=1.0, interleaved=False):
    """x [rows, heads, D] (f64), pos [rows], freq [pairs]."""
    y = x.double().clone()
    n = len(freq)
    if n == 0:
        return y
    ang = pos.double()[:, None] * torch.as_tensor(freq, dtype=torch.float64)
    c, s = torch.cos(ang)[:, None] * scale, torch.sin(ang)[:, None] * scale
    a = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    b = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    p, q = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = p * c - q * s, p * s + q * c
    return y


def mxfp4(x):
    """Values that a 4-bit cache holds for x [..., D] (f64): per block of 32 a
    scale 2^(floor(log2 max) - 2), at least 2^-127; nearest code, ties to the
    even one; NaN where the block holds an infinity or NaN."""
    b = x.double().reshape(-1, 32)
    top = b.abs().amax(1, keepdim=True)
    bad = ~torch.isfinite(b).all(1, keepdim=True)
    e = (torch.frexp(torch.where(bad, 0.0, top))[1].double() - 3).clamp(min=-127)
    step = torch.exp2(torch.where(top > 0, e, -127.0))
    m = (b.abs() / step).clamp(max=6)
    d = (m[..., None] - CODES).abs()
    near = d == d.amin(-1, keepdim=True)
    even = near & (torch.arange(8) % 2 == 0)
    pick = torch.where(even.any(-1), even.double().argmax(-1), near.double().argmax(-1))
    out = torch.where(bad, math.nan, CODES[pick] * step * torch.sign(b))
    return out.reshape(x.shape)


def held(x, cache):
    """x (f64) as the cache holds it."""
    return mxfp4(x) if cache == "mxfp4" else x.to(TYPES[cache]).double()


def attend(q, k, v, pos, rows, cache, scale=None, cap=0.0, slopes=None, sinks=None, window=0, first=None, prefix=0):
    """Attention of q [n, H, D] at positions pos [n] over k, v [L, KV, D] (f64).
    Returns (out, tol): the exact result and how far a kernel may be from it.

    The bound: a product of D terms in f32 is off by at most
    (D + 8) 2^-23 sum|q k| (2^-23: a tensor-core add may truncate), times
    scale; the transforms after it by a few units of the score's own size; so a
    weight by twice that (the maximum is off as well), and the sum of L weighted
    values by (L + 16) 2^-23 more.  Rows of 16 bits round each weight once (half
    a step) and, like every type, the result once.

    f16 weights (f16 rows, and every 16-bit row over a 4-bit cache, where the
    weight carries the block's scale) have a smallest step of 2^-24, half of
    which is an absolute error; the kernels lift the largest weight to 2^9 or
    more, so it is at most 2^-34 of the largest weight, for each seen value of
    up to |v| (4 bits: 6 times the largest seen scale of the block, which is at
    most twice the block's largest |v|, so 2^-33 * 6 * max|v|)."""
    n, H, D = q.shape
    L, KV = k.shape[0], k.shape[1]
    G = H // KV
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(n, H, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    j = torch.arange(L)
    see = (j[None] <= pos[:, None]) | (j[None] < prefix)
    if first is not None:
        see &= j[None] >= first[:, None]
    if window:
        see &= j[None] > pos[:, None] - window
    u, ulp = unit(rows), 2.0 ** -23
    least = torch.finfo(TYPES[rows]).smallest_normal * torch.finfo(TYPES[rows]).eps / 2  # half a step among subnormals
    for h in range(H):
        kk, vv, qq = k[:, h // G], v[:, h // G], q[:, h].double()
        for i in range(n):
            sel = see[i]
            if not sel.any():
                continue
            ks, vs = kk[sel], vv[sel]
            s = (ks @ qq[i]) * scale
            err = (D + 8) * ulp * (ks.abs() @ qq[i].abs()) * abs(scale)
            if cap:
                s = cap * torch.tanh(s / cap)
                err = err + 4 * ulp * cap
            if slopes is not None:
                far = (pos[i] - j[sel]).abs().double()
                s = s - float(slopes[h]) * far
                err = err + 4 * ulp * abs(float(slopes[h])) * far
            err = err + 8 * ulp * (s.abs() + 1)
            top = s.max()
            if sinks is not None:
                top = torch.maximum(top, torch.as_tensor(float(sinks[h]), dtype=torch.float64))
            w = torch.exp(s - top)
            total = w.sum() + (math.exp(float(sinks[h]) - float(top)) if sinks is not None else 0.0)
            p = w / total
            out[i, h] = p @ vs
            e = err[torch.isfinite(err)]
            e = float(e.max()) if len(e) else 0.0
            size = p @ vs.abs()
            if rows != "f32" and cache == "mxfp4":
                top_v = vs.abs().reshape(len(vs), -1, 32).amax((0, 2)).repeat_interleave(32)
                floor = len(vs) * 2.0 ** -33 * float(p.max()) * 6 * torch.nan_to_num(top_v, 0, 0)
            elif rows == "f16":
                floor = 2.0 ** -34 * float(p.max()) * vs.abs().sum(0)
            else:
                floor = 0.0
            tol[i, h] = (2 * e + (L + 16) * ulp + (u if rows != "f32" else 0.0)) * 1.01 * size + u * out[i, h].abs() + least + floor
    return out, tol
