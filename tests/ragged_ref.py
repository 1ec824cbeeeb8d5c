"""Plain 64-bit forms of the rotary positions, the paged cache and the attention of packed sequences, and the bounds
their 16-bit results are held to. Written from the definitions, one sequence and one head at a time."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def rope64(x, positions, inv_freq, interleaved=False, mscale=1.0):
    x = x.double()
    f = inv_freq.shape[0]
    ang = positions.double()[:, None, None] * inv_freq.double()
    cos, sin = torch.cos(ang) * mscale, torch.sin(ang) * mscale
    out = x.clone()
    a, b = (x[..., 0:2 * f:2], x[..., 1:2 * f:2]) if interleaved else (x[..., :f], x[..., f:2 * f])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    if interleaved:
        out[..., 0:2 * f:2], out[..., 1:2 * f:2] = ra, rb
    else:
        out[..., :f], out[..., f:2 * f] = ra, rb
    return out


def rope_bound(x, out64, inv_freq, interleaved=False, mscale=1.0):
    """Half a step of the type, plus fp32: sine and cosine within 2^-22 (2 ulps, and the angle's remainder of at most
    pi / 4 rounded once), two products and a sum of 2^-24 each: less than 2^-21 (|a| + |b|) mscale in all. fp16 results
    below 2^-14 step by 2^-24."""
    f = inv_freq.shape[0]
    x = x.double().abs()
    mag = torch.zeros_like(x)
    if interleaved:
        s = x[..., 0:2 * f:2] + x[..., 1:2 * f:2]
        mag[..., 0:2 * f:2], mag[..., 1:2 * f:2] = s, s
    else:
        s = x[..., :f] + x[..., f:2 * f]
        mag[..., :f], mag[..., f:2 * f] = s, s
    return mag * mscale * 2.0 ** -21


def check(got, want, extra, dtype):
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    err = (got.double() - want).abs()
    tol = HALF_STEP[dtype] * (want.abs() + extra) + extra + tiny
    assert torch.isfinite(got).all()
    worst = (err - tol).max().item() if err.numel() else -1
    assert worst <= 0, f"off by {err.max().item():.3e}, {worst:.3e} more than allowed"


def pages_of(k_cache, table, b, length):
    """[length, kv_heads, dim] of sequence b."""
    ps = k_cache.shape[1]
    j = torch.arange(length, device=k_cache.device)
    return k_cache[table[b, j // ps].long(), j % ps]


def attend64(q, k, v, scale=None, causal=True, softcap=0.0, window=0, slopes=None, prefix=0):
    """q [n, H, D], k and v [m, Hkv, D] of one sequence. Returns (out, lse, allowance): float64 [n, H, D], [n, H] and
    sum_j softmax_ij |v_j|, which the allowance for 16-bit weights is a multiple of."""
    n, H, D = q.shape
    m, Hkv = k.shape[0], k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    pos = torch.arange(n, device=q.device)[:, None] + (m - n)
    key = torch.arange(m, device=q.device)[None, :]
    seen = torch.ones((n, m), dtype=torch.bool, device=q.device)
    if causal:
        seen &= (key <= pos) | (key < prefix)
    if window:
        seen &= pos - key < window
    out = torch.zeros((n, H, D), dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    lse = torch.full((n, H), -math.inf, dtype=torch.float64, device=q.device)
    for h in range(H):
        kk, vv = k[:, h * Hkv // H].double(), v[:, h * Hkv // H].double()
        s = q[:, h].double() @ kk.t() * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:
            s = s - slopes[h].double() * (pos - key).abs()
        for i in range(n):
            j = seen[i].nonzero().flatten()
            if len(j):
                w = torch.softmax(s[i, j], 0)
                out[i, h], mass[i, h] = w @ vv[j], w @ vv[j].abs()
                lse[i, h] = torch.logsumexp(s[i, j], 0)
    return out, lse, mass


def attend_check(got, out64, mass, dtype, keys, vmax):
    """The kernel rounds each weight to the inputs' type (half a step, relative), and its scores are off by less than
    1e-4 in the base-2 exponent (fp32 sums of dim products, 2^-22 exponentials, the cap's cancellation): 2e-4 in the
    weight and as much in the sum. fp16 weights, scaled to a maximum of at least 1, step by 2^-24 below 2^-14."""
    under = keys * 2.0 ** -25 * vmax if dtype == torch.float16 else 0.0
    extra = (HALF_STEP[dtype] + 4e-4) * mass + under
    check(got, out64, extra, dtype)
