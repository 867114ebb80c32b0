"""Attention from its definition in 64 bits, with the elementwise bound that the kernels' arithmetic allows."""
import math

import torch


def attend(q, k, v, seen, scale):
    """q [n, Hq, D], k and v [m, Hk, D], seen [n] (keys 0 .. seen-1 of each row) -> (out, lse, sum p |v|) in float64.

    Keys that no row sees are left out; a key that only some rows see reaches only those, also where it holds NaN."""
    n, Hq, D = q.shape
    Hk = k.shape[1]
    G = Hq // Hk
    seen = seen.to(q.device)
    m = int(seen.max()) if n else 0
    out = torch.zeros(n, Hq, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    lse = torch.full((n, Hq), -math.inf, dtype=torch.float64, device=q.device)
    if m <= 0:
        return out, lse, mag
    qd = q.double().reshape(n, Hk, G, D)
    kd, vd = k[:m].double(), v[:m].double()
    s = torch.einsum("nhgd,mhd->nhgm", qd, kd) * scale
    hide = torch.arange(m, device=q.device)[None, :] >= seen[:, None]
    s = s.masked_fill(hide[:, None, None, :], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    clean = torch.nan_to_num(vd, nan=0.0, posinf=0.0, neginf=0.0)
    out = torch.einsum("nhgm,mhd->nhgd", torch.nan_to_num(p, nan=0.0), clean)
    mag = torch.einsum("nhgm,mhd->nhgd", torch.nan_to_num(p, nan=0.0), clean.abs())
    for j, h, d in (~torch.isfinite(vd)).nonzero().tolist():  # what is not finite reaches the rows that see it
        out[seen > j, h, :, d] += vd[j, h, d]
    nan_row = torch.isnan(lse)  # a score that is NaN or +Inf
    none = seen <= 0
    lse = lse.reshape(n, Hq)
    out = out.masked_fill(nan_row[..., None], math.nan)
    out, mag = out.reshape(n, Hq, D), mag.reshape(n, Hq, D)
    out[none], mag[none], lse[none] = 0.0, 0.0, -math.inf
    return out, lse, mag


def bound(out, mag, dtype, score_error=1e-4):
    """Elementwise bound of |kernel - out|, half steps u = eps / 2 of the 16-bit type:
    u for each softmax weight's rounding (sum of u p |v| = u mag), u |result| for the output's, and 2 score_error mag
    for the scores: fp32 sums of D <= 128 products (at most D 2^-24 sum |q k| scale, 5e-5 for the N(0, 1) inputs here),
    the exponent's argument and the approximate exp2 (2^-22)."""
    u = torch.finfo(dtype).eps / 2
    return u * mag + u * (out.abs() + u * mag) + 2 * score_error * mag + 1e-6


def check(got, out, mag, dtype, score_error=1e-4):
    got = got.double()
    fine = torch.isfinite(out)
    assert torch.equal(torch.isnan(got), torch.isnan(out)), "NaN at other places"
    assert torch.equal(got[~fine & ~torch.isnan(out)], out[~fine & ~torch.isnan(out)])
    off = ((got - out).abs() - bound(out, mag, dtype, score_error))[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, f"over the bound by {float(off.max()):.3e}"


def check_lse(got, lse, score_error=1e-4):
    """lse: the scores' error, and fp32 rounding of the value itself."""
    got = got.double()
    none = torch.isneginf(lse)
    assert torch.equal(torch.isneginf(got), none)
    fine = torch.isfinite(lse)
    assert float(((got - lse).abs() - score_error - 2.0 ** -22 * lse.abs())[fine].clamp(min=0).sum()) == 0
