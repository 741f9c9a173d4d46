"""Dense attention in 64 bits, one sequence and head at a time, with bounds of what rounding may do to the results
(for the tests of sddmm_attention_*; all on the CPU)."""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def ranges(n_q, n_k, left, right, prefix):
    """Positions of the rows and the keys [lo, hi) that each sees (include/sddmm.h)."""
    pos = torch.arange(n_q) + (n_k - n_q)
    lo = torch.zeros_like(pos) if left < 0 else (pos - left).clamp(min=0)
    hi = torch.full_like(pos, n_k) if right < 0 else torch.maximum(pos + right + 1, torch.full_like(pos, prefix)).clamp(max=n_k)
    return pos, lo, hi


def head(q, k, v, left, right, prefix, scale, cap, slope, dout=None):
    """One head of one sequence: a dict of results in 64 bits and, under "<name>_tol", how far results of the operands' type may be
    off.  With u = half a step of the type and e = 2^-24: a score is off by ds = e ((D + 8) scale sum|q k| + 8 |s| + 4 cap) at
    most (a product of D terms in fp32, its scaling, bending and bias), so a probability, relative to itself, by
    2 ds + (n + 32) e (its own score, the row's sum, n terms) and, rounded to the type, by u more."""
    u, e = HALF[q.dtype], 2.0 ** -24
    up = 0.0 if q.dtype == torch.float32 else u
    q, k, v = q.double(), k.double(), v.double()
    n_q, n_k, dim = len(q), len(k), q.shape[1]
    pos, lo, hi = ranges(n_q, n_k, left, right, prefix)
    j = torch.arange(n_k)
    seen = (j[None] >= lo[:, None]) & (j[None] < hi[:, None])
    far = (pos[:, None] - j[None]).abs().double()
    t = q @ k.T * scale
    bent = torch.tanh(t / cap) if cap else None
    s = bent * cap if cap else t.clone()
    s = s - slope * far
    ds = e * ((dim + 8) * scale * (q.abs() @ k.abs().T) + 8 * (s.abs() + slope * far) + 4 * cap)
    s = torch.where(seen, s, -math.inf)
    some = seen.any(1)
    top = torch.where(some, s.amax(1) if n_k else torch.zeros(n_q, dtype=torch.float64), 0.0)
    p = torch.exp(s - top[:, None])
    total = p.sum(1)
    lse = torch.where(some, top + torch.log(total), -math.inf)
    p = p / torch.where(some, total, 1.0)[:, None]
    worst = torch.where(seen, ds, 0.0).amax(1) if n_k else torch.zeros(n_q, dtype=torch.float64)
    rel = 2 * worst + (n_k + 32) * e  # of a probability
    out = p @ v
    r = dict(out=out, lse=lse)
    r["out_tol"] = u * out.abs() + (up + rel)[:, None] * 1.02 * (p @ v.abs()) + 1e-30
    r["lse_tol"] = worst + (n_k + 32) * e + 4 * e * torch.where(some, lse.abs(), 0.0)
    if dout is None:
        return r
    do = dout.double()
    dp = do @ v.T
    delta = (do * out).sum(1, keepdim=True)
    ds_ = p * (dp - delta)
    slope_of = 1 - bent ** 2 if cap else torch.ones_like(t)
    dt = ds_ * slope_of * scale
    r["dv"], r["dq"], r["dk"] = p.T @ do, dt @ k, dt.T @ q
    r["dslope"] = -(ds_ * far).sum()
    # what enters them: probabilities off by `rel` (and u where they are rounded), dp by (D + 8) e sum|do v|, delta by what the
    # output's own rounding and error make of it, the gradient of a score, rounded, by u; sums of n terms in fp32
    sums = (max(n_q, n_k) + 32) * e
    off_dp = (dim + 8) * e * (do.abs() @ v.abs().T)
    off_delta = (do.abs() * r["out_tol"]).sum(1, keepdim=True) + (dim + 8) * e * (do.abs() * out.abs()).sum(1, keepdim=True)
    # (1 - tanh^2 is off by 2 |tanh| times the bent score's own error, in units of cap)
    off_slope = 2 * (ds / cap) + 8 * e if cap else torch.zeros_like(t)
    off_ds = p * (off_dp + off_delta) + rel[:, None] * ds_.abs()
    off_dt = scale * (off_ds * slope_of + ds_.abs() * off_slope) + (up + 2 * e) * dt.abs()
    small = 0.0 if up == 0.0 or u == 2.0 ** -8 else 2.0 ** -25  # (fp16: steps below its normal range)
    r["dv_tol"] = u * r["dv"].abs() + ((p * (up + rel[:, None] + sums)) + small * seen).T @ do.abs() * 1.02 + 1e-30
    r["dq_tol"] = u * r["dq"].abs() + (off_dt + sums * dt.abs() + small * scale * seen) @ k.abs() * 1.02 + 1e-30
    r["dk_tol"] = u * r["dk"].abs() + (off_dt + sums * dt.abs() + small * scale * seen).T @ q.abs() * 1.02 + 1e-30
    r["dslope_tol"] = ((off_ds + (n_q * n_k + 32) ** 0.5 * 4 * e * ds_.abs()) * far).sum() + 1e-30
    if u == 2.0 ** -11:  # results below fp16's normal range
        for name in ("out", "dv", "dq", "dk"):
            r[name + "_tol"] = r[name + "_tol"] + 2.0 ** -25
    return r
