"""Attention and its gradient in 64 bits, one head of one sequence at a time, with a bound on how far a kernel of a given
element type may be from it, element by element.

Roundings that the bounds count: a product of n terms accumulated in fp32 errs by at most n 2^-23 of the sum of the terms'
sizes; the weights P and the score gradients dS are rounded once to the inputs' type (half a step, u, of their size; for
fp16 at least 2^-25, half its smallest step); results are rounded once more, by the same rule (an fp16
result below 2^-14 lies on a grid of 2^-24, whatever its size: u of its size alone would be too little); 2^x errs by 2^-21 of its value."""
import math

import torch

STEP = 2.0 ** -23
U = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FLOOR = {torch.float64: 0.0, torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def head(q, k, v, shift, causal, scale, dtype, do=None):
    """q [n, D], k and v [m, D] (any type), row i sees keys j <= i + shift.  Returns [(value, bound)] of out (dq, dk, dv)."""
    q, k, v = q.double(), k.double(), v.double()
    n, m, D = q.shape[0], k.shape[0], q.shape[1]
    u, floor, low = U[dtype], FLOOR[dtype], 0.0 if dtype == torch.float32 else U[dtype]
    i, j = torch.arange(n, device=q.device)[:, None], torch.arange(m, device=q.device)[None, :]
    seen = (j <= i + shift) if causal else torch.ones(n, m, dtype=torch.bool, device=q.device)
    some = seen.any(1, keepdim=True)
    s = (q @ k.T) * scale
    s_size = (q.abs() @ k.abs().T) * scale
    s_err = (D + 4) * STEP * s_size + 4 * STEP * s.abs()
    s = s.masked_fill(~seen, -math.inf)
    top = torch.where(some, s.amax(1, keepdim=True) if m else torch.zeros(n, 1, device=q.device).double(), 0.0)
    e = torch.exp(s - top)
    p = torch.where(some, e / e.sum(1, keepdim=True), 0.0)
    # relative error of a weight: of its score, of the row's maximum (as a multiple of it is subtracted), of 2^x
    worst = torch.where(seen, s_err, 0.0).amax(1, keepdim=True) if m else torch.zeros(n, 1, device=q.device).double()
    p_rel = 2 * (s_err + worst + 4 * STEP * top.abs()) + 8 * STEP + (m + 4) * STEP
    p_err = p * (p_rel + low) + floor * seen
    out = p @ v
    out_err = p_err @ v.abs() + (m + 4) * STEP * (p @ v.abs()) + u * out.abs() + floor
    out_err = out_err * (1 + 4 * u) + 1e-30
    if do is None:
        return [(out, out_err)]
    do = do.double()
    dp, dp_size = do @ v.T, do.abs() @ v.abs().T
    delta = (do * out).sum(1, keepdim=True)
    delta_err = (do.abs() * out_err).sum(1, keepdim=True) + (D + 4) * STEP * (do * out).abs().sum(1, keepdim=True)
    ds = p * (dp - delta)
    ds_err = p * p_rel * (dp - delta).abs() + p * ((D + 4) * STEP * dp_size + delta_err) + 4 * STEP * ds.abs()
    ds_err = ds_err + low * (ds.abs() + ds_err) + floor * seen
    got = [(out, out_err)]
    for a, a_err, b, f, terms in ((ds, ds_err, k, scale, m), (ds.T, ds_err.T, q, scale, n), (p.T, p_err.T, do, 1.0, n)):
        x = (a @ b) * f
        err = f * (a_err @ b.abs() + (terms + 4) * STEP * (a.abs() @ b.abs())) + u * x.abs() + floor
        got.append((x, err * (1 + 4 * u) + 1e-30))
    return got


def packed(q, k, v, lengths, key_lengths, causal, scale, do=None):
    """[(value, bound)] of out, dq, dk, dv for packed sequences; a shared head's gradient is the sum over its group, whose
    bounds add (the sum is one accumulation: no rounding between)."""
    H, Hk = q.shape[1], k.shape[1]
    zeros = lambda x: [torch.zeros(x.shape, dtype=torch.float64, device=x.device) for _ in range(2)]  # noqa: E731
    res = [zeros(q)] + ([zeros(q), zeros(k), zeros(v)] if do is not None else [])
    r = c = 0
    for n, m in zip(lengths, key_lengths):
        for h in range(H):
            g = h // (H // Hk)
            one = head(q[r:r + n, h], k[c:c + m, g], v[c:c + m, g], m - n, causal, scale, q.dtype, None if do is None else do[r:r + n, h])
            for slot, (value, bound) in enumerate(one):
                at = (slice(r, r + n), h) if slot < 2 else (slice(c, c + m), g)
                res[slot][0][at] += value
                res[slot][1][at] += bound
        r, c = r + n, c + m
    return res


def within(got, want, what=""):
    value, bound = want
    assert got.shape == value.shape, (what, got.shape, value.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got.double() - value).abs() - bound
    worst = int(over.argmax()) if over.numel() else 0
    assert not over.numel() or float(over.reshape(-1)[worst]) <= 0, (
        f"{what}: element {worst}: {float(got.reshape(-1)[worst]):.6e} for {float(value.reshape(-1)[worst]):.6e}, "
        f"bound {float(bound.reshape(-1)[worst]):.2e}; worst error {float((got.double() - value).abs().max()):.2e}")


def turned(x, positions, frequencies, interleaved, multiplier, sign=1.0):
    """(value, bound) of rotary positions: pairs as complex numbers."""
    R = 2 * frequencies.numel()
    y = x.double().clone()
    size = y.abs()
    i = torch.arange(R // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    angle = sign * positions.double()[:, None] * frequencies
    z = torch.complex(y[..., a], y[..., b]) * torch.polar(torch.full_like(angle, multiplier), angle)[:, None]
    both = (size[..., a] + size[..., b]) * abs(multiplier)
    y[..., a], y[..., b] = z.real, z.imag
    bound = torch.zeros_like(y)
    # cos and sin: half a step of an angle reduced to a quarter half-turn, the functions themselves, their scaling
    bound[..., a] = bound[..., b] = 8 * 2.0 ** -24 * both
    return y, bound + U[x.dtype] * y.abs() * (1 + 2.0 ** -7) + (2.0 ** -25 if x.dtype == torch.float16 else 0.0) * (bound > 0)
