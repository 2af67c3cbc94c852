"""The operators between the q | k | v projection and the output projection, from their definitions in 64 bits, and the
bounds their rounded results must keep (used by the CPU and the GPU tests)."""

import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}  # half the smallest subnormal


def speeds(rot, base, scaling="none", factor=1.0, original_len=0.0, fast=32.0, slow=1.0):
    """Radians per position of each pair, and the amplitude."""
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    w = [base ** (-2 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        w = [x / factor for x in w]
    if scaling == "yarn":
        ramp = [min(1.0, max(0.0, (original_len * x / (2 * math.pi) - slow) / (fast - slow))) for x in w]
        w = [x * r + x / factor * (1 - r) for x, r in zip(w, ramp)]
    return torch.tensor(w, dtype=torch.float64), 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0


def rotate64(x, positions, w, amplitude, interleaved):
    """x [T, H, D] float64; also the magnitude amplitude * (|a| + |b|) that a rotated value's errors are relative to."""
    rot = 2 * len(w)
    angle = positions.double()[:, None, None] * w.to(x.device)
    c, s = torch.cos(angle) * amplitude, torch.sin(angle) * amplitude
    y, mag = x.clone(), x.abs().clone()
    ia = torch.arange(0, rot, 2, device=x.device) if interleaved else torch.arange(rot // 2, device=x.device)
    ib = ia + (1 if interleaved else rot // 2)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = amplitude * (a.abs() + b.abs())
    return y, mag


def norm64(x, weight, eps, zero_centred):
    w = weight.double() + 1 if zero_centred else weight.double()
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w


def rotation_bound(y, mag, dtype, dim, normed):
    """One rounding to the output's type; before it, in fp32: the angle's cos and sin (2^-22 of the magnitude: the reduced
    angle rounded once, the function within 2 ulp, the amplitude), two products and a sum (3 half steps); with the norm, the sum of squares
    (at most dim half steps, half of it after the root), the root (2 ulp) and three products."""
    u = 2.0 ** -24
    fp32 = 4 * u + 3 * u + ((dim / 2 + 8) * u if normed else 0)
    return HALF_STEP[dtype] * y.abs() * (1 + 2.0 ** -7) + fp32 * mag + TINY[dtype] + 1e-37


def sees(positions, j, window, sinks):
    ok = j[None, :] <= positions[:, None]
    if window:
        ok &= (j[None, :] > positions[:, None] - window) | (j[None, :] < sinks)
    return ok


def attention64(q, k, v, new, kv, window, sinks, scale):
    """One sequence: q [new, H, D], k and v [kv, Hk, D] in their own types -> out, lse and the bound on out (float64).

    The bound: the result is rounded once (half a step of its type, relative to it); each probability is rounded once
    to the inputs' type before it meets its value, which moves the result by at most half a step of sum p |v|; a score is an fp32
    sum of D products (at most (D + 8) 2^-24 of scale sum |q| |k|), which changes a probability by that and the normaliser
    by no more; exp and the sums over the keys stay within 2^-20 of sum p |v| + (keys 2^-24) of it. A probability below
    the type's subnormals is lost whole: keys * half the smallest one * max |v|. Doubled rounding steps meet at most once more."""
    dt = q.dtype
    H, D = q.shape[1], q.shape[2]
    G = H // max(k.shape[1], 1)
    out = torch.zeros(new, H, D, dtype=torch.float64, device=q.device)
    bound = torch.full_like(out, 1e-30)
    lse = torch.full((new, H), -math.inf, dtype=torch.float64, device=q.device)
    lse_bound = torch.full_like(lse, 0.0)
    if new == 0 or kv == 0:
        return out, lse, bound, lse_bound
    pos = torch.arange(kv - new, kv, device=q.device)
    ok = sees(pos, torch.arange(kv, device=q.device), window, sinks)
    live = ok.any(-1)
    u = HALF_STEP[dt]
    for h in range(H):
        K, V, Q = k[:, h // G].double(), v[:, h // G].double(), q[:, h].double()
        s = (Q @ K.T * scale).masked_fill(~ok, -math.inf)
        err = ((D + 8) * 2.0 ** -24 * abs(scale) * (Q.abs() @ K.abs().T)).masked_fill(~ok, 0).amax(-1, keepdim=True) + 2.0 ** -20 + kv * 2.0 ** -24
        p = torch.softmax(s, -1).masked_fill(~live[:, None], 0)
        Vs = V.masked_fill(~ok.any(0)[:, None], 0)  # what no row sees plays no part, whatever it holds
        o = p @ Vs
        spread = p @ Vs.abs()
        out[:, h] = o
        e = (u + 2 * err) * spread + kv * TINY[dt] * Vs.abs().max()
        bound[:, h] = (u * o.abs() + e) * (1 + 2.0 ** -6) + TINY[dt]
        lse[:, h] = torch.logsumexp(s, -1).masked_fill(~live, -math.inf)
        # the normaliser's relative error, and fp32's rounding of m + ln l
        lse_bound[:, h] = (2 * err[:, 0] + 2.0 ** -22 * (1 + lse[:, h].abs())).masked_fill(~live, 0)
    return out, lse, bound, lse_bound
