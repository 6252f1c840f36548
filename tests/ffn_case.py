"""Float64 restatements of the dense gated block and of MXFP4, with bounds on what the kernels may be off.

A bound is a sum over what is rounded on the way to a value, element by element:
  * a float32 sum of K products is off by at most 2 K 2^-24 times the sum of the products' magnitudes;
  * a value stored in bfloat16 is off by at most 2^-8 of itself, one in float32 by 2^-24 (`half`);
  * below 2^-126 float32 has no more relative precision: its numbers lie 2^-149 apart there, and each product and
    each stored value may be off by half of that too (`TINY`, taken whole);
  * sigmoid(w) is off by (4 + 4 |w|) 2^-24 of itself with the library's exponential and division
    (float32 layers: one step each for w, exp, 1 + e and the division, and |w| of w's own), and by
    (8 + 8 |w|) 2^-23 with the hardware's (bfloat16 layers).
"""
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TINY = 2.0 ** -149
C = (2.0 / torch.pi) ** 0.5


def parts(g, act):
    """(a, slope, w, dw) of the activation in float64."""
    if act == "silu":
        w, dw = g, torch.ones_like(g)
    else:
        w, dw = 2 * C * (g + 0.044715 * g ** 3), 2 * C * (1 + 3 * 0.044715 * g ** 2)
    s = torch.sigmoid(w)
    return g * s, s + g * s * (1 - s) * dw, w, dw, s


def _sum_error(K):
    return 2.0 * K * 2.0 ** -24


def block(x, w13, w2, act, dy=None):
    """{name: (value, bound)} of y and, with dy, dx, dw13 and dw2; all float64, for inputs of x's dtype."""
    half = HALF[x.dtype]
    unit = 2.0 ** -24 if x.dtype == torch.float32 else 2.0 ** -22
    X, W13, W2 = (t.detach().double().reshape(-1, t.shape[-1]) for t in (x, w13, w2))
    H, I = W2.shape
    Wg, Wu = W13[:I], W13[I:]
    g, u = X @ Wg.t(), X @ Wu.t()
    eg, eu = (_sum_error(H) * (X.abs() @ w.abs().t()) + H * TINY for w in (Wg, Wu))
    a, slope, w, dw, s = parts(g, act)
    rel = (4 + 4 * w.abs()) * unit
    # a's own error, and g's through the largest slope (1.13 for both activations)
    ea = rel * a.abs() + 1.13 * eg
    h = a * u
    eh = ea * (u.abs() + eu) + a.abs() * eu
    eh = eh + half * (h.abs() + eh) + 2.0 ** -24 * h.abs() + 3 * TINY
    y = h @ W2.t()
    ey = eh @ W2.abs().t() + _sum_error(I) * ((h.abs() + eh) @ W2.abs().t()) + I * TINY
    out = {"y": (y, ey + half * (y.abs() + ey))}
    if dy is None:
        return out
    DY = dy.detach().double().reshape(-1, H)
    T = X.shape[0]
    dh = DY @ W2
    edh = _sum_error(H) * (DY.abs() @ W2.abs())
    # the second derivative of both activations is at most 1.1
    eslope = 4 * rel * (s + a.abs() * dw) + 1.1 * eg + 4 * 2.0 ** -24 * (s + a.abs() * dw)
    dg, du = dh * u * slope, dh * a
    edg = edh * (u.abs() + eu) * (slope.abs() + eslope) + dh.abs() * (eu * (slope.abs() + eslope) + u.abs() * eslope)
    edu = edh * (a.abs() + ea) + dh.abs() * ea
    edg, edu = (e + (half + 2.0 ** -23) * (v.abs() + e) for e, v in ((edg, dg), (edu, du)))
    d, ed = torch.cat((dg, du), -1), torch.cat((edg, edu), -1)
    dx = d @ W13
    edx = ed @ W13.abs() + _sum_error(2 * I) * ((d.abs() + ed) @ W13.abs())
    dw13 = d.t() @ X
    edw13 = ed.t() @ X.abs() + _sum_error(T) * ((d.abs() + ed).t() @ X.abs())
    dw2 = DY.t() @ h
    edw2 = DY.abs().t() @ eh + _sum_error(T) * (DY.abs().t() @ (h.abs() + eh))
    for name, v, e in (("dx", dx, edx), ("dw13", dw13, edw13), ("dw2", dw2, edw2)):
        out[name] = (v, e + half * (v.abs() + e))
    return out


def check(got, value, bound, what):
    got = got.detach().double().reshape(value.shape)
    assert torch.isfinite(got).all(), what + ": not finite"
    over = (got - value).abs() - bound * (1 + 1e-9) - 1e-300
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0, "%s: %d of %d values beyond their bound, by up to %.3g (bound there %.3g)" % (
        what, int((over > 0).sum()), over.numel(), worst, float(bound.reshape(-1)[int(over.argmax())]))


# ------------------------------------------------------------------ MXFP4
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def mx_values(codes, scales):
    """float64 values [..., K] of codes [..., K/2] and scales [..., K/32]."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64, device=codes.device)
    at = torch.stack((codes.long() % 16, codes.long() // 16), -1).flatten(-2)
    s = torch.where(scales == 255, float("nan"), torch.exp2(scales.double() - 127)).repeat_interleave(32, -1)
    return grid[at] * s


def mx_encode(x):
    """(codes, scales) of x [..., K] by the definition, in float64 and integers."""
    v = x.detach().double().reshape(*x.shape[:-1], -1, 32)
    most = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    e = torch.frexp(torch.where(bad | (most == 0), 1.0, most)).exponent.long() - 3
    e = torch.where(most == 0, -127, e).clamp(min=-127)
    m = torch.where(bad[..., None], 0.0, v.abs()) * torch.exp2(-e.double())[..., None]
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    code = torch.bucketize(m, mid)  # a tie stays below its midpoint: code k - 1 ...
    tie = (m[..., None] == mid).any(-1)
    code = code + (tie & (code % 2 == 1)).long()  # ... unless that code is odd
    code = code + 8 * torch.signbit(v).long()
    code = code.reshape(x.shape)
    codes = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)
    scales = torch.where(bad, 255, e + 127).to(torch.uint8)
    return codes, scales
