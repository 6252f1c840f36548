"""Float64 restatements of what stands around a layer's blocks, with bounds on what the kernels may be off.

A bound counts what is rounded on the way to a value, element by element: a float32 operation is off by 2^-24 of its result, a
stored value by half a step of its type (`HALF`), a sum of n float32 terms by n 2^-24 of the sum of their magnitudes. Below
2^-126 float32 results of the exponential are zeros (`TINY`).
"""
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TINY = 2.0 ** -126
U = 2.0 ** -24


def check(got, value, bound, what):
    got = got.detach().double().reshape(value.shape)
    assert torch.isfinite(got).all(), what + ": not finite"
    over = (got - value).abs() - bound * (1 + 1e-9)
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0, "%s: %d of %d values beyond their bound, by up to %.3g (bound there %.3g)" % (
        what, int((over > 0).sum()), over.numel(), worst, float(bound.expand(value.shape).reshape(-1)[int(over.argmax())]))


# ------------------------------------------------------------------ the router's choice
def ranks(logits, able):
    """Of each logit how many candidates are ahead of it: greater, or equal at a lower place. E where it is none."""
    T, E = logits.shape
    v = logits.double().masked_fill(~able, float("-inf"))
    lower = torch.ones(E, E, device=logits.device).triu(1).bool()  # [i, j]: i < j
    out = torch.empty(T, E, dtype=torch.int64, device=logits.device)
    for lo in range(0, T, 1024):
        a, b = v[lo:lo + 1024, :, None], v[lo:lo + 1024, None, :]
        out[lo:lo + 1024] = (((a > b) | ((a == b) & lower)) & able[lo:lo + 1024, :, None]).sum(1)
    return out.masked_fill(~able, E)


def route(logits, k, renormalize, mask=None, dw=None, db=None, dz=None):
    """{name: (value, bound)}; experts and counts without a bound. logits [T, E]; d*: the outputs' gradients, or None."""
    raw = logits.detach()
    T, E = raw.shape
    able = raw > torch.finfo(raw.dtype).min
    if mask is not None:
        able = able & mask[:, None]
    L = raw.double().masked_fill(~able, 0.0).requires_grad_()
    some = able.any(1)
    m = L.detach().masked_fill(~able, float("-inf")).amax(1, keepdim=True).masked_fill(~some[:, None], 0.0)
    e = torch.exp(L - m) * able
    s = e.sum(1, keepdim=True).masked_fill(~some[:, None], 1.0)
    p = e / s
    lse = (m + torch.log(s)) * some[:, None]
    rank = ranks(raw, able)
    win = rank < k
    experts = torch.full((T, k), -1, dtype=torch.int64, device=raw.device)
    t, c = win.nonzero(as_tuple=True)
    experts[t, rank[t, c]] = c
    filled, at = experts >= 0, experts.clamp(min=0)
    of = (e * win).sum(1, keepdim=True).masked_fill(~some[:, None], 1.0) if renormalize else s
    w = torch.gather(e, 1, at) * filled / of
    counts = win.sum(0)
    n, slots = max(1, int(some.sum())), max(1, int(counts.sum()))
    balance = E * (counts.double() / slots * p.sum(0) / n).sum()
    zed = (lse ** 2).sum() / n
    # a probability: the difference (|x| 2^-24 of the power), the exponential (8), the sum of up to 256 as 16 + 4 steps of terms
    # that are off by as much (whose |x| is 6 on average at most), a division and a product
    x = (L.detach() - m).abs()
    rel = (x + 50) * U
    P, Z = p.detach(), lse.detach()
    elsewhere = (Z.abs() + m.abs() + 60) * U  # of a logarithm of a sum
    out = {"experts": experts, "counts": counts,
           "weights": (w.detach(), torch.gather(rel, 1, at) * w.detach() + TINY),
           # all terms are positive; sums over tokens in at most T / 4096 + 30 steps
           "balance_loss": (balance.detach(), balance.detach() * (T / 4096 + 90) * U + TINY),
           "z_loss": (zed.detach(), (2 * Z.abs() * elsewhere).sum() / n + zed.detach() * (T / 4096 + 90) * U + TINY)}
    if dw is None and db is None and dz is None:
        return out
    loss = L.sum() * 0
    for d, v in ((dw, w), (db, balance), (dz, zed)):
        if d is not None:
            loss = loss + (d.double() * v).sum()
    grad, = torch.autograd.grad(loss, L)
    grad = grad * able
    W = w.detach()
    D = dw.double().abs() * filled if dw is not None else torch.zeros_like(W)
    big = torch.zeros_like(P).scatter_add_(1, at, W * (D + (W * D).sum(1, keepdim=True)) * filled)
    g = (0.0 if db is None else abs(float(db))) * E * counts.double() / (slots * n)
    pull = (0.0 if dz is None else 2 * abs(float(dz))) / n
    factor = g + (P * g).sum(1, keepdim=True) + pull * (Z.abs() + elsewhere / U)
    if not renormalize:
        factor = factor + (W * D).sum(1, keepdim=True)
    # a probability below 2^-126 is taken as zero, and what multiplies it is lost with it
    out["dlogits"] = (grad, (big + P * factor) * (rel + 60 * U) + HALF[raw.dtype] * grad.abs() + TINY * (1 + factor))
    return out
