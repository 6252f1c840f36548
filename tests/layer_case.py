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
    # a probability: of the power x 2^-24 each for the difference and for its product with log2(e), a fifth of that for the constant
    # (log2(e) is held to 1.4 * 10^-8 of itself, 0.23 * 2^-24), the exponential (8 steps), the sum of up to 256 as 16 + 4 steps of
    # terms that are off by as much (whose |x|, weighted with them, is the entropy less log s: 5.6 at most, 13 of its steps), a
    # division and a product
    x = (L.detach() - m).abs()
    rel = (2.25 * x + 50) * U
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


# ------------------------------------------------------------------ the norms around a block
def _mean(v):
    return v.mean(-1, keepdim=True)


def join(x, branch=None, post=None, gate=None, next_weight=None, alpha=1.0, beta=1.0, eps=1e-6, dy=None, dh=None):
    """{name: (value, bound)} of y, h, and with dy or dh of the gradients "x", "branch", "post", "gate", "next_weight". Without a
    branch y = x. Shapes as the operator takes them.

    One over a root mean square is off by 40 steps of float32 of itself (a lane's 32 squares, 10 steps across lanes and waves, the
    mean, eps and the root: half of those relative to it); sums over a row by 60 steps of their magnitudes, sums over tokens
    by T / 256 + 80 (a workgroup's rows, the rows it has at once, up to 512 workgroups sixteen at a time)."""
    half, H = HALF[x.dtype], x.shape[-1]
    X, B, P, G, W, DY, DH = (None if t is None else t.detach().double() for t in (x, branch, post, gate, next_weight, dy, dh))
    zero = torch.zeros_like(X)
    if B is None:
        y, ey = X, zero
    else:
        rb = 1 / (_mean(B * B) + eps).sqrt() if P is not None else torch.ones_like(_mean(B))
        u = B * rb
        eu = 42 * U * u.abs() if P is not None else zero
        w = P if P is not None else torch.ones_like(zero)
        z, ez = u * w, eu * w.abs() + U * (u * w).abs()
        g = G if G is not None else torch.ones_like(z)
        y = alpha * X + beta * g * z
        ey = 2 * U * (alpha * X).abs() + abs(beta) * g.abs() * (ez + 3 * U * z.abs()) + U * y.abs()
    out = {} if B is None else {"y": (y, ey + half * (y.abs() + ey))}
    if W is not None:
        ry = 1 / (_mean(y * y) + eps).sqrt()
        er = 40 * U + _mean(ey * ey).sqrt() * ry
        v = y * ry
        ev = ey * ry + v.abs() * (er + U)
        out["h"] = (v * W, ev * W.abs() + 2 * U * (v * W).abs() + half * ((v * W).abs() + ev * W.abs()))
    if dy is None and dh is None:
        return out
    rows = X.numel() // H
    tokens = (rows / 256 + 80) * U
    columns = lambda t: t.reshape(-1, H).sum(0)  # noqa: E731

    def stored(name, value, bound):
        out[name] = (value, bound + half * (value.abs() + bound) + TINY)

    t, et = (zero, zero) if DY is None else (DY, zero)
    if W is not None:
        if DH is None:
            stored("next_weight", torch.zeros_like(W), torch.zeros_like(W))
        else:
            stored("next_weight", columns(DH * v), columns(DH.abs() * ev) + tokens * columns((DH * v).abs()))
            q = DH * W
            c = _mean(q * v)
            ec = _mean(q.abs() * ev + 60 * U * (q * v).abs())
            t = t + ry * (q - v * c)
            et = ry * ((q.abs() + (v * c).abs()) * (er + 4 * U) + ev * c.abs() + v.abs() * ec) + 2 * U * ((0 if DY is None else DY.abs()) + t.abs())
    stored("x", (alpha if B is not None else 1.0) * t, (abs(alpha) if B is not None else 1.0) * et + U * t.abs())
    if B is None:
        return out
    d, ed = beta * t, abs(beta) * et + U * (beta * t).abs()
    if G is not None:
        value, bound = d * z, ed * z.abs() + d.abs() * ez + U * (d * z).abs()
        size, steps = value.abs(), 0.0
        shape = (1,) * (X.dim() - G.dim()) + tuple(G.shape)
        over = [i for i in range(X.dim()) if shape[i] != X.shape[i]]
        if over:
            value, bound, size = (s.sum(over, keepdim=True) for s in (value, bound, size))
            steps = 60 * U + tokens
        stored("gate", value.reshape(G.shape), (bound + (steps + 2 * U) * size).reshape(G.shape))
    q, eq = d * g * w, ed * (g * w).abs() + 3 * U * (d * g * w).abs()
    if P is not None:
        stored("post", columns(d * g * u), columns((g * u).abs() * ed + (d * g).abs() * eu + 3 * U * (d * g * u).abs()) + tokens * columns((d * g * u).abs()))
        c = _mean(q * u)
        ec = _mean(u.abs() * eq + q.abs() * eu + 64 * U * (q * u).abs())
        value = rb * (q - u * c)
        eq = rb * (eq + u.abs() * ec + c.abs() * eu + 46 * U * (q.abs() + (u * c).abs()))
        q = value
    stored("branch", q, eq)
    return out


# ------------------------------------------------------------------ adapters beside a projection
def adapters(y, x, down, up, scales, ids):
    """(value, bound) of y + s (x A^T) B^T. Sums of n products are off by 2 n steps of their magnitudes; between the two products
    the vector instructions take float32, the matrix instructions two bfloat16 parts (2^-16 is left out) in twice the products."""
    Y, X = y.double(), x.double()
    r, K = down.shape[1:]
    value, bound = Y.clone(), torch.zeros_like(Y)
    for i in ids.unique().tolist():
        if i < 0 or i >= down.shape[0]:
            continue
        rows = ids == i
        A, B, s = down[i].double(), up[i].double(), float(scales[i])
        u, size = X[rows] @ A.t() * s, X[rows].abs() @ A.abs().t() * abs(s)
        eu = (2 * K + 2) * U * size + 2.0 ** -16 * u.abs()
        value[rows] += u @ B.t()
        bound[rows] = eu @ B.abs().t() + (4 * r + 8) * U * (u.abs() + eu) @ B.abs().t()
    return value, bound + U * value.abs() + HALF[y.dtype] * (value.abs() + bound)
