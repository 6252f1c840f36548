"""Single float32 products through the dense block's tiles: inputs whose sums have one term each, so that what a product
leaves out of itself cannot hide among a sum's roundings.

A tile multiplies float32 values as three bfloat16 parts, x = hi + mid + lo, each the rest rounded to nearest, and adds up
six of the nine products of parts, the small ones first. With |x| = 1 .. 2 the rest behind hi is at most 2^-8 and the one
behind mid at most 2^-17, so what is left out (mid lo + lo mid + lo lo) is below 2^-24 of the product. A matrix instruction adds its
products to an accumulator below them with an error of up to one step of the result's last place, which is 2^-23 of it at
most (measured: 0.98 to 1.00 steps where the accumulator is 2^-6 to 2^-15 of the product, 0.5 where it is the larger one). That
is the last addition; the two before it make sums below 2^-6.9 of the product, the three before them below 2^-14, so these
add at most (2 * 2^-6.9 + 3 * 2^-14) 2^-23 < 2^-28. So a product is off by at most DELTA = 2^-23 + 2^-24 + 2^-28 of itself."""
import pytest
import torch

DELTA = 2.0 ** -23 + 2.0 ** -24 + 2.0 ** -28


def parts(x, cut):
    """hi, mid, lo of float32 x as float64: rounded to nearest bfloat16, or cut off."""
    out, rest = [], x.clone()
    for _ in range(3):
        p = (rest.view(torch.int32) & -65536).view(torch.float32) if cut else rest.to(torch.bfloat16).float()
        out.append(p.double())
        rest = rest - p
    assert not rest.any()
    return out


def left_out(a, b, cut):
    """What the six products of parts miss of a b, relative to it."""
    (ah, am, al), (bh, bm, bl) = parts(a, cut), parts(b, cut)
    whole = a.double() * b.double()
    six = ah * bh + ah * bm + am * bh + am * bm + ah * bl + al * bh
    return ((whole - six) / whole).abs()


def awkward(n, seed):
    """Values of every mantissa, and those whose parts leave out most."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.rand(n, generator=gen) + 1
    worst = torch.tensor([1 + 2.0 ** -7 - 2.0 ** -23, 1.0038986, 1 + 2.0 ** -8 - 2.0 ** -16, 1 + 2.0 ** -8 - 2.0 ** -17, 2 - 2.0 ** -23,
                          1 + 2.0 ** -8 + 2.0 ** -17 + 2.0 ** -23, 1 + 127 * 2.0 ** -15 + 2.0 ** -16 - 2.0 ** -23])
    x[::3] = worst[torch.arange(0, n, 3) // 3 % len(worst)]
    return x * torch.exp2(torch.randint(-3, 4, (n,), generator=gen).float()) * (1 - 2 * torch.randint(0, 2, (n,), generator=gen).float())


def test_parts_rounded_to_nearest_leave_out_less_than_a_rounding():
    a, b = awkward(1 << 20, 0), awkward(1 << 20, 1)
    for x, y in ((a, b), (a, a), (b, b)):
        assert float(left_out(x, y, False).max()) < 2.0 ** -24
    # parts that are cut off leave out eight times as much, and always of the product's sign
    assert float(left_out(a, a, True).max()) > 2.0 ** -21.2


def single_products(T, H, I):
    """x: 64 in its first column and one value more a row, in a column of its own. Every gate is 64, where silu is its argument
    and its slope 1; an up projection is one product, an output and a gradient's element one more."""
    assert T <= H - 1
    x = torch.zeros(T, H)
    rows = torch.arange(T)
    x[:, 0] = 64
    x[rows, 1 + rows] = awkward(T, 2)
    w13 = torch.zeros(2 * I, H)
    w13[:I, 0] = 1
    w13[I:, 1:] = awkward(I * (H - 1), 3).reshape(I, H - 1)
    w2 = torch.zeros(H, I)
    w2[torch.arange(H), torch.arange(H) % I] = awkward(H, 4)
    dy = torch.zeros(T, H)
    dy[rows, rows] = awkward(T, 5)
    return x, w13, w2, dy


def close(got, want, times, what):
    want = want.to(got.device)
    got = got.detach()
    off = (got.double() - want).abs() - times * DELTA * want.abs()
    assert float(off.max()) <= 0, "%s: off by %.3g of %.3g" % (what, float(((got.double() - want) / want).abs().nan_to_num(0).max()), times * DELTA)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,I", [(33, 40, 16), (65, 136, 72), (130, 264, 328), (200, 1304, 736), (1001, 2048, 768), (700, 1400, 4096)])
def test_one_product_a_sum(T, H, I):
    from flash_distributed_moe_amd import flashFfnOp as ops

    x, w13, w2, dy = single_products(T, H, I)
    leaves = [t.cuda().requires_grad_() for t in (x, w13, w2)]
    y = ops.gated_ffn(*leaves)
    dx, dw13, dw2 = torch.autograd.grad(y, leaves, dy.cuda())
    x, w13, w2, dy = (t.double() for t in (x, w13, w2, dy))
    u = x[:, 1:] @ w13[I:, 1:].t()
    h, dh = 64 * u, dy @ w2
    close(y, h @ w2.t(), 2, "y")                                 # h and its product
    close(dw2, dy.t() @ h, 2, "dw2")
    close(dx[:, 1:], (64 * dh) @ w13[I:, 1:], 2, "dx")           # dh and its product
    close(dx[:, 0], (dh * u).sum(1), 3, "dx of the gate")        # dh, u and their product's rounding (the sum has one term)
    close(dw13[I:, 1:], (64 * dh).t() @ x[:, 1:], 2, "dw13, up")
    close(dw13[:I, 1:], (dh * u).t() @ x[:, 1:], 4, "dw13, gate")
    # with weights of 1 behind it the up projection comes out as it is: one product alone
    one = torch.zeros(H, I)
    one[torch.arange(H), torch.arange(H) % I] = 1
    close(ops.gated_ffn(leaves[0].detach(), leaves[1].detach(), one.cuda()), h @ one.double().t(), 1, "one product")
