"""The dense block and MXFP4 products on whole numbers, where float32 sums are exact in any order: a k that a tile, a group
of waves or a split leaves out or takes twice is a difference in the results' bits. And float32 on ordinary values, held
to the error that a plain float32 evaluation has itself."""
import pytest
import torch

from tests.test_ffn_products import parts

WHOLE = 2.0 ** 24  # float32 holds every whole number up to here
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
# few rows; each size of tile, groups of waves and splits; sums that end inside a step (see the other tests' shapes)
SHAPES = [(1, 136, 72), (9, 520, 264), (31, 2048, 768), (33, 520, 264), (65, 1344, 736), (130, 264, 136), (257, 136, 328), (300, 512, 1024),
          (67, 384, 7680), (50, 4360, 72), (2100, 200, 3000), (3841, 72, 3600), (77, 3600, 3904), (3841, 3600, 40), (1100, 1304, 2600),
          (8200, 72, 40), (1001, 2048, 768)]


def signs(gen, share, *shape):
    """-1, 0 and 1; `share` of them not zero."""
    v = torch.rand(shape, generator=gen)
    return (v < share / 2).double() - (v > 1 - share / 2).double()


def exactly(a, b):
    """a @ b, both whole; the sums' magnitudes have to be what float32 holds."""
    assert float((a.abs() @ b.abs()).max()) < WHOLE
    return a @ b


def whole_block(T, H, I, seed=0):
    """x, w13, w2, dy of whole numbers. Every gate lies around 512, far above where SiLU is its argument and its slope 1."""
    gen = torch.Generator().manual_seed(seed)
    x = signs(gen, 0.25, T, H)
    x[:, 0] = 512
    w13 = signs(gen, min(1.0, 400.0 / H), 2 * I, H)
    w13[:I, 0], w13[I:, 0] = 1, 0
    w2 = signs(gen, min(0.5, 150.0 / I), H, I)
    dy = signs(gen, min(0.5, 3.0 / H), T, H)
    return x, w13, w2, dy


def definition(x, w13, w2, dy, dtype):
    """y, dx, dw13, dw2, with the roundings that the kernels have: h and the projections' gradients to `dtype`."""
    I = w2.shape[1]
    g, u = exactly(x, w13[:I].t()), exactly(x, w13[I:].t())
    assert float(g.min()) > 20
    h = (g * u).to(dtype).double()
    dh = exactly(dy, w2)
    d = torch.cat((dh * u, dh * g), 1).to(dtype).double()
    return dict(y=exactly(h, w2.t()), dx=exactly(d, w13), dw13=exactly(d.t(), x[:, 1:]), dw2=exactly(dy.t(), h))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("T,H,I", SHAPES)
def test_block_on_whole_numbers(T, H, I, dtype):
    from flash_distributed_moe_amd import flashFfnOp as ops

    dt = DTYPES[dtype]
    data = [t.cuda() for t in whole_block(T, H, I, seed=T)]
    want = definition(*data, dt)
    leaves = [t.to(dt).requires_grad_() for t in data[:3]]
    assert all(torch.equal(a.detach().double(), b) for a, b in zip(leaves, data))
    y = ops.gated_ffn(*leaves)
    dx, dw13, dw2 = torch.autograd.grad(y, leaves, data[3].to(dt))
    # (the first column of dw13 sums over the tokens' 512: not exact)
    for name, got in (("y", y.detach()), ("dx", dx), ("dw13", dw13[:, 1:]), ("dw2", dw2)):
        different = int((got != want[name].to(dt)).sum())
        assert different == 0, "%s: %d of %d values" % (name, different, got.numel())


@pytest.mark.gpu
@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 136, 96), (5, 520, 4096), (31, 264, 16384), (5, 264, 17408), (33, 1000, 384), (64, 128, 512), (65, 384, 288),
                                   (130, 257, 320), (257, 520, 544), (300, 1000, 1056), (3841, 3600, 160), (1024, 8200, 256), (256, 8200, 512),
                                   (520, 8192, 2080), (40, 37, 5120), (93, 200, 7520), (703, 72, 4096)])
def test_products_on_whole_numbers(M, N, K, both):
    """Halves, in fact: weights of the grid's smaller values under scales of 1/2, 1 and 2."""
    from flash_distributed_moe_amd import flashFfnOp as ops
    from tests.ffn_case import mx_values

    gen = torch.Generator().manual_seed(M)

    def packed(rows):
        return ops.Mxfp4(torch.randint(0, 256, (rows, K // 2), dtype=torch.uint8, generator=gen).cuda(),
                         torch.randint(126, 129, (rows, K // 32), dtype=torch.uint8, generator=gen).cuda())

    w = packed(N)
    x = packed(M) if both else signs(gen, 0.5, M, K).cuda().to(torch.bfloat16)
    value = mx_values(*x) if both else x.double()
    want = exactly(16 * value, mx_values(*w).t()) / 16  # quarters times quarters
    got = ops.mxfp4_linear(x, w)
    different = int((got != want.to(torch.bfloat16)).sum())
    assert different == 0, "%d of %d values" % (different, got.numel())


# ------------------------------------------------------------------ float32 on ordinary values
def plain(x, w13, w2, dy, dtype):
    """The block and its gradients by elementary operations in `dtype`."""
    x, w13, w2, dy = (t.to(dtype) for t in (x, w13, w2, dy))
    g, u = (x @ w13.t()).chunk(2, -1)
    s = torch.sigmoid(g)
    a, slope = g * s, s + g * s * (1 - s)
    h, dh = a * u, dy @ w2
    d = torch.cat((dh * u * slope, dh * a), 1)
    return dict(y=h @ w2.t(), dx=d @ w13, dw13=d.t() @ x, dw2=dy.t() @ h)


def rms(t):
    return float(t.double().square().mean().sqrt())


def normal(T, H, I, seed=0, device="cpu"):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * f).to(device) for s, f in
            (((T, H), 1.0), ((2 * I, H), H ** -0.5), ((H, I), I ** -0.5), ((T, H), 1.0))]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,I", [s for s in SHAPES if s[0] * s[1] * s[2] < 2 ** 32])
def test_float32_is_as_near_as_float32_is(T, H, I):
    """A tile rounds its sums six times in 32 k, a float32 evaluation once in each k, or once in four on the matrix
    instructions: the errors' root mean square, over all elements, is at most twice as large."""
    from flash_distributed_moe_amd import flashFfnOp as ops

    data = normal(T, H, I, seed=T, device="cuda")
    want, other = plain(*data, torch.float64), plain(*data, torch.float32)
    leaves = [t.clone().requires_grad_() for t in data[:3]]
    y = ops.gated_ffn(*leaves)
    got = dict(zip(("y", "dx", "dw13", "dw2"), (y.detach(), *torch.autograd.grad(y, leaves, data[3]))))
    for name in want:
        mine, theirs = rms(got[name] - want[name]), rms(other[name] - want[name])
        assert mine <= 2 * theirs, "%s: %.3g against %.3g" % (name, mine, theirs)


def test_what_these_checks_see():
    """One of a product's six parts left out, and one step of a long sum: planted in the definitions, on the CPU."""
    gen = torch.Generator().manual_seed(1)
    a, b = torch.randn(64, 2048, generator=gen), torch.randn(64, 2048, generator=gen)
    want = a.double() @ b.double().t()
    own = rms((a @ b.t()).double() - want)
    # a float32 sum of 2048 products one after another, the most that any evaluation rounds
    total = torch.zeros(64, 64)
    for k in range(2048):
        total += a[:, k, None] * b[None, :, k]
    worst = max(own, rms(total.double() - want))
    pa, pb = parts(a, False), parts(b, False)
    six = [(0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)]
    whole = sum(pa[i] @ pb[j].t() for i, j in six)
    assert rms(whole - want) < 0.5 * own
    for left_out in six:
        i, j = left_out
        assert rms(whole - pa[i] @ pb[j].t() - want) > 2 * worst, left_out
    # whole numbers: each step of 32 k changes results in either type
    data = whole_block(40, 520, 264)
    for dtype in DTYPES.values():
        right = definition(*data, dtype)
        for step in range(1, 520 // 32):
            x = data[0].clone()
            x[:, 32 * step:32 * step + 32] = 0
            assert not torch.equal(definition(x, *data[1:], dtype)["y"].to(dtype), right["y"].to(dtype))
        for step in range(264 // 32):
            w2 = data[2].clone()
            w2[:, 32 * step:32 * step + 32] = 0
            assert not torch.equal(definition(*data[:2], w2, data[3], dtype)["y"].to(dtype), right["y"].to(dtype))
