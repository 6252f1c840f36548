"""float32 operands that bfloat16 parts do not hold, in every product of the dense block: very small ones beside very
large ones, infinities and NaN. The sums are float32's all the same: single products to their roundings, and infinities and
NaN where the definition has them."""
import pytest
import torch

from tests import ffn_case
from tests.test_ffn_products import DELTA, single_products

pytestmark = pytest.mark.gpu

SHAPES = [(33, 40, 16), (65, 136, 72), (130, 264, 328), (700, 1400, 4096)]


def close(got, want, times, what, other=0.0):
    """A product that is taken again is rounded once; `times` products in a row stay within DELTA each, and beyond float32's
    normal numbers within 2^-149 of each value. A sum is not taken again if it comes out as zero, which a single product
    does if an operand is below 2^-134 and has no parts: it is then below 2^-134 times the other one, of up to `other`."""
    got, want = got.detach().double(), want.to(got.device)
    off = (got - want).abs() - times * (DELTA * want.abs() + 2.0 ** -149)
    off = torch.where((got == 0) & (want.abs() < 2.0 ** -134 * other), -1.0, off)
    assert torch.isfinite(got).all() and float(off.max()) <= 0, what


# powers of two for the tokens' values, the up weights, the down weights and the output's gradient; products stay within
# float32's range, and the tokens' constant column and the gates are 64 as ever
@pytest.mark.parametrize("scales", [(-118, 60, 0, 0), (60, -118, 0, 0), (-126, 90, 0, 0), (-140, 100, 0, 0), (-100, 30, 0, 0),
                                    (-60, -20, 0, 0), (0, 0, 60, -118), (0, 0, -118, 60), (-10, -5, 100, -110), (0, -8, -115, 100),
                                    (45, 40, -40, -50)])
@pytest.mark.parametrize("T,H,I", SHAPES)
def test_products_of_operands_far_apart(T, H, I, scales):
    from flash_distributed_moe_amd import flashFfnOp as ops

    sx, sw, sv, sd = (2.0 ** s for s in scales)
    x, w13, w2, dy = single_products(T, H, I)
    x[:, 1:] = (x[:, 1:].double() * sx).float()
    w13[I:] = (w13[I:].double() * sw).float()
    w2, dy = (w2.double() * sv).float(), (dy.double() * sd).float()
    leaves = [t.cuda().requires_grad_() for t in (x, w13, w2)]
    y = ops.gated_ffn(*leaves)
    dx, dw13, dw2 = torch.autograd.grad(y, leaves, dy.cuda())
    x, w13, w2, dy = (t.double() for t in (x, w13, w2, dy))
    u = x[:, 1:] @ w13[I:, 1:].t()
    h, dh = 64 * u, dy @ w2
    close(y, h @ w2.t(), 2, "y")
    close(dw2, dy.t() @ h, 2, "dw2")
    close(dx[:, 1:], (64 * dh) @ w13[I:, 1:], 2, "dx")
    close(dw13[I:, 1:], (64 * dh).t() @ x[:, 1:], 2, "dw13, up", other=min(2.0 ** 32, float((64 * dh).abs().max())))


def make(T, H, I, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(4000 + seed)

    def normal(s, *shape):
        return torch.empty(shape, device="cuda").normal_(0.0, s, generator=gen)

    return normal(1.0, T, H), normal(H ** -0.5, 2 * I, H), normal(I ** -0.5, H, I), normal(1.0, T, H)


def run(x, w13, w2, dy):
    from flash_distributed_moe_amd import flashFfnOp as ops

    leaves = [t.detach().requires_grad_() for t in (x, w13, w2)]
    y = ops.gated_ffn(*leaves)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy))


@pytest.mark.parametrize("T,H,I", [(40, 64, 48), (300, 264, 136), (67, 384, 7680), (1001, 512, 768)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_backward_of_one_token_that_holds_no_number(T, H, I, value):
    """Its own rows and the weights' gradients hold none, other tokens' rows keep every bit."""
    x, w13, w2, dy = make(T, H, I)
    clean = run(x, w13, w2, dy)
    rest = [t for t in range(T) if t != T // 2]
    x[T // 2, 7] = value
    y, dx, dw13, dw2 = run(x, w13, w2, dy)
    assert torch.equal(y[rest], clean[0][rest]) and torch.equal(dx[rest], clean[1][rest])
    assert not torch.isfinite(y[T // 2]).any() and not torch.isfinite(dx[T // 2]).any()
    # a gate of minus infinity gives no number either; whatever h is, its gradient sums over that token
    assert not torch.isfinite(dw2).any() and not torch.isfinite(dw13).any()
    # a bad gradient of one output: its token's rows, that output's weights and all projections' gradients
    x, w13, w2, dy = make(T, H, I)
    dy[T // 2, 5] = value
    y, dx, dw13, dw2 = run(x, w13, w2, dy)
    assert torch.equal(y, clean[0]) and torch.equal(dx[rest], clean[1][rest])
    assert not torch.isfinite(dx[T // 2]).any() and not torch.isfinite(dw2[5]).any()
    others = [h for h in range(H) if h != 5]
    assert torch.equal(dw2[others], clean[3][others])


@pytest.mark.parametrize("T,H,I", [(40, 64, 48), (300, 264, 136), (67, 384, 7680)])
def test_infinities_of_one_sign_stay_infinities(T, H, I):
    x, w13, w2, dy = (t.abs() for t in make(T, H, I, seed=1))
    x[3, 5] = float("inf")
    y, _, _, dw2 = run(x, w13, w2, dy)
    assert torch.isposinf(y[3]).all() and torch.isfinite(y[:3]).all() and torch.isfinite(y[4:]).all()
    assert torch.isposinf(dw2).all()


@pytest.mark.parametrize("scale", [-60, -100, -120])
def test_gradients_of_tiny_outputs(scale):
    """A gradient so small that every sum behind it is: to the last step of a value that has all its bits."""
    T, H, I = 300, 264, 136
    x, w13, w2, dy = make(T, H, I, seed=2)
    plain = run(x, w13, w2, dy)
    tiny = run(x, w13, w2, dy * 2.0 ** scale)
    want = ffn_case.block(x, w13, w2, "silu", dy * 2.0 ** scale)
    for name, p, t in zip(("dx", "dw13", "dw2"), plain[1:], tiny[1:]):
        value, bound = want[name]
        ffn_case.check(t, value, bound + 1e4 * 2.0 ** -149, name)
        assert p.abs().max() > 0


def test_rows_and_columns_of_zeros():
    T, H, I = 200, 264, 136
    x, w13, w2, dy = make(T, H, I, seed=3)
    x[::3] = 0
    dy[1::4] = 0
    w13[5] = 0
    w2[:, 7] = 0
    want = ffn_case.block(x, w13, w2, "silu", dy)
    for name, got in zip(("y", "dx", "dw13", "dw2"), run(x, w13, w2, dy)):
        ffn_case.check(got, *want[name], name)
        assert torch.equal(got == 0, want[name][0].reshape(got.shape) == 0)
