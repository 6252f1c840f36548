"""float32 products whose sums bfloat16 parts do not give: infinities, NaN, and sums of very small values, in every product of
the dense block, forward and backward."""
import pytest
import torch

from tests import ffn_case

pytestmark = pytest.mark.gpu


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
