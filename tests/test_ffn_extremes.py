"""Gates so large that their squares are beyond float32: the activation's slope is 1 or 0 there, and so the gradients are numbers."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [8, 64])  # as few rows, and as tiles
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 63, 2.0 ** 70, 2.0 ** 110])
def test_gradients_of_saturated_gates(T, act, dtype, size):
    from flash_distributed_moe_amd import flashFfnOp as ops

    H = I = 64
    x = torch.eye(T, H, dtype=dtype, device="cuda")
    gates = torch.full((I, H), size, device="cuda")
    gates[I // 2:] = -size
    w13 = torch.cat((gates, torch.ones(I, H, device="cuda"))).to(dtype)  # gate(t, i) = +-size, up = 1
    w2, dy = torch.eye(H, I, dtype=dtype, device="cuda"), torch.ones(T, H, dtype=dtype, device="cuda")
    leaves = [t.requires_grad_() for t in (x, w13, w2)]
    y = ops.gated_ffn(*leaves, activation=act)
    dx, dw13, dw2 = torch.autograd.grad(y, leaves, dy)
    # the projections' gradients are dh * up * slope = slope and dh * act = act, and every value here is a power of two or zero
    assert torch.equal(y[:, :I // 2], torch.full_like(y[:, :I // 2], size)) and not y[:, I // 2:].any()
    slope = (torch.arange(I, device="cuda") < I // 2).to(dtype)[:, None]
    seen = (torch.arange(H, device="cuda") < T).to(dtype)[None]  # tokens are unit vectors
    assert torch.equal(dw13[:I], slope * seen) and torch.equal(dw13[I:], slope * size * seen)
    assert torch.equal(dw2, slope.t() * size * torch.full((H, 1), float(T), device="cuda", dtype=dtype))
    # dx: 32 gates' slope times the gate weight and act times 1
    assert torch.equal(dx, torch.full_like(dx, 64 * size))
