"""FlashGatedFfn over the blocks that models have: what it takes from one, what it refuses, and training through it."""
import pytest
import torch

from flash_distributed_moe_amd import flashFfnOp as ops
from tests import ffn_case


class Block(torch.nn.Module):
    def __init__(self, hidden=64, intermediate=32, bias=(False, False), act_fn=None, dtype=torch.float32, device=None):
        super().__init__()
        self.gate_up_proj = torch.nn.Linear(hidden, 2 * intermediate, bias=bias[0], dtype=dtype, device=device)
        self.down_proj = torch.nn.Linear(intermediate, hidden, bias=bias[1], dtype=dtype, device=device)
        if act_fn is not None:
            self.act_fn = act_fn


class SiluAndMul(torch.nn.Module):
    def forward(self, x):
        g, u = x.chunk(2, -1)
        return torch.nn.functional.silu(g) * u


@pytest.mark.parametrize("bias", [(True, False), (False, True)])
def test_biases_are_refused(bias):
    with pytest.raises(RuntimeError, match="has a bias"):
        ops.FlashGatedFfn(Block(bias=bias))


@pytest.mark.parametrize("act_fn,name", [(None, "silu"), (torch.nn.SiLU(), "silu"), (torch.nn.functional.silu, "silu"), (SiluAndMul(), "silu"),
                                         (torch.nn.GELU(approximate="tanh"), "gelu_tanh")])
def test_the_block_says_which_activation(act_fn, name):
    assert ops.FlashGatedFfn(Block(act_fn=act_fn)).activation == name
    assert ops.FlashGatedFfn(Block(act_fn=act_fn), activation="gelu_tanh").activation == "gelu_tanh"


@pytest.mark.parametrize("act_fn", [torch.nn.GELU(), torch.nn.ReLU(), torch.sum, "silu", lambda x: 1 / 0])
def test_another_activation_is_refused(act_fn):
    block = Block()
    block.act_fn = act_fn
    with pytest.raises(RuntimeError, match="pass activation"):
        ops.FlashGatedFfn(block)
    assert ops.FlashGatedFfn(block, activation="silu").activation == "silu"


def test_the_parameters_stay_the_block_s():
    block = Block()
    module = ops.FlashGatedFfn(block)
    assert module.w13 is block.gate_up_proj.weight and module.w2 is block.down_proj.weight
    assert len(list(module.parameters())) == 2 and not list(module.buffers())


@pytest.mark.gpu
@pytest.mark.parametrize("act_fn,name", [(torch.nn.SiLU(), "silu"), (torch.nn.GELU(approximate="tanh"), "gelu_tanh")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_through_the_module(dtype, act_fn, name):
    """Gradients reach the block's parameters and add up over two batches, and an optimiser's step moves both the
    block's weights and the module's answers."""
    torch.manual_seed(5)
    block = Block(136, 72, act_fn=act_fn, dtype=dtype, device="cuda")
    module = ops.FlashGatedFfn(block)
    total = {}
    for T in (40, 7):
        x, dy = torch.randn(T, 136, device="cuda", dtype=dtype), torch.randn(T, 136, device="cuda", dtype=dtype)
        w13, w2 = block.gate_up_proj.weight, block.down_proj.weight
        module(x).backward(dy)
        want = ffn_case.block(x, w13, w2, name, dy)
        for k in ("dw13", "dw2"):
            value, bound = want[k]
            if k in total:  # added in the gradients' type, rounded once more
                value, bound = value + total[k][0], bound + total[k][1]
                bound = bound + ffn_case.HALF[dtype] * (value.abs() + bound)
            total[k] = value, bound
    for k, p in (("dw13", block.gate_up_proj.weight), ("dw2", block.down_proj.weight)):
        ffn_case.check(p.grad, *total[k], k)
    x = torch.randn(5, 136, device="cuda", dtype=dtype)
    before = module(x).detach()
    torch.optim.SGD(module.parameters(), lr=0.5).step()
    after = module(x).detach()
    assert not torch.equal(before, after)
    ffn_case.check(after, *ffn_case.block(x, block.gate_up_proj.weight, block.down_proj.weight, name)["y"], "after a step")
