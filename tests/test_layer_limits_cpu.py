"""What the operators around a layer's blocks refuse of torch's other kinds of tensors, before anything is enqueued, so without a GPU: those
that stand for others and have no memory (their null addresses would stand for arguments that are left out, and those of views of
them for memory that is not there), results that carry a tangent, and scales that are learnt."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses import FakeTensorMode

from flash_distributed_moe_amd import flashFfnOp as fops, flashLayerOp as ops

B = torch.bfloat16


def fake(*shape, dtype=torch.float32, view=False):
    with FakeTensorMode():
        t = torch.ones((2, *shape), dtype=dtype, device="cuda")
        return t[1] if view else t[0]


@pytest.mark.parametrize("view", [False, True])
@pytest.mark.parametrize("call", [
    lambda f: ops.route(f(6, 16), 2), lambda f: ops.route(f(6, 16), 2, mask=f(6, dtype=torch.bool)),
    lambda f: ops.block_norm(f(6, 64), f(64)), lambda f: ops.block_join(f(6, 64), f(6, 64), f(64), f(64), f(64)),
    lambda f: fops.add_adapters(f(6, 64, dtype=B), f(6, 64, dtype=B), fops.Adapters(f(1, 8, 64, dtype=B), f(1, 64, 8, dtype=B), f(1)),
                                f(6, dtype=torch.int32)),
    lambda f: fops.quantize_mxfp4(f(6, 64)), lambda f: fops.gated_ffn(f(6, 64), f(128, 64), f(64, 64)),
    lambda f: fops.dequantize_mxfp4(fops.Mxfp4(f(6, 32, dtype=torch.uint8), f(6, 2, dtype=torch.uint8))),
    lambda f: fops.mxfp4_linear(f(6, 64, dtype=B), fops.Mxfp4(f(64, 32, dtype=torch.uint8), f(64, 2, dtype=torch.uint8))),
])
def test_tensors_without_memory_are_refused(call, view):
    with pytest.raises(RuntimeError, match="no memory of its own"):
        call(lambda *shape, dtype=torch.float32: fake(*shape, dtype=dtype, view=view))


def test_results_with_a_tangent_are_refused():
    """What is written into them would leave their tangent as it was."""
    with fwd.dual_level():
        out = fwd.make_dual(torch.zeros(3, 24, dtype=B), torch.ones(3, 24, dtype=B))
        a = fops.Adapters(torch.zeros(2, 8, 16, dtype=B), torch.zeros(2, 24, 8, dtype=B), torch.zeros(2))
        with pytest.raises(RuntimeError, match="forward-mode"):
            fops.add_adapters(torch.zeros(3, 24, dtype=B), torch.zeros(3, 16, dtype=B), a, torch.zeros(3, dtype=torch.int32), out=out)


@pytest.mark.parametrize("name", ["residual_scale", "branch_scale", "eps"])
def test_scales_that_are_learnt_are_refused(name):
    """They would be read as numbers, without a gradient."""
    x, v = torch.zeros(3, 8), torch.tensor(1.0, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.block_join(x, x, **{name: v})
    if name == "eps":
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.block_norm(x, torch.ones(8), eps=v)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.block_join(x, x, **{name: v})
