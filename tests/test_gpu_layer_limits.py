"""Calls of the operators around a layer's blocks at the limits of what is documented: values next to the end of their type's range."""
import pytest
import torch

from flash_distributed_moe_amd import flashFfnOp as fops
from tests import layer_case

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ values next to the end of the range
# rows by themselves, tiles of 16, tiles of 64 (K=N=4096 and rank 16, as in the rule's comment)
@pytest.mark.parametrize("T", [4, 900, 2000])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_adapters_between_the_products(T, sign):
    """x A^T is finite in float32 and nearer to infinity than bfloat16's greatest: the result is a number all the same, and so
    are the other ranks' shares; an infinity stays one."""
    K, N, r = 4096, 4096, 16
    x = torch.zeros(T, K, dtype=torch.bfloat16, device="cuda")
    x[:, 0], x[:, 1] = sign * 2.0 ** 64, sign * 2.0 ** 64
    down, up = torch.zeros(1, r, K, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, N, r, dtype=torch.bfloat16, device="cuda")
    # (2 - 2^-9) 2^127, exact in float32; half way to 2^128 from bfloat16's greatest is (2 - 2^-8) 2^127
    down[0, 3, 0], down[0, 3, 1] = (2 - 2.0 ** -7) * 2.0 ** 63, 3 * 2.0 ** -9 * 2.0 ** 63
    down[0, 5, 0] = 2.0 ** 50
    up[0, :, 3], up[0, :, 5] = 2.0 ** -20, -2.0 ** -12
    y, ids = torch.ones(T, N, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    one = torch.ones(1, device="cuda")
    got = fops.add_adapters(y, x, fops.Adapters(down, up, one), ids)
    layer_case.check(got, *layer_case.adapters(y, x, down, up, one, ids), "T=%d" % T)
    x[T // 2, 2] = float("inf")
    down[0, 3, 2] = 1.0
    down[0, :3, 2], down[0, 4:, 2] = 2.0 ** -100, 2.0 ** -100
    up[0, :, :] = 2.0 ** -20
    got = fops.add_adapters(y, x, fops.Adapters(down, up, one), ids)
    rest = torch.arange(T, device="cuda") != T // 2
    assert torch.isinf(got[T // 2]).all() and torch.isfinite(got[rest]).all()
