"""The operators around a layer's blocks on arrays whose last values lie more than 2^31 values, or 2^32 bytes, behind the first: the last
rows against their definition, and against what a call on them alone gives."""
import pytest
import torch

from flash_distributed_moe_amd import flashFfnOp as fops, flashLayerOp as ops
from tests import layer_case

pytestmark = pytest.mark.gpu

TAIL = 200


def filled(rows, width, dtype, seed):
    """Random rows at the end, zeros in front."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.zeros(rows, width, dtype=dtype, device="cuda")
    t[-TAIL:] = torch.empty(TAIL, width, device="cuda").normal_(generator=gen).to(dtype)
    return t


def test_route():
    E, k, T = 256, 4, (1 << 31) // 256 + 1000
    logits = filled(T, E, torch.bfloat16, 1).requires_grad_()
    got = ops.route(logits, k)
    want = layer_case.route(logits[-TAIL:], k, True)
    assert torch.equal(got.experts[-TAIL:].long(), want["experts"])
    layer_case.check(got.weights[-TAIL:], *want["weights"], "weights")
    front = torch.zeros(E, dtype=torch.int64, device="cuda")
    front[:k] = T - TAIL  # zeros are equals
    assert torch.equal(got.counts.long(), want["counts"] + front)
    dw = torch.zeros_like(got.weights)
    dw[-TAIL:] = torch.randn(TAIL, k, device="cuda")
    grad, = torch.autograd.grad(got.weights, logits, dw)
    layer_case.check(grad[-TAIL:], *layer_case.route(logits[-TAIL:], k, True, dw=dw[-TAIL:])["dlogits"], "dlogits")
    assert not grad[:-TAIL].any()


def test_join():
    H, T = 4096, (1 << 31) // 4096 + 500
    x, branch, dy = (filled(T, H, torch.bfloat16, s) for s in (2, 3, 4))
    w = [torch.rand(H, device="cuda").bfloat16() + 0.5 for _ in range(2)]
    x.requires_grad_(), branch.requires_grad_()
    y, h = ops.block_join(x, branch, w[0], None, w[1], eps=1e-3)
    want = layer_case.join(x[-TAIL:], branch[-TAIL:], w[0], None, w[1], eps=1e-3, dy=dy[-TAIL:], dh=dy[-TAIL:])
    grads = torch.autograd.grad([y, h], [x, branch], [dy, dy])
    for name, t in zip(("y", "h", "x", "branch"), (y, h, *grads)):
        layer_case.check(t[-TAIL:], *want[name], name)
        assert not t[:-TAIL].any(), name


def test_adapters():
    N, K, T = 8192, 64, (1 << 31) // 8192 + 700
    x, y = filled(T, K, torch.bfloat16, 5), filled(T, N, torch.bfloat16, 6)
    a = [torch.randn(3, 16, K, device="cuda").bfloat16() * 0.1, torch.randn(3, N, 16, device="cuda").bfloat16() * 0.3, torch.rand(3, device="cuda")]
    ids = torch.randint(-1, 3, (T,), device="cuda", dtype=torch.int32)
    got = fops.add_adapters(y, x, fops.Adapters(*a), ids)
    layer_case.check(got[-TAIL:], *layer_case.adapters(y[-TAIL:], x[-TAIL:], *a, ids[-TAIL:]), "rows")
    assert not got[:-TAIL].any()


def test_many_adapters():
    """The last adapter's matrices lie more than 2^31 values behind the first's."""
    N, K, r, n = 24576, 8, 128, 700
    up = torch.zeros(n, N, r, dtype=torch.bfloat16, device="cuda")
    down = torch.randn(n, r, K, device="cuda").bfloat16()
    up[-1].normal_()
    for T in (20, 300):
        x, y = torch.randn(T, K, device="cuda").bfloat16(), torch.randn(T, N, device="cuda").bfloat16()
        ids = torch.randint(n - 2, n, (T,), device="cuda", dtype=torch.int32)
        got = fops.add_adapters(y, x, fops.Adapters(down, up, torch.ones(n, device="cuda")), ids)
        layer_case.check(got, *layer_case.adapters(y, x, down[-2:], up[-2:], torch.ones(2, device="cuda"), ids - (n - 2)), "T=%d" % T)
