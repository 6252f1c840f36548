"""Calls of the operators around a layer's blocks at the limits of what is documented: values next to the end of their
type's range, views that are negated when they are read, tensors without memory, results over other operands."""
import pytest
import torch
from torch._subclasses import FakeTensorMode

from flash_distributed_moe_amd import flashFfnOp as fops, flashLayerOp as ops
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_squares_beyond_float32(dtype):
    """The row's norm is zeros, as documented, its sum with the branch is not, and no other row notices."""
    x, w = torch.randn(5, 264, device="cuda").to(dtype), torch.ones(264, device="cuda", dtype=dtype)
    large = x.clone()
    large[2] = 2.0 ** 70
    rest = torch.arange(5, device="cuda") != 2
    h = ops.block_norm(large, w)
    assert not h[2].any() and torch.equal(h[rest], ops.block_norm(x, w)[rest])
    y, h = ops.block_join(x, large, w, None, w)
    assert torch.equal(y[2], x[2])
    y, h = ops.block_join(large, x, None, None, w)
    assert (y[2] == 2.0 ** 70).all() and not h[2].any()


# ------------------------------------------------------------------ views that are negated when they are read
def negated(values):
    """-values as a view that carries the negation with it."""
    t = torch.complex(torch.zeros_like(values), values).conj().imag
    assert t.is_neg()
    return t


def test_negated_gradients_of_the_losses():
    gen = torch.Generator(device="cuda").manual_seed(8000)
    logits = torch.empty(100, 24, device="cuda").normal_(generator=gen)
    db, dz = negated(torch.tensor(-0.3, device="cuda")), negated(torch.tensor(0.2, device="cuda"))
    dw = negated(torch.empty(100, 4, device="cuda").normal_(generator=gen))
    leaf = logits.clone().requires_grad_()
    r = ops.route(leaf, 4)
    got, = torch.autograd.grad([r.weights, r.balance_loss, r.z_loss], leaf, [dw, db, dz])
    layer_case.check(got, *layer_case.route(logits, 4, True, None, dw.resolve_neg(), db.resolve_neg(), dz.resolve_neg())["dlogits"], "dlogits")


@pytest.mark.parametrize("packed", [False, True])
def test_negated_inputs(packed):
    """Rows, gates and upstream gradients; packed: without gaps, as torch keeps the negation of some of its own results."""
    gen = torch.Generator(device="cuda").manual_seed(8001)
    draw = lambda *s: torch.empty(s, device="cuda").normal_(generator=gen)  # noqa: E731
    turn = (lambda t: torch._neg_view(t)) if packed else negated  # noqa: E731
    x, branch, gate, dy, w = draw(6, 64), draw(6, 64), draw(6, 1), draw(6, 64), draw(64)
    leaves = [t.clone().requires_grad_() for t in (x, branch, gate, w)]
    y, h = ops.block_join(turn(leaves[0]), turn(leaves[1]), leaves[3], turn(leaves[2]), leaves[3])
    want = layer_case.join(-x, -branch, w, -gate, w)
    layer_case.check(y, *want["y"], "y")
    layer_case.check(h, *want["h"], "h")
    plain = [t.clone().requires_grad_() for t in (-x, -branch, -gate)]
    py, ph = ops.block_join(plain[0], plain[1], w, plain[2], w)
    got = torch.autograd.grad([y, h], leaves[:3], [turn(dy), turn(dy)])
    want = torch.autograd.grad([py, ph], plain, [-dy, -dy])
    for a, b in zip(got, want):
        assert torch.equal(a, -b)
    logits = draw(9, 1)
    assert torch.equal(ops.route(turn(logits), 1).z_loss, ops.route(-logits, 1).z_loss)
    one = draw(1)
    assert torch.equal(ops.route(turn(one), 1).z_loss, ops.route(-one, 1).z_loss)
    q = fops.quantize_mxfp4(turn(x))
    assert torch.equal(fops.dequantize_mxfp4(q), fops.dequantize_mxfp4(fops.quantize_mxfp4(-x)))


@pytest.mark.parametrize("which", ["post", "next", "weight", "down", "up", "scales"])
def test_negated_weights_are_refused(which):
    """Weights are not copied at every call."""
    turn = lambda t, name: torch._neg_view(t) if name == which else t  # noqa: E731
    x, w = torch.randn(3, 64, device="cuda"), torch.ones(64, device="cuda")
    b = x.bfloat16()
    a = dict(down=torch.zeros(1, 8, 64, device="cuda").bfloat16(), up=torch.zeros(1, 64, 8, device="cuda").bfloat16(), scales=torch.ones(1, device="cuda"))
    with pytest.raises(RuntimeError, match="negated"):
        if which in a:
            fops.add_adapters(b, b, fops.Adapters(**{k: turn(t, k) for k, t in a.items()}), torch.zeros(3, dtype=torch.int32, device="cuda"))
        elif which == "weight":
            ops.block_norm(x, turn(w, "weight"))
        else:
            ops.block_join(x, x, turn(w, "post"), None, turn(w, "next"))


# ------------------------------------------------------------------ tensors without memory
def fake(*shape, dtype=torch.float32, view=False):
    with FakeTensorMode():
        t = torch.ones((2, *shape), dtype=dtype, device="cuda")
        return t[1] if view else t[0]


@pytest.mark.parametrize("view", [False, True])
@pytest.mark.parametrize("which", ["mask", "post", "gate", "next", "branch", "ids", "scales"])
def test_arguments_without_memory_are_refused(which, view):
    """They would count as left out: rows without a mask, a norm without its weight."""
    pick = lambda name, t: fake(*t.shape, dtype=t.dtype, view=view) if name == which else t  # noqa: E731
    x, w = torch.randn(3, 64, device="cuda"), torch.ones(64, device="cuda")
    b, ids = x.bfloat16(), torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="no memory of its own"):
        if which == "mask":
            ops.route(x, 2, mask=pick("mask", torch.ones(3, dtype=torch.bool, device="cuda")))
        elif which in ("ids", "scales"):
            a = fops.Adapters(torch.zeros(1, 8, 64, device="cuda").bfloat16(), torch.zeros(1, 64, 8, device="cuda").bfloat16(),
                              pick("scales", torch.ones(1, device="cuda")))
            fops.add_adapters(b, b, a, pick("ids", ids))
        else:
            ops.block_join(x, pick("branch", x), pick("post", w), pick("gate", w), pick("next", w))


def test_gradients_of_zeros_without_memory():
    """What torch makes for derivatives that are nothing counts as zeros."""
    x, w = torch.randn(6, 64, device="cuda"), torch.ones(64, device="cuda")
    leaves = [x.clone().requires_grad_(), x.clone().requires_grad_()]
    dy = torch.randn(6, 64, device="cuda")
    nothing = torch._efficientzerotensor((6, 64), device="cuda")
    y, h = ops.block_join(*leaves, w, None, w)
    got = torch.autograd.grad([y, h], leaves, [dy, nothing], retain_graph=True)
    for a, b in zip(got, torch.autograd.grad(y, leaves, dy)):
        assert torch.equal(a, b)
    r = ops.route(leaves[0], 3)
    got, = torch.autograd.grad([r.weights, r.z_loss], leaves[0], [dy[:, :3], torch._efficientzerotensor((), device="cuda")], retain_graph=True)
    want, = torch.autograd.grad(r.weights, leaves[0], dy[:, :3])
    assert torch.equal(got, want)


# ------------------------------------------------------------------ results over other operands
@pytest.mark.parametrize("T", [4, 900])
def test_results_over_the_adapters_are_refused(T):
    """Rows that are written while others' adapters are still read."""
    r, n = 8, 300
    K = N = 64
    buffer = torch.zeros(n * N * r + n * r * K, device="cuda", dtype=torch.bfloat16)
    up, down = buffer[:n * N * r].view(n, N, r), buffer[n * N * r:].view(n, r, K)
    x, y = torch.randn(T, K, device="cuda").bfloat16(), torch.randn(T, N, device="cuda").bfloat16()
    places = torch.zeros(T, N // 2, device="cuda", dtype=torch.int32)  # as many bytes as y: ids are a column of it
    ids, scales = places[:, 0], torch.ones(n, device="cuda")
    a = fops.Adapters(down, up, scales)
    for out in (buffer[:T * N].view(T, N), buffer[-T * N:].view(T, N), buffer[n * N * r - T * N // 2:][:T * N].view(T, N), places.view(torch.bfloat16)):
        with pytest.raises(RuntimeError, match="apart from the adapters and ids"):
            fops.add_adapters(y, x, a, ids, out=out)
    # next to them on either side
    whole = torch.zeros(2 * T * N + N * r, device="cuda", dtype=torch.bfloat16)
    one = fops.Adapters(torch.zeros(1, r, K, device="cuda").bfloat16(), whole[T * N:T * N + N * r].view(1, N, r), scales[:1])
    for out in (whole[:T * N].view(T, N), whole[T * N + N * r:][:T * N].view(T, N)):
        assert fops.add_adapters(y, x, one, ids, out=out) is out and torch.equal(out, y)
