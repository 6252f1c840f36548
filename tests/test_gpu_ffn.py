"""The dense gated feed-forward block against its definition in float64: forward, backward, the ways
a caller may hand tensors over, capture into a graph."""
import ctypes

import pytest
import torch

from flash_distributed_moe_amd import _lib
from tests import ffn_case

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
# tokens, hidden, intermediate: one of everything, odd numbers of tokens, sizes on and around the
# tiles' 64, 128 and 256, k that ends inside a step
SHAPES = [(1, 8, 8), (3, 64, 32), (16, 256, 128), (17, 72, 40), (33, 520, 264), (64, 128, 512), (65, 1344, 736),
          (129, 264, 136), (130, 256, 128), (257, 136, 328), (300, 512, 1024), (5, 4096, 72), (12, 72, 4104), (27, 2048, 6144)]


@pytest.fixture(scope="module")
def ops():
    from flash_distributed_moe_amd import flashFfnOp

    return flashFfnOp


def make(T, H, I, dtype, seed=0, sigma=1.0):
    gen = torch.Generator(device="cuda").manual_seed(1000 + seed)

    def normal(s, *shape):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, s, generator=gen)

    return normal(sigma, T, H), normal(H ** -0.5, 2 * I, H), normal(I ** -0.5, H, I), normal(1.0, T, H)


def run(ops, x, w13, w2, dy, act):
    leaves = [t.detach().requires_grad_() for t in (x, w13, w2)]
    y = ops.gated_ffn(*leaves, activation=act)
    dx, dw13, dw2 = torch.autograd.grad(y, leaves, dy)
    return dict(y=y, dx=dx, dw13=dw13, dw2=dw2)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("T,H,I", SHAPES)
def test_forward_and_backward(ops, T, H, I, act, dtype):
    x, w13, w2, dy = make(T, H, I, DTYPES[dtype], sigma=2.0)
    want = ffn_case.block(x, w13, w2, act, dy)
    got = run(ops, x, w13, w2, dy, act)
    for name, t in got.items():
        assert t.dtype == DTYPES[dtype] and t.is_contiguous()
        ffn_case.check(t, *want[name], "%s of T=%d H=%d I=%d" % (name, T, H, I))
    # without gradients the same values come out, and nothing is kept
    y = ops.gated_ffn(x, w13, w2, activation=act)
    assert not y.requires_grad and torch.equal(y, got["y"])


# many tiles of the largest size in one product each: gated and slope / both weights' gradients / output and x's gradient
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("T,H,I", [(3841, 72, 3600), (77, 3600, 3904), (3841, 3600, 40), (2000, 640, 1000), (1100, 1304, 2600)])
def test_large_tiles(ops, T, H, I, dtype):
    x, w13, w2, dy = make(T, H, I, DTYPES[dtype], seed=6)
    want = ffn_case.block(x, w13, w2, "silu", dy)
    got = run(ops, x, w13, w2, dy, "silu")
    for name, t in got.items():
        ffn_case.check(t, *want[name], "%s of T=%d H=%d I=%d" % (name, T, H, I))


# few tiles and long sums, shared between workgroups: gated (H long), output and x's gradient (I long), slope (H long),
# the weights' gradients (T long)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("T,H,I", [(67, 384, 7680), (9, 136, 4104), (50, 4360, 72), (8200, 72, 40), (2100, 200, 3000), (1, 136, 5000)])
def test_long_sums(ops, T, H, I, dtype):
    x, w13, w2, dy = make(T, H, I, DTYPES[dtype], seed=7)
    want = ffn_case.block(x, w13, w2, "gelu_tanh", dy)
    got = run(ops, x, w13, w2, dy, "gelu_tanh")
    for name, t in got.items():
        ffn_case.check(t, *want[name], "%s of T=%d H=%d I=%d" % (name, T, H, I))
    for name, t in run(ops, x, w13, w2, dy, "gelu_tanh").items():
        assert torch.equal(t, got[name]), name
    for only in ("dx", "dw13", "dw2"):
        leaves = [v.detach().requires_grad_(n == only) for n, v in (("dx", x), ("dw13", w13), ("dw2", w2))]
        leaf = next(v for v in leaves if v.requires_grad)
        one, = torch.autograd.grad(ops.gated_ffn(*leaves, activation="gelu_tanh"), [leaf], dy)
        ffn_case.check(one, *want[only], "%s alone of T=%d H=%d I=%d" % (only, T, H, I))


def test_saving_without_a_workspace():
    """A C caller's forward pass that keeps its results needs no workspace, and then shares no sums; with one it
    writes nothing behind it."""
    lib = _lib.load()
    T, H, I = 67, 384, 7680
    x, w13, w2, _ = make(T, H, I, torch.bfloat16, seed=8)
    want = ffn_case.block(x, w13, w2, "silu")["y"]
    d = _lib.FfnDesc(H, I, _lib.BF16, _lib.ACT_SILU, _lib.FFN_ROW_MAJOR, w13.data_ptr(), w2.data_ptr(), None, None)
    saved, work = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert lib.flashMoeFfnBytes(ctypes.byref(d), T, ctypes.byref(saved), None, None) == 0
    assert lib.flashMoeFfnSavingBytes(ctypes.byref(d), T, ctypes.byref(work)) == 0
    assert work.value > 0
    keep = torch.full((saved.value + 256,), 0xA5, dtype=torch.uint8, device="cuda")
    room = torch.full((work.value + 256,), 0xA5, dtype=torch.uint8, device="cuda")
    for workspace in (None, room.data_ptr()):
        y = torch.empty_like(x)
        rc = lib.flashMoeFfnForward(ctypes.byref(d), x.data_ptr(), H, y.data_ptr(), H, T, keep.data_ptr(), workspace,
                                    torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == 0
        ffn_case.check(y, *want, "y")
    assert (keep[saved.value:] == 0xA5).all() and (room[work.value:] == 0xA5).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_gradients_against_differences(ops, dtype):
    """Central differences of the float64 definition along random directions: the analytic gradients
    are those of the function that the forward pass computes."""
    T, H, I = 9, 64, 48
    x, w13, w2, dy = make(T, H, I, torch.float32, seed=3)
    x, w13, w2, dy = (t.to(DTYPES[dtype]) for t in (x, w13, w2, dy))
    got = run(ops, x, w13, w2, dy, "gelu_tanh")
    want = ffn_case.block(x, w13, w2, "gelu_tanh", dy)

    def loss(a, b, c):
        g, u = (a @ b.t()).chunk(2, -1)
        return float(((ffn_case.parts(g, "gelu_tanh")[0] * u) @ c.t() * dy.double()).sum())

    base = [t.double() for t in (x, w13, w2)]
    eps = 1e-5
    for i, name in enumerate(("dx", "dw13", "dw2")):
        for k in range(4):
            d = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(k), dtype=torch.float64).to("cuda")
            up, down = list(base), list(base)
            up[i], down[i] = base[i] + eps * d, base[i] - eps * d
            slope = (loss(*up) - loss(*down)) / (2 * eps)
            # third derivatives times eps^2, rounding of a loss of size ~100 over eps: both below 1e-6
            far = float((want[name][1].reshape(d.shape) * d.abs()).sum()) + 1e-6 * (1 + abs(slope))
            assert abs(float((got[name].double() * d).sum()) - slope) <= far


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_strides_and_leading_dimensions(ops, dtype):
    dt = DTYPES[dtype]
    T, H, I = 21, 136, 72
    x, w13, w2, dy = make(T, H, I, dt, seed=1)
    plain = run(ops, x, w13, w2, dy, "silu")
    wide = torch.full((T, 3 * H), float("nan"), dtype=dt, device="cuda")
    wide[:, H:2 * H] = x
    odd = torch.full((T * H + 1,), float("nan"), dtype=dt, device="cuda")
    odd[1:] = x.reshape(-1)
    for name, xs in (("rows apart", wide[:, H:2 * H]), ("not on 16 bytes", odd[1:].view(T, H)),
                     ("columns apart", x.t().contiguous().t()), ("3 x 7", x.view(3, 7, H)),
                     ("1 x 21", x[None])):
        got = run(ops, xs, w13, w2, dy.view(xs.shape), "silu")
        for k in plain:
            assert torch.equal(got[k].reshape(plain[k].shape), plain[k]), "%s: %s" % (name, k)
    one = ops.gated_ffn(x[4], w13, w2)
    assert one.shape == (H,)
    ffn_case.check(one, *ffn_case.block(x[4:5], w13, w2, "silu")["y"], "a row without a batch")
    # a gradient that is one value for everything
    leaves = [t.detach().requires_grad_() for t in (x, w13, w2)]
    ops.gated_ffn(*leaves).sum().backward()
    want = ffn_case.block(x, w13, w2, "silu", torch.ones_like(x))
    for leaf, name in zip(leaves, ("dx", "dw13", "dw2")):
        ffn_case.check(leaf.grad, *want[name], name + " of a sum")


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_broadcast_rows_and_gradients(ops, dtype):
    """A row of x that all tokens share, and an output's gradient that is one number or lies transposed."""
    dt = DTYPES[dtype]
    T, H, I = 19, 72, 40
    x, w13, w2, dy = make(T, H, I, dt, seed=9)
    one = x[:1]
    want = ffn_case.block(one.expand(T, H), w13, w2, "silu", torch.ones_like(x))
    leaves = [v.detach().requires_grad_() for v in (one, w13, w2)]
    ops.gated_ffn(leaves[0].expand(T, H), *leaves[1:]).sum().backward()
    dx, far = want["dx"]
    # autograd adds the rows' gradients in float32 and rounds once
    total = 2 * T * 2.0 ** -24 * (dx.abs() + far).sum(0) + far.sum(0)
    ffn_case.check(leaves[0].grad, dx.sum(0)[None], (total + ffn_case.HALF[dt] * (dx.sum(0).abs() + total))[None], "shared row")
    for name, leaf in (("dw13", leaves[1]), ("dw2", leaves[2])):
        ffn_case.check(leaf.grad, *want[name], name)
    plain = run(ops, x, w13, w2, dy, "silu")
    for other in (dy.t().contiguous().t(), torch.cat((dy, dy), 1)[:, :H]):
        for name, v in run(ops, x, w13, w2, other, "silu").items():
            assert torch.equal(v, plain[name]), name


def test_graph_kept_and_weights_used_twice(ops):
    T, H, I = 23, 64, 48
    x, w13, w2, dy = make(T, H, I, torch.float32, seed=10)
    leaves = [v.detach().requires_grad_() for v in (x, w13, w2)]
    y = ops.gated_ffn(*leaves)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, dy)
    # the same block twice, one output the other's input: the weights' gradients add up
    mid = ops.gated_ffn(*leaves)
    got = torch.autograd.grad(ops.gated_ffn(mid, *leaves[1:]), leaves, dy)
    second = run(ops, mid.detach(), w13, w2, dy, "silu")
    below = run(ops, x, w13, w2, second["dx"], "silu")
    assert torch.equal(got[0], below["dx"])
    assert torch.equal(got[1], second["dw13"] + below["dw13"]) and torch.equal(got[2], second["dw2"] + below["dw2"])


def test_no_tokens(ops):
    x, w13, w2, dy = make(4, 64, 32, torch.bfloat16)
    got = run(ops, x[:0], w13, w2, dy[:0], "silu")
    assert got["y"].shape == (0, 64) and got["dx"].shape == (0, 64)
    assert not got["dw13"].any() and not got["dw2"].any() and got["dw13"].shape == w13.shape


@pytest.mark.parametrize("want", [(True, False, False), (False, True, False), (False, False, True), (False, True, True)])
def test_some_gradients_only(ops, want):
    x, w13, w2, dy = make(40, 128, 96, torch.bfloat16, seed=5)
    full = run(ops, x, w13, w2, dy, "silu")
    leaves = [t.detach().requires_grad_(need) for t, need in zip((x, w13, w2), want)]
    y = ops.gated_ffn(*leaves)
    y.backward(dy)
    for leaf, need, name in zip(leaves, want, ("dx", "dw13", "dw2")):
        assert (leaf.grad is not None) == need
        if need:
            assert torch.equal(leaf.grad, full[name])


def test_twice_differentiated_is_refused(ops):
    x, w13, w2, dy = make(4, 64, 32, torch.float32)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="no second derivatives"):
        torch.autograd.grad(ops.gated_ffn(x, w13, w2), x, dy, create_graph=True)


def test_changed_inputs_are_noticed(ops):
    x, w13, w2, dy = make(4, 64, 32, torch.float32)
    w2.requires_grad_()
    y = ops.gated_ffn(x, w13, w2)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_rows_with_infinities_and_nan_keep_to_themselves(ops, value, dtype):
    """A row that holds no number has no number as its result, and no other row changes."""
    T, H, I = 70, 128, 64
    x, w13, w2, dy = make(T, H, I, DTYPES[dtype], seed=2)
    clean = ops.gated_ffn(x, w13, w2)
    x[5, 7] = value
    got = ops.gated_ffn(x, w13, w2)
    rest = [t for t in range(T) if t != 5]
    assert torch.equal(got[rest], clean[rest])
    assert not torch.isfinite(got[5]).any()


def test_float32_beyond_what_bfloat16_parts_hold(ops):
    """Inputs so small that their parts are below bfloat16's range, and infinities of one sign: the sums are
    float32's all the same."""
    T, H, I = 130, 64, 64
    x, w13, w2, dy = make(T, H, I, torch.float32, seed=8)
    tiny = 2.0 ** -115
    for scaled in ((x * tiny, w13, w2), (x, w13 * tiny, w2), (x, w13, w2 * tiny)):
        want = ffn_case.block(*scaled, "silu")["y"]
        ffn_case.check(ops.gated_ffn(*scaled), *want, "a tiny operand")
    # positive everything: an infinite token gives infinite outputs, not NaN
    x, w13, w2 = x.abs(), w13.abs(), w2.abs()
    x[3, 5] = float("inf")
    y = ops.gated_ffn(x, w13, w2)
    assert torch.isposinf(y[3]).all() and torch.isfinite(y[:3]).all() and torch.isfinite(y[4:]).all()


def test_large_projections_saturate(ops):
    """Gates far out: silu is the gate itself or zero there, and no exponential's overflow shows."""
    H = I = 64
    for dt in DTYPES.values():
        x = torch.eye(H, dtype=dt, device="cuda")
        w13 = torch.cat((torch.full((I, H), -3e4), torch.ones(I, H))).to("cuda", dt)
        w13[:I // 2] = 3e4
        w2 = torch.eye(I, dtype=dt, device="cuda")
        for act in ("silu", "gelu_tanh"):
            y = ops.gated_ffn(x, w13, w2, activation=act)
            assert not y[:, I // 2:].any()
            assert torch.equal(y[:, :I // 2], w13[:I // 2].t().contiguous())


def test_on_another_stream_and_two_at_once(ops):
    x, w13, w2, dy = make(200, 512, 256, torch.bfloat16, seed=7)
    want = run(ops, x, w13, w2, dy, "silu")
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for rep in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run(ops, x, w13, w2, dy, "silu"))
    torch.cuda.synchronize()
    for g in got:
        for k in want:
            assert torch.equal(g[k], want[k])


@pytest.mark.parametrize("T", [1, 48, 300])
def test_captured_step(ops, T):
    """Forward and backward in one graph, replayed with fresh inputs; two graphs of different batches
    alternate and each finds its own workspace."""
    def captured(T, seed):
        x, w13, w2, dy = make(T, 256, 136, torch.bfloat16, seed=seed)
        leaves = [t.detach().requires_grad_() for t in (x, w13, w2)]

        def step():
            y = ops.gated_ffn(*leaves)
            return (y, *torch.autograd.grad(y, leaves, dy))

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        return graph, leaves, dy, out

    graphs = [captured(T, 11), captured(T + 5, 12)]
    for rep in range(4):
        for graph, leaves, dy, out in graphs:
            with torch.no_grad():
                for t in (*leaves, dy):
                    t.copy_(torch.randn(t.shape, device="cuda") * t.shape[-1] ** -0.5)
            graph.replay()
            torch.cuda.synchronize()
            want = run(ops, leaves[0], leaves[1], leaves[2], dy, "silu")
            for a, k in zip(out, ("y", "dx", "dw13", "dw2")):
                assert torch.equal(a, want[k]), "replay %d: %s" % (rep, k)


def test_capture_beside_a_living_eager_graph_is_refused(ops):
    """Its leaves' accumulators belong to the eager graph's stream, which a captured backward pass would make wait."""
    x, w13, w2, dy = make(20, 64, 32, torch.bfloat16)
    leaves = [t.detach().requires_grad_() for t in (x, w13, w2)]
    alive = ops.gated_ffn(*leaves)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph):
            ops.gated_ffn(*leaves)
    # without gradients there is nothing to refuse, and the eager graph still works
    plain = torch.cuda.CUDAGraph()
    with torch.cuda.graph(plain), torch.no_grad():
        y = ops.gated_ffn(*leaves)
    plain.replay()
    alive.backward(dy)
    torch.cuda.synchronize()
    assert torch.equal(y, alive)
    ffn_case.check(leaves[1].grad, *ffn_case.block(x, w13, w2, "silu", dy)["dw13"], "dw13")


def test_same_bits_every_time(ops):
    x, w13, w2, dy = make(700, 512, 264, torch.bfloat16, seed=9)
    first = run(ops, x, w13, w2, dy, "silu")
    for _ in range(3):
        again = run(ops, x, w13, w2, dy, "silu")
        for k in first:
            assert torch.equal(first[k], again[k])


def test_c_abi_in_place_and_neighbours_left_alone():
    """Output over input, rows apart; what lies between and behind the rows stays as it was."""
    lib = _lib.load()
    T, H, I, ld = 37, 72, 40, 88
    x, w13, w2, _ = make(T, H, I, torch.bfloat16, seed=4)
    buf = torch.full((T + 2, ld), 7.0, dtype=torch.bfloat16, device="cuda")
    buf[:T, :H] = x
    d = _lib.FfnDesc(H, I, _lib.BF16, _lib.ACT_SILU, _lib.FFN_ROW_MAJOR, w13.data_ptr(), w2.data_ptr(), None, None)
    n = ctypes.c_size_t(0)
    assert lib.flashMoeFfnBytes(ctypes.byref(d), T, None, ctypes.byref(n), None) == 0
    work = torch.full((n.value + 256,), 0xA5, dtype=torch.uint8, device="cuda")
    rc = lib.flashMoeFfnForward(ctypes.byref(d), buf.data_ptr(), ld, buf.data_ptr(), ld, T, None, work.data_ptr(),
                                torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0
    ffn_case.check(buf[:T, :H], *ffn_case.block(x, w13, w2, "silu")["y"], "in place")
    assert (buf[T:] == 7).all() and (buf[:, H:] == 7).all()
    assert (work[n.value:] == 0xA5).all()
