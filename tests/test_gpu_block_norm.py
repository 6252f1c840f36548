"""The norms before and after a block, the gate and the residual's scale against their definition in float64, forward and backward."""
import pytest
import torch

from tests import layer_case

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
# batch, tokens of a sequence, width: one piece of a row, ragged ones, around a wave's, two waves', four waves' and eight waves' widths,
# one token, more tokens than workgroups, few tokens spread over many lanes and many that are not
SHAPES = [(1, 1, 8), (1, 1, 8192), (1, 3, 72), (2, 5, 264), (3, 7, 1024), (1, 13, 1032), (2, 16, 2048), (1, 9, 2056), (1, 33, 4096), (5, 3, 4104),
          (1, 17, 5120), (7, 200, 136), (2, 600, 1344), (3, 400, 8192), (1, 4100, 520)]
GATES = {"none": lambda B, S, H: None, "channel": lambda B, S, H: (H,), "sequence": lambda B, S, H: (B, 1, H), "token": lambda B, S, H: (B, S, 1),
         "full": lambda B, S, H: (B, S, H)}


@pytest.fixture(scope="module")
def ops():
    from flash_distributed_moe_amd import flashLayerOp

    return flashLayerOp


def make(B, S, H, dtype, gate="channel", post=True, nxt=True, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(5000 + seed)

    def normal(sigma, *shape, mean=0.0):
        return torch.empty(shape, device="cuda").normal_(mean, sigma, generator=gen).to(dtype)

    shape = GATES[gate](B, S, H)
    return dict(x=normal(1.0, B, S, H), branch=normal(3.0, B, S, H), post=normal(0.5, H, mean=1.0) if post else None,
                gate=normal(0.5, *shape, mean=0.5) if shape else None, next_weight=normal(0.5, H, mean=1.0) if nxt else None), \
        dict(dy=normal(1.0, B, S, H), dh=normal(1.0, B, S, H) if nxt else None)


def run(ops, given, up, alpha=0.75, beta=1.5, eps=1e-6):
    leaves = {k: t.detach().requires_grad_() for k, t in given.items() if t is not None}
    got = ops.block_join(leaves["x"], leaves["branch"], leaves.get("post"), leaves.get("gate"), leaves.get("next_weight"),
                         residual_scale=alpha, branch_scale=beta, eps=eps)
    out = dict(zip(("y", "h"), got if given["next_weight"] is not None else (got,)))
    pairs = [(out[k], up["d" + k]) for k in out if up.get("d" + k) is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [d for _, d in pairs], allow_unused=True)
    return {**out, **dict(zip(leaves, grads))}


def compare(ops, given, up, what, alpha=0.75, beta=1.5, eps=1e-6, **given_as):
    want = layer_case.join(**given, alpha=alpha, beta=beta, eps=eps, **up)
    got = run(ops, {**given, **given_as}, up, alpha, beta, eps)
    assert set(got) == set(want)
    for name, t in got.items():
        assert t.dtype == given["x"].dtype and t.shape == (given.get(name, given["x"]) if name in given else given["x"]).shape
        layer_case.check(t, *want[name], "%s of %s" % (name, what))
    return got


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("gate", sorted(GATES))
@pytest.mark.parametrize("B,S,H", SHAPES)
def test_join(ops, B, S, H, gate, dtype):
    given, up = make(B, S, H, DTYPES[dtype], gate)
    got = compare(ops, given, up, "%s %s" % ((B, S, H), gate))
    # without gradients the same values come out
    y, h = ops.block_join(given["x"], given["branch"], given["post"], given["gate"], given["next_weight"], 0.75, 1.5)
    assert not y.requires_grad and torch.equal(y, got["y"]) and torch.equal(h, got["h"])


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("gate", sorted(GATES))
@pytest.mark.parametrize("post,nxt", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("B,S,H", [(3, 50, 200), (2, 300, 4096)])
def test_parts_of_a_join(ops, B, S, H, post, nxt, gate, dtype):
    given, up = make(B, S, H, DTYPES[dtype], gate, post, nxt, seed=1)
    compare(ops, given, up, "%s %s" % ((B, S, H), gate))


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("B,S,H", SHAPES)
def test_norm(ops, B, S, H, dtype):
    given, up = make(B, S, H, DTYPES[dtype], "none", seed=2)
    want = layer_case.join(given["x"], next_weight=given["next_weight"], eps=1e-5, dh=up["dh"])
    leaves = [given[k].detach().requires_grad_() for k in ("x", "next_weight")]
    h = ops.block_norm(*leaves, eps=1e-5)
    grads = torch.autograd.grad(h, leaves, up["dh"])
    for name, t in zip(("h", "x", "next_weight"), (h, *grads)):
        layer_case.check(t, *want[name], "%s of %s" % (name, (B, S, H)))
    assert torch.equal(ops.block_norm(given["x"], given["next_weight"], eps=1e-5), h)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("B,S", [(1, 2000), (2000, 1), (700, 3), (3, 700), (513, 5), (64, 64), (600, 2)])
def test_groups_of_rows(ops, B, S, dtype):
    """Gates of few long and of many short sequences: parts of a group a workgroup, and several groups."""
    given, up = make(B, S, 136, DTYPES[dtype], "sequence", seed=3)
    got = compare(ops, given, up, "%d x %d" % (B, S))
    for name, t in run(ops, given, up).items():
        assert torch.equal(t, got[name]), name


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_one_upstream_gradient_alone(ops, dtype):
    given, up = make(2, 70, 1000, DTYPES[dtype], "channel", seed=4)
    compare(ops, given, dict(dy=up["dy"], dh=None), "dy alone")
    compare(ops, given, dict(dy=None, dh=up["dh"]), "dh alone")


@pytest.mark.parametrize("gate", sorted(GATES))
def test_one_input_s_gradient_alone(ops, gate):
    given, up = make(2, 70, 264, torch.float32, gate, seed=5)
    whole = run(ops, given, up)
    for name, t in given.items():
        if t is None:
            continue
        leaf = t.detach().requires_grad_()
        args = {**given, name: leaf}
        out = ops.block_join(args["x"], args["branch"], args["post"], args["gate"], args["next_weight"], 0.75, 1.5)
        grad, = torch.autograd.grad(out, [leaf], [up["dy"], up["dh"]])
        assert torch.equal(grad, whole[name]), name


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_ways_to_hand_rows_over(ops, dtype):
    """Rows that lie apart, columns, odd places, expanded inputs and gradients, gates as slices of one projection."""
    B, S, H = 2, 40, 264
    given, up = make(B, S, H, DTYPES[dtype], "sequence", seed=6)
    wide = torch.full((B, S, H + 24), 7.0, dtype=given["x"].dtype, device="cuda")
    wide[..., 8:H + 8] = given["x"]
    odd = torch.full((B, S, H + 5), 7.0, dtype=given["x"].dtype, device="cuda")
    odd[..., 3:H + 3] = given["branch"]
    compare(ops, given, up, "rows apart", x=wide[..., 8:H + 8], branch=odd[..., 3:H + 3])
    compare(ops, given, up, "transposed", x=given["x"].transpose(0, 1).contiguous().transpose(0, 1))
    six = torch.zeros(B, 6 * H, dtype=given["x"].dtype, device="cuda")
    six[:, H:2 * H] = given["gate"][:, 0]
    compare(ops, given, up, "a slice of a projection", gate=six.chunk(6, -1)[1].unsqueeze(1))
    same = {**given, "x": given["x"][:1].expand(B, S, H)}
    one = dict(dy=up["dy"][..., :1].expand(B, S, H), dh=up["dh"][:, :1].expand(B, S, H))
    compare(ops, same, one, "expanded")
    gate = given["gate"].expand(B, S, H)
    compare(ops, {**given, "gate": gate}, up, "an expanded gate")
    compare(ops, {**given, "gate": given["gate"][:1, 0]}, up, "a gate of [1, H]")


def test_rows_that_are_zero_or_not_finite(ops):
    given, up = make(1, 30, 512, torch.float32, "channel", seed=7)
    given["x"][0, 3] = 0
    given["branch"][0, 3] = 0
    compare(ops, given, up, "a row of zeros", eps=1e-2)
    bad = {**given, "x": given["x"].clone()}
    bad["x"][0, 11, 100] = float("nan")
    a, b = run(ops, given, up), run(ops, bad, up)
    rest = torch.arange(30, device="cuda") != 11
    for name in ("y", "h", "x", "branch"):
        assert torch.equal(a[name][0, rest], b[name][0, rest]), name
    assert torch.isnan(b["h"][0, 11]).all() and torch.isnan(b["x"][0, 11]).any() and torch.isnan(b["next_weight"]).all()


def test_no_tokens(ops):
    for gate in sorted(GATES):
        given, up = make(2, 0, 64, torch.bfloat16, gate)
        got = run(ops, given, up)
        assert got["y"].shape == (2, 0, 64) and not got["next_weight"].any() and not got["post"].any()
        if gate in ("channel", "sequence"):
            assert not got["gate"].any()


@pytest.mark.parametrize("gate", [(3, 1), (1,), (2, 1, 1), (1, 5, 64), (1, 1, 2, 5, 64), (64, 1)])
def test_gates_of_other_shapes_are_refused(ops, gate):
    x = torch.zeros(2, 5, 64, device="cuda")
    with pytest.raises(RuntimeError, match="gate"):
        ops.block_join(x, x, gate=torch.zeros(gate, device="cuda"))


@pytest.mark.parametrize("change", [dict(branch=(2, 5, 56)), dict(post=(56,)), dict(next_weight=(1, 64)), dict(x=(2, 5, 63)), dict(x=(2, 5, 8200))])
def test_other_shapes_are_refused(ops, change):
    args = {k: torch.zeros(change.get(k, s), device="cuda") for k, s in dict(x=(2, 5, 64), branch=(2, 5, 64), post=(64,), gate=(64,), next_weight=(64,)).items()}
    with pytest.raises(RuntimeError):
        ops.block_join(*args.values())
    with pytest.raises(RuntimeError, match="dtype"):
        ops.block_join(torch.zeros(2, 64, device="cuda"), torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16))


def test_second_derivatives_are_refused(ops):
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(ops.block_norm(x, torch.ones(64, device="cuda")).sum(), x, create_graph=True)


@pytest.mark.parametrize("gate", ["channel", "sequence", "token"])
def test_captured_step(ops, gate):
    given, up = make(2, 300, 2048, torch.bfloat16, gate, seed=8)
    still = {k: t.clone() for k, t in given.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(ops, still, up)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(ops, still, up)
    for rep in range(4):
        fresh, _ = make(2, 300, 2048, torch.bfloat16, gate, seed=20 + rep)
        for k, t in fresh.items():
            still[k].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for name, t in run(ops, fresh, up).items():
            assert torch.equal(t, got[name]), "%s, replay %d" % (name, rep)


def test_two_streams_at_once(ops):
    """Calls that overlap share nothing."""
    cases = [make(1, 500, 2048, torch.float32, "channel", seed=30 + i) for i in range(2)]
    want = [run(ops, *c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for s, c in zip(streams, cases):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([run(ops, *c) for _ in range(5)])
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for g in gs:
            assert all(torch.equal(g[k], w[k]) for k in w)
