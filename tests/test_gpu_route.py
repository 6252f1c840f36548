"""The router's choice and its losses against their definition in float64, forward and backward."""
import pytest
import torch

from tests import layer_case

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
# tokens, experts, k: one of everything, odd and whole fours, around 16 lanes, 64 columns, workgroups of 16 and 64 rows, and
# beyond one workgroup
SHAPES = [(1, 1, 1), (1, 128, 8), (3, 4, 4), (5, 7, 3), (16, 60, 4), (17, 64, 16), (63, 65, 17), (64, 128, 8), (65, 130, 32), (100, 17, 17),
          (257, 256, 32), (300, 255, 1), (1000, 32, 32), (4096, 64, 6), (4097, 200, 8), (9000, 128, 16)]


@pytest.fixture(scope="module")
def ops():
    from flash_distributed_moe_amd import flashLayerOp

    return flashLayerOp


def make(T, E, dtype, seed=0, sigma=2.0):
    gen = torch.Generator(device="cuda").manual_seed(4000 + seed)
    logits = torch.empty(T, E, device="cuda").normal_(0.0, sigma, generator=gen).to(dtype)
    return logits, gen


def compare(ops, logits, k, renormalize=True, mask=None, dw=None, db=None, dz=None, rows=None, what=""):
    """rows: how the operator is given the logits, if otherwise than as they are."""
    want = layer_case.route(logits, k, renormalize, mask, dw, db, dz)
    given = (logits if rows is None else rows).detach()
    train = "dlogits" in want
    leaf = given.requires_grad_(train)
    got = ops.route(leaf, k, renormalize=renormalize, mask=mask)
    assert got.experts.dtype == got.counts.dtype == torch.int32 and got.weights.dtype == torch.float32
    assert torch.equal(got.experts.long(), want["experts"]), what + " experts"
    assert torch.equal(got.counts.long(), want["counts"]), what + " counts"
    for name in ("weights", "balance_loss", "z_loss"):
        layer_case.check(getattr(got, name), *want[name], what + " " + name)
    if train:
        pairs = [(o, d) for o, d in ((got.weights, dw), (got.balance_loss, db), (got.z_loss, dz)) if d is not None]
        grad, = torch.autograd.grad([o for o, _ in pairs], [leaf], [d for _, d in pairs])
        assert grad.dtype == logits.dtype and grad.shape == logits.shape
        layer_case.check(grad, *want["dlogits"], what + " dlogits")
    return got


def upstream(T, k, gen):
    return dict(dw=torch.empty(T, k, device="cuda").normal_(generator=gen), db=torch.tensor(0.3, device="cuda"), dz=torch.tensor(-0.2, device="cuda"))


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("T,E,k", SHAPES)
def test_forward_and_backward(ops, T, E, k, dtype, renormalize):
    logits, gen = make(T, E, DTYPES[dtype])
    compare(ops, logits, k, renormalize, **upstream(T, k, gen), what="T=%d E=%d k=%d" % (T, E, k))


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("T,E,k", [(70, 60, 4), (5000, 128, 8), (33, 9, 9)])
def test_padding_and_barred_experts(ops, T, E, k, dtype):
    """Padding, experts at -inf, at the type's lowest value and NaN for some tokens, tokens with fewer candidates than k, tokens with none."""
    logits, gen = make(T, E, DTYPES[dtype], seed=1)
    mask = torch.rand(T, device="cuda", generator=gen) < 0.7
    draw = torch.rand(T, E, device="cuda", generator=gen)
    logits[draw < 0.2] = float("-inf")
    logits[(draw >= 0.2) & (draw < 0.3)] = torch.finfo(logits.dtype).min
    logits[(draw >= 0.3) & (draw < 0.4)] = float("nan")
    logits[::7] = float("-inf")
    logits[1::14, 2] = -3.0
    for renormalize in (True, False):
        got = compare(ops, logits, k, renormalize, mask, **upstream(T, k, gen), what="T=%d E=%d" % (T, E))
    assert (got.experts[0] == -1).all() and (got.weights[0] == 0).all()
    nothing = compare(ops, logits, k, True, torch.zeros_like(mask), **upstream(T, k, gen), what="all padding")
    assert float(nothing.balance_loss.detach()) == 0 and float(nothing.z_loss.detach()) == 0


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("E,k", [(256, 32), (128, 8), (60, 17), (16, 16)])
def test_equal_logits_go_to_the_lowest_expert(ops, E, k, dtype):
    logits, gen = make(200, E, DTYPES[dtype], seed=2)
    logits[:50] = 1.25
    logits[50:100] = torch.randint(0, 3, (50, E), device="cuda", generator=gen).to(logits.dtype)  # equals in many places
    logits[100:150] = -logits[50:100] * 1e30
    logits[150:160] = 0.0
    logits[150:160, ::2] = -0.0
    got = compare(ops, logits, k, **upstream(200, k, gen), what="E=%d" % E)
    assert torch.equal(got.experts[0].long(), torch.arange(k, device="cuda"))
    assert torch.equal(got.experts[150].long(), torch.arange(k, device="cuda"))


@pytest.mark.parametrize("E,k", [(256, 32), (128, 8), (40, 16), (256, 16), (17, 17)])
def test_neighbouring_floats(ops, E, k):
    """float32 logits that differ in their last bits only: among the winners, across the border between 16 and 17, and at the last winner."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    T = 256
    steps = torch.stack([torch.randperm(E, device="cuda", generator=gen) for _ in range(T)])
    logits = (1.0 + steps.float() * 2.0 ** -23) * torch.where(torch.arange(T, device="cuda") % 2 == 0, 1.0, -2.0)[:, None]
    compare(ops, logits, k, what="E=%d" % E)
    # only two of a row are neighbours, anywhere in its order
    logits, _ = make(T, E, torch.float32, seed=6)
    order = logits.argsort(1, descending=True)
    rows = torch.arange(T, device="cuda")
    j = rows % (E - 1)
    a, b = order[rows, j], order[rows, j + 1]
    logits[rows, b] = torch.nextafter(logits[rows, a], torch.full((T,), -1e9, device="cuda"))
    swap = rows % 2 == 0
    logits[rows[swap], a[swap]], logits[rows[swap], b[swap]] = logits[rows[swap], b[swap]].clone(), logits[rows[swap], a[swap]].clone()
    compare(ops, logits, k, what="E=%d pairs" % E)


def test_extremes(ops):
    """Large logits, far apart ones, and infinity, which makes a token's probabilities NaN and nobody else's choice."""
    logits, gen = make(40, 96, torch.float32, seed=3, sigma=1000.0)
    logits[5] *= 1e12
    compare(ops, logits, 6, **upstream(40, 6, gen), what="far apart")
    logits, gen = make(40, 96, torch.float32, seed=4)
    bad = logits.clone()
    bad[7, 11] = float("inf")
    got, fine = ops.route(bad, 6), ops.route(logits, 6)
    rest = torch.arange(40, device="cuda") != 7
    assert got.experts[7, 0] == 11 and torch.isnan(got.weights[7]).all()
    assert torch.equal(got.weights[rest], fine.weights[rest]) and torch.equal(got.experts[rest], fine.experts[rest])
    assert torch.isnan(got.balance_loss) and not torch.isfinite(got.z_loss)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_ways_to_hand_logits_over(ops, dtype):
    """Rows that lie apart, that begin at odd places, that are columns; more dimensions; other streams."""
    T, E, k = 130, 64, 8
    logits, gen = make(T, E, DTYPES[dtype], seed=7)
    up = upstream(T, k, gen)
    wide = torch.full((T, E + 11), 9.0, dtype=logits.dtype, device="cuda")
    for first in (0, 3, 4):
        rows = wide[:, first:first + E]
        rows.copy_(logits)
        compare(ops, logits, k, **up, rows=rows, what="from column %d" % first)
    compare(ops, logits, k, **up, rows=logits.t().contiguous().t(), what="transposed")
    flat = ops.route(logits, k)
    mask = torch.rand(T, device="cuda", generator=gen) < 0.5
    cube = ops.route(logits.view(13, 10, E), k, mask=mask.view(13, 10))
    assert cube.weights.shape == (13, 10, k) and cube.counts.shape == (E,)
    want = ops.route(logits, k, mask=mask)
    assert torch.equal(cube.experts.view(T, k), want.experts) and torch.equal(cube.balance_loss, want.balance_loss)
    one = ops.route(logits[3], k)
    assert one.weights.shape == (k,) and torch.equal(one.experts, flat.experts[3])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = ops.route(logits, k)
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(flat, other):
        assert torch.equal(a, b)


@pytest.mark.parametrize("only", ["dw", "db", "dz"])
def test_one_gradient_alone(ops, only):
    logits, gen = make(500, 48, torch.float32, seed=8)
    up = upstream(500, 5, gen)
    for renormalize in (True, False):
        compare(ops, logits, 5, renormalize, **{only: up[only]}, what=only)
    # as a step of several uses would hand it over: strided
    wide = torch.empty(500, 10, device="cuda").normal_(generator=gen)
    compare(ops, logits, 5, dw=wide[:, ::2], what="strided gradient")


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_gradients_of_slots_without_a_winner_are_not_read(ops, dtype, renormalize):
    """Such a slot's weight is a constant, whatever arrives for it."""
    E, k = 20, 18
    logits, gen = make(40, E, DTYPES[dtype], seed=12)
    logits[::2, 10:] = float("-inf")  # slots from the tenth on have no winner
    logits[::8] = float("-inf")
    mask = torch.arange(40, device="cuda") % 5 != 0
    won = ops.route(logits, k, mask=mask).experts >= 0
    dw = torch.empty(40, k, device="cuda").normal_(generator=gen)
    grads = []
    for fill in (0.0, float("nan"), float("inf")):
        leaf = logits.clone().requires_grad_()
        got = ops.route(leaf, k, renormalize=renormalize, mask=mask)
        grads += torch.autograd.grad(got.weights, leaf, torch.where(won, dw, fill))
    assert torch.isfinite(grads[0]).all() and grads[0].any()
    for g in grads[1:]:
        assert torch.equal(g, grads[0])


def test_no_tokens(ops):
    leaf = torch.empty(0, 32, device="cuda", requires_grad=True)
    got = ops.route(leaf, 4)
    assert got.weights.shape == (0, 4) and not got.counts.any() and float(got.balance_loss.detach()) == 0 and float(got.z_loss.detach()) == 0
    grad, = torch.autograd.grad(got.balance_loss + got.z_loss, leaf)
    assert grad.shape == (0, 32)


def test_equal_calls_give_equal_bits(ops):
    logits, gen = make(20000, 128, torch.float32, seed=9)
    first = ops.route(logits, 8)
    for _ in range(3):
        for a, b in zip(first, ops.route(logits, 8)):
            assert torch.equal(a, b)


def test_counts_of_other_ranks_may_be_added(ops):
    """What is done to the returned counts does not reach the gradient."""
    logits, gen = make(300, 40, torch.float32, seed=11)
    leaf = logits.requires_grad_()
    got, want = ops.route(leaf, 4), ops.route(leaf, 4)
    got.counts.data.mul_(7)
    a, b = (torch.autograd.grad(r.balance_loss, leaf)[0] for r in (got, want))
    assert torch.equal(a, b)


def test_second_derivatives_are_refused(ops):
    logits, _ = make(8, 16, torch.float32)
    leaf = logits.requires_grad_()
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(ops.route(leaf, 2).z_loss, leaf, create_graph=True)


@pytest.mark.parametrize("T", [48, 5000])
def test_captured_step(ops, T):
    """A captured forward and backward pass, replayed with fresh logits, eager work and synchronisations between."""
    E, k = 128, 8
    logits, gen = make(T, E, torch.float32, seed=10)
    up = upstream(T, k, gen)
    still = logits.clone().requires_grad_()

    def step():
        r = ops.route(still, k)
        return r, torch.autograd.grad([r.weights, r.balance_loss, r.z_loss], [still], [up["dw"], up["db"], up["dz"]])[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, grad = step()
    for rep in range(4):
        fresh, _ = make(T, E, torch.float32, seed=20 + rep)
        with torch.no_grad():
            still.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        leaf = fresh.requires_grad_()
        e = ops.route(leaf, k)
        want = torch.autograd.grad([e.weights, e.balance_loss, e.z_loss], [leaf], [up["dw"], up["db"], up["dz"]])[0]
        for a, b in zip((*r, grad), (*e, want)):
            assert torch.equal(a, b), "replay %d" % rep
        del e, leaf


def test_a_step_beside_an_eager_graph_is_not_captured(ops):
    """The eager graph of the same leaf, reached through an operation, would end the process in the capture: refused instead."""
    leaf = torch.randn(64, 32, device="cuda", requires_grad=True)
    alive = ops.route(leaf * 2, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="still alive"):
            ops.route(leaf * 2, 4)
    assert torch.isfinite(alive.z_loss)
