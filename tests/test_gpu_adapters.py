"""Adapters of many requests beside a projection against their definition in float64."""
import pytest
import torch

from tests import layer_case

pytestmark = pytest.mark.gpu

# rows, K, N, rank, adapters: one of everything, what is done row by row, in tiles of 16 and of 64 rows with every number of rank
# blocks and steps, k that ends inside a step, columns that end inside a unit, one row to a tile
SHAPES = [(1, 8, 8, 8, 1), (1, 4096, 1024, 16, 3), (3, 136, 72, 24, 2), (16, 2048, 520, 64, 5), (33, 1000, 4096, 128, 48), (64, 72, 200, 40, 1000),
          (333, 64, 264, 72, 60), (4096, 264, 72, 8, 3),
          (700, 8192, 4104, 24, 3), (1150, 4104, 4096, 8, 70), (610, 4096, 2056, 40, 7), (400, 4104, 2120, 128, 5), (1500, 4096, 4096, 16, 1000),
          (1000, 2048, 8200, 64, 2), (5001, 200, 1032, 48, 9), (4500, 1032, 136, 128, 100), (9000, 72, 2048, 56, 2), (4097, 8, 8, 8, 1),
          (6000, 136, 72, 16, 500), (4200, 520, 136, 32, 3)]
# (rows, K, N) at rank 16 of a few adapters: row by row, tiles of 16, tiles of 64
WAYS = [(7, 264, 136), (900, 2048, 4096), (4200, 264, 136)]


@pytest.fixture(scope="module")
def ops():
    from flash_distributed_moe_amd import flashFfnOp

    return flashFfnOp


def make(T, K, N, r, n, order="any", seed=0):
    gen = torch.Generator(device="cuda").manual_seed(6000 + seed)

    def normal(sigma, *shape):
        return torch.empty(shape, device="cuda").normal_(0.0, sigma, generator=gen).bfloat16()

    ids = torch.randint(-1, n, (T,), device="cuda", generator=gen, dtype=torch.int32)
    if order == "runs":
        ids = ids.sort().values
    return normal(1.0, T, N), normal(1.0, T, K), (normal(K ** -0.5, n, r, K), normal(r ** -0.5, n, N, r), torch.randn(n, device="cuda", generator=gen)), ids


def compare(ops, y, x, a, ids, got, what):
    layer_case.check(got, *layer_case.adapters(y, x, *a, ids), what)
    assert torch.equal(got[ids < 0], y[ids < 0]), what + ": rows without an adapter"


@pytest.mark.parametrize("order", ["any", "runs"])
@pytest.mark.parametrize("T,K,N,r,n", SHAPES)
def test_adapters(ops, T, K, N, r, n, order):
    y, x, a, ids = make(T, K, N, r, n, order)
    before = y.clone()
    got = ops.add_adapters(y, x, ops.Adapters(*a), ids)
    assert torch.equal(y, before) and got.shape == y.shape and got.dtype == torch.bfloat16
    compare(ops, y, x, a, ids, got, "%s" % ((T, K, N, r, n),))
    for _ in range(2):
        assert torch.equal(ops.add_adapters(y, x, ops.Adapters(*a), ids), got)
    assert ops.add_adapters(y, x, ops.Adapters(*a), ids, out=y) is y and torch.equal(y, got)


@pytest.mark.parametrize("T,K,N", WAYS + [(1, 264, 136)])
def test_no_row_one_row_and_all_rows_have_an_adapter(ops, T, K, N):
    y, x, a, ids = make(T, K, N, 16, 6, seed=1)
    for which in (torch.full_like(ids, -1), torch.full_like(ids, -2 ** 31), torch.full_like(ids, 5),
                  torch.where(torch.arange(T, device="cuda") == T // 2, 3, -7).int()):
        compare(ops, y, x, a, which, ops.add_adapters(y, x, ops.Adapters(*a), which), "T=%d" % T)


@pytest.mark.parametrize("T,K,N", WAYS)
def test_adapters_that_are_not_there(ops, T, K, N):
    """Their rows become NaN, and nobody else's."""
    y, x, a, ids = make(T, K, N, 16, 4, seed=2)
    bad = torch.arange(T, device="cuda") % 3 == 1
    wrong = torch.where(bad, torch.where(torch.arange(T, device="cuda") % 2 == 0, 4, 2 ** 31 - 1).int(), ids)
    got = ops.add_adapters(y, x, ops.Adapters(*a), wrong)
    assert torch.isnan(got[bad]).all()
    assert torch.equal(got[~bad], ops.add_adapters(y, x, ops.Adapters(*a), ids)[~bad])


@pytest.mark.parametrize("T,K,N", WAYS)
def test_rows_that_are_not_finite(ops, T, K, N):
    """A row's infinities and NaN stay its own, whoever shares its tile; so do an adapter's."""
    y, x, a, ids = make(T, K, N, 16, 3, "runs", seed=3)
    want = ops.add_adapters(y, x, ops.Adapters(*a), ids)
    bad = x.clone()
    bad[T // 2, 5], bad[T - 1, 9] = float("nan"), float("inf")
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[[T // 2, T - 1]] = False
    got = ops.add_adapters(y, bad, ops.Adapters(*a), torch.where(rest, ids, 1))
    assert torch.equal(got[rest], want[rest]) and torch.isnan(got[T // 2]).all() and not torch.isfinite(got[T - 1]).any()
    up = a[1].clone()
    up[2] = float("nan")
    got = ops.add_adapters(y, x, ops.Adapters(a[0], up, a[2]), ids)
    assert torch.equal(got[ids != 2], want[ids != 2])


@pytest.mark.parametrize("T,K,N", [(12, 264, 136)] + WAYS[1:])
def test_ways_to_hand_rows_over(ops, T, K, N):
    y, x, a, ids = make(T, K, N, 16, 6, seed=4)
    want = ops.add_adapters(y, x, ops.Adapters(*a), ids)
    wide = torch.zeros(T, K + N + 16, dtype=torch.bfloat16, device="cuda")
    wide[:, :K], wide[:, K:K + N] = x, y
    got = ops.add_adapters(wide[:, K:K + N], wide[:, :K], ops.Adapters(*a), ids)
    assert torch.equal(got, want)
    out = wide[:, K:K + N]
    assert torch.equal(ops.add_adapters(y, x, ops.Adapters(*a), ids, out=out), want) and not wide[:, K + N:].any() and torch.equal(wide[:, :K], x)
    wide[:, K:K + N] = y
    ops.add_adapters(out, wide[:, :K], ops.Adapters(*a), ids, out=out)
    assert torch.equal(wide[:, K:K + N], want) and not wide[:, K + N:].any() and torch.equal(wide[:, :K], x)
    odd = torch.zeros(T, K + 3, dtype=torch.bfloat16, device="cuda")
    odd[:, 3:] = x
    assert torch.equal(ops.add_adapters(y, odd[:, 3:], ops.Adapters(*a), ids), want)
    twice = torch.stack((ids, ids), 1)[:, 0]
    cube = ops.add_adapters(y.view(2, -1, N), x.view(2, -1, K), ops.Adapters(*a), twice.view(2, -1))
    assert torch.equal(cube.view(T, N), want)
    # columns side by side of one buffer with more dimensions, and columns that overlap
    both = torch.zeros(2, T // 2, K + N, dtype=torch.bfloat16, device="cuda")
    both[..., :K], both[..., K:] = x.view(2, -1, K), y.view(2, -1, N)
    ops.add_adapters(both[..., K:], both[..., :K], ops.Adapters(*a), ids.view(2, -1), out=both[..., K:])
    assert torch.equal(both[..., K:].reshape(T, N), want) and torch.equal(both[..., :K].reshape(T, K), x)
    with pytest.raises(RuntimeError, match="apart from x"):
        ops.add_adapters(y.view(2, -1, N), both[..., :K], ops.Adapters(*a), ids.view(2, -1), out=both[..., K - 8:K - 8 + N])
    one = ops.add_adapters(y[1], x[1], ops.Adapters(*a), ids[1])
    layer_case.check(one[None], *(v[1:2] for v in layer_case.adapters(y, x, *a, ids)), "one row")


def test_refusals(ops):
    y, x, a, ids = make(4, 64, 32, 8, 2, seed=5)
    ad = ops.Adapters(*a)
    wide = torch.zeros(4, 40, dtype=torch.bfloat16, device="cuda")
    calls = {
        "bfloat16": lambda: ops.add_adapters(y.float(), x, ad, ids), "int32": lambda: ops.add_adapters(y, x, ad, ids.long()),
        "leading": lambda: ops.add_adapters(y, x, ad, ids[:3]), r"\[..., K\]": lambda: ops.add_adapters(y, x[:, :56], ad, ids),
        r"\[..., N\]": lambda: ops.add_adapters(y[:, :24], x, ad, ids), "rank": lambda: ops.add_adapters(y, x, ops.Adapters(a[0][:, :4].contiguous(), a[1][..., :4].contiguous(), a[2]), ids),
        "float32": lambda: ops.add_adapters(y, x, ops.Adapters(a[0], a[1], a[2].bfloat16()), ids),
        "contiguous": lambda: ops.add_adapters(y, x, ops.Adapters(a[0].transpose(0, 1).contiguous().transpose(0, 1), a[1], a[2]), ids),
        "out must be y or apart": lambda: ops.add_adapters(wide[:, :32], x, ad, ids, out=wide[:, 8:]),
        "out must have rows": lambda: ops.add_adapters(y, x, ad, ids, out=torch.zeros(32, 4, dtype=torch.bfloat16, device="cuda").t()),
        "out must have y's shape": lambda: ops.add_adapters(y, x, ad, ids, out=y[:3]),
        "no backward pass": lambda: ops.add_adapters(y, x.requires_grad_(), ad, ids),
    }
    for message, call in calls.items():
        with pytest.raises(RuntimeError, match=message):
            call()
    with torch.no_grad():
        ops.add_adapters(y, x, ad, ids)
    empty = ops.add_adapters(y[:0], x.detach()[:0], ad, ids[:0])
    assert empty.shape == (0, 32)


@pytest.mark.parametrize("T", [3, 40, 300])
def test_beside_a_projection_in_4_bits(ops, T):
    """`mxfp4_linear` with adapters: the projection's rounded result and what the adapters add to it."""
    y, x, a, ids = make(T, 256, 192, 16, 5, seed=6)
    w = ops.quantize_mxfp4(torch.randn(192, 256, device="cuda") * 0.05)
    plain = ops.mxfp4_linear(x, w)
    got = ops.mxfp4_linear(x, w, ops.Adapters(*a), ids)
    assert torch.equal(got, ops.add_adapters(plain, x, ops.Adapters(*a), ids))
    layer_case.check(got, *layer_case.adapters(plain, x, *a, ids), "T=%d" % T)
    for bad in (lambda: ops.mxfp4_linear(x, w, ops.Adapters(*a)), lambda: ops.mxfp4_linear(x, w, ids=ids),
                lambda: ops.mxfp4_linear(ops.quantize_mxfp4(x), w, ops.Adapters(*a), ids)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("T,K,N", WAYS)
def test_captured(ops, T, K, N):
    y, x, a, ids = make(T, K, N, 16, 6, seed=7)
    ad = ops.Adapters(*a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.add_adapters(y, x, ad, ids)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.add_adapters(y, x, ad, ids)
    for rep in range(4):
        fresh = make(T, K, N, 16, 6, order=("any", "runs")[rep % 2], seed=20 + rep)
        y.copy_(fresh[0]), x.copy_(fresh[1]), ids.copy_(fresh[3])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ops.add_adapters(fresh[0], fresh[1], ad, fresh[3]), got), "replay %d" % rep


def test_two_streams_at_once(ops):
    cases = [make(4300 if i else 900, 2048, 4096, 24, 6, seed=30 + i) for i in range(2)]
    want = [ops.add_adapters(y, x, ops.Adapters(*a), ids) for y, x, a, ids in cases]
    torch.cuda.synchronize()
    got = []
    for s, (y, x, a, ids) in zip([torch.cuda.Stream() for _ in cases], cases):
        with torch.cuda.stream(s):
            got.append([ops.add_adapters(y, x, ops.Adapters(*a), ids) for _ in range(5)])
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(g, w) for g in gs)


def test_results_in_place_are_noticed_by_autograd(ops):
    """A product that another operator saved for its backward pass, and that out= wrote over, is not differentiated."""
    y, x, a, ids = make(8, 64, 32, 8, 2, seed=8)
    leaf = y.float().requires_grad_()
    saved = torch.exp(leaf)
    other = saved.detach().bfloat16()
    z = torch.exp(y.detach().requires_grad_())
    with torch.no_grad():
        ops.add_adapters(other, x, ops.Adapters(*a), ids, out=other)
        ops.add_adapters(z, x, ops.Adapters(*a), ids, out=z)
    saved.sum().backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    with torch.inference_mode():
        w = y.clone()
        ops.add_adapters(w, x, ops.Adapters(*a), ids, out=w)
