"""The operators around a layer's blocks where a workgroup takes rows again and again, under autograd's other ways of running
a graph, and beside the projection that they follow."""
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from flash_distributed_moe_amd import flashFfnOp as fops, flashLayerOp as ops
from tests import layer_case
from tests.test_gpu_layer_run import serving_case

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def normal(gen, sigma, *shape, mean=0.0, dtype=torch.float32):
    return torch.empty(shape, device="cuda").normal_(mean, sigma, generator=gen).to(dtype)


# ------------------------------------------------------------------ more rows than workgroups have at once
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("E,k,ragged", [(60, 4, 0), (60, 4, 3), (128, 8, 0), (200, 3, 0)])
def test_route_of_many_tokens(E, k, ragged, dtype):
    """Several trips of every loop over rows, forward and backward, with what was asked for ahead; whole and ragged rows."""
    T = 70001
    gen = torch.Generator(device="cuda").manual_seed(9000 + E)
    logits = normal(gen, 2.0, T, E, dtype=DTYPES[dtype])
    logits[torch.rand(T, E, device="cuda", generator=gen) < 0.05] = float("-inf")
    mask = torch.rand(T, device="cuda", generator=gen) < 0.9
    dw, db, dz = normal(gen, 1.0, T, k), torch.tensor(0.3, device="cuda"), torch.tensor(-0.2, device="cuda")
    rows = torch.zeros(T, E + ragged, dtype=logits.dtype, device="cuda")[:, :E]
    leaf = rows.copy_(logits).requires_grad_()
    want = layer_case.route(logits, k, True, mask, dw, db, dz)
    got = ops.route(leaf, k, mask=mask)
    assert torch.equal(got.experts.long(), want["experts"]) and torch.equal(got.counts.long(), want["counts"])
    grad, = torch.autograd.grad([got.weights, got.balance_loss, got.z_loss], leaf, [dw, db, dz])
    for name, t in (("weights", got.weights), ("balance_loss", got.balance_loss), ("z_loss", got.z_loss), ("dlogits", grad)):
        layer_case.check(t, *want[name], name)


@pytest.mark.parametrize("T,H,dtype", [(20000, 2048, "f32"), (9000, 4104, "bf16"), (9001, 2056, "f32")])
@pytest.mark.parametrize("what", ["norm", "post", "both", "neither"])
def test_norms_of_many_rows(T, H, dtype, what):
    """Several trips where several waves have a row, with one norm, two and none."""
    gen = torch.Generator(device="cuda").manual_seed(9100 + H)
    x, branch, dy, dh = (normal(gen, 1.0, T, H, dtype=DTYPES[dtype]) for _ in range(4))
    post, nxt = (normal(gen, 0.5, H, mean=1.0, dtype=DTYPES[dtype]) for _ in range(2))
    given = dict(x=x, next_weight=nxt) if what == "norm" else dict(x=x, branch=branch, **(dict(post=post) if what in ("post", "both") else {}),
                                                                    **(dict(next_weight=nxt) if what == "both" else {}))
    up = dict(dh=dh) if what == "norm" else dict(dy=dy, **(dict(dh=dh) if what == "both" else {}))
    want = layer_case.join(**given, **up)
    leaves = {name: t.detach().requires_grad_() for name, t in given.items()}
    if what == "norm":
        out = dict(h=ops.block_norm(leaves["x"], leaves["next_weight"]))
    else:
        out = ops.block_join(leaves["x"], leaves["branch"], leaves.get("post"), None, leaves.get("next_weight"))
        out = dict(zip("yh", out if what == "both" else (out,)))
    grads = torch.autograd.grad(list(out.values()), list(leaves.values()), [up["d" + name] for name in out])
    for name, t in {**out, **dict(zip(leaves, grads))}.items():
        layer_case.check(t, *want[name], "%s, %s" % (name, what))


# ------------------------------------------------------------------ beside the projection
@pytest.mark.parametrize("T", [1, 16, 300, 4100])
def test_the_first_projection_of_a_serving_step(T):
    """The gate's and up projection's adapters from the normalised rows, as a serving step calls them."""
    w, x, ids = serving_case(T, 140 + T)
    h = ops.block_norm(x, w["norm"])
    got = fops.mxfp4_linear(h, w["q13"], w["a13"], ids)
    layer_case.check(got, *layer_case.adapters(fops.mxfp4_linear(h, w["q13"]), h, *w["a13"], ids), "T=%d" % T)


# ------------------------------------------------------------------ autograd's other ways
def step(p):
    """Both nodes in one graph, with views and rows apart among what they keep."""
    h = ops.block_norm(p["x"], p["norm"])
    r = ops.route(h[:, :20] * p["router"], 4, mask=p["mask"])
    y, out = ops.block_join(p["x"], h * 0.5, p["post"], r.weights[..., :1], p["next"])
    return (y * y).sum() * 1e-3 + out.sum() * 1e-3 + r.balance_loss + r.z_loss


def parameters(seed, T=300, H=264):
    gen = torch.Generator(device="cuda").manual_seed(9200 + seed)
    p = dict(x=normal(gen, 1.0, T, H + 8)[:, :H], norm=normal(gen, 0.2, H, mean=1.0), router=normal(gen, 1.0, 20),
             post=normal(gen, 0.2, H, mean=1.0), next=normal(gen, 0.2, H, mean=1.0))
    p = {k: t.detach().requires_grad_() for k, t in p.items()}
    return {**p, "mask": torch.rand(T, device="cuda", generator=gen) < 0.8}


def gradients(loss, p):
    leaves = [t for t in p.values() if t.requires_grad]
    return [loss.detach(), *torch.autograd.grad(loss, leaves)]


def test_saved_tensors_on_the_host_and_checkpoints():
    p = parameters(0)
    want = gradients(step(p), p)
    with torch.autograd.graph.save_on_cpu():
        loss = step(p)
    ways = {"host": gradients(loss, p), "checkpoint": gradients(checkpoint(step, p, use_reentrant=False), p)}
    for name, got in ways.items():
        for a, b in zip(got, want):
            assert torch.equal(a, b), name


@pytest.mark.parametrize("transform", ["vmap", "grad", "jvp", "functionalize"])
def test_transforms_of_functions_are_refused(transform):
    """Their tensors stand for others, and have no memory to be read."""
    H = 64
    x, w, ids = torch.randn(3, 5, H, device="cuda"), torch.ones(H, device="cuda"), torch.zeros(3, 5, dtype=torch.int32, device="cuda")
    a = fops.Adapters(*(torch.zeros(s, device="cuda", dtype=torch.bfloat16) for s in ((1, 8, H), (1, H, 8))), torch.ones(1, device="cuda"))
    calls = [lambda v: ops.route(v, 2).z_loss, lambda v: ops.block_norm(v, w).sum(), lambda v: ops.block_join(v, v, w, None, w)[1].sum(),
             lambda v: ops.block_join(x[0] if transform == "vmap" else x, x[0] if transform == "vmap" else x, w, v, w)[1].sum(),
             lambda v: fops.add_adapters(v.bfloat16(), v.bfloat16(), a, ids[0] if transform == "vmap" else ids).float().sum()]
    for call in calls:
        with pytest.raises(RuntimeError):
            if transform == "vmap":
                torch.func.vmap(call)(x)
            elif transform == "grad":
                torch.func.grad(call)(x)
            elif transform == "jvp":
                torch.func.jvp(call, (x,), (x,))
            else:
                torch.func.functionalize(call)(x)


def test_several_threads_at_once():
    """Each on a stream of its own, forward and backward."""
    cases = [parameters(i, T=300 + 500 * i) for i in range(4)]
    want = [gradients(step(p), p) for p in cases]
    torch.cuda.synchronize()
    got, failed = [[] for _ in cases], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(8):
                    got[i].append(gradients(step(cases[i]), cases[i]))
            stream.synchronize()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for gs, w in zip(got, want):
        assert len(gs) == 8
        for g in gs:
            for a, b in zip(g, w):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    """The router's calls that overlap share nothing."""
    gen = torch.Generator(device="cuda").manual_seed(9300)
    cases = [normal(gen, 2.0, T, 128).requires_grad_() for T in (9000, 12000)]

    def run(leaf):
        r = ops.route(leaf, 8)
        return [*r, *torch.autograd.grad(r.balance_loss + r.z_loss, leaf)]

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    got = []
    for c in cases:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append([run(c) for _ in range(5)])
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for g in gs:
            assert all(torch.equal(a, b) for a, b in zip(g, w))
