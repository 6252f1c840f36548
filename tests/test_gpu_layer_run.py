"""The operators around a layer's blocks together with the blocks they stand around, as a model would use them: a training step
with a router's losses and a gated shared expert, and decoding and prompts of many requests on weights in 4 bits."""
import pytest
import torch

from flash_distributed_moe_amd import flashFfnOp as fops, flashLayerOp as ops
from tests import layer_case

pytestmark = pytest.mark.gpu


def normal(gen, sigma, *shape, mean=0.0, dtype=torch.float32):
    return torch.empty(shape, device="cuda").normal_(mean, sigma, generator=gen).to(dtype)


# ------------------------------------------------------------------ training
B, S, H, I, E, K = 3, 50, 256, 136, 24, 4


def layer(p, x, mask, norm, route, ffn, join):
    """One layer: the router looks at the normalised tokens, a shared expert with a gate a token is the branch."""
    h = norm(x, p["norm"])
    r = route(h @ p["router"].t(), K, mask)
    branch = ffn(h, p["w13"], p["w2"])
    gate = torch.sigmoid(h @ p["token_gate"].t()) + r[0].sum(-1, keepdim=True) * 0.1 + r[0][..., :1]
    y, out = join(x, branch, p["post"], gate, p["next"])
    return y, out, r


def plain_layer(p, x, mask):
    def norm(v, w):
        return v / ((v * v).mean(-1, keepdim=True) + 1e-6).sqrt() * w

    def route(logits, k, mask):
        prob = torch.softmax(logits, -1) * mask[..., None]
        top, at = torch.sort(logits, dim=-1, descending=True, stable=True)
        w = torch.gather(prob, -1, at[..., :k])
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        counts = torch.zeros(E, dtype=torch.float64, device=logits.device).scatter_add_(
            0, at[..., :k].reshape(-1), mask[..., None].expand(*mask.shape, k).reshape(-1).double())
        n = mask.sum()
        balance = E * (counts / counts.sum() * prob.reshape(-1, E).sum(0)).sum() / n
        return w, at[..., :k], counts, balance, ((torch.logsumexp(logits, -1) * mask) ** 2).sum() / n

    def ffn(v, w13, w2):
        g, u = (v @ w13.t()).chunk(2, -1)
        return (torch.nn.functional.silu(g) * u) @ w2.t()

    def join(v, branch, post, gate, nxt):
        y = 0.9 * v + 0.7 * gate * norm(branch, post)
        return y, norm(y, nxt)

    return layer(p, x, mask, norm, route, ffn, join)


def own_layer(p, x, mask):
    return layer(p, x, mask, ops.block_norm, lambda logits, k, m: ops.route(logits, k, mask=m), fops.gated_ffn,
                 lambda v, b, post, gate, nxt: ops.block_join(v, b, post, gate, nxt, residual_scale=0.9, branch_scale=0.7))


def training_case(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    p = dict(norm=normal(gen, 0.2, H, mean=1.0), router=normal(gen, H ** -0.5, E, H), w13=normal(gen, H ** -0.5, 2 * I, H),
             w2=normal(gen, I ** -0.5, H, I), token_gate=normal(gen, H ** -0.5, 1, H), post=normal(gen, 0.2, H, mean=1.0),
             next=normal(gen, 0.2, H, mean=1.0))
    x = normal(gen, 1.0, B, S, H)
    mask = torch.rand(B, S, device="cuda", generator=gen) < 0.8
    return p, x, mask, normal(gen, 1.0, B, S, H), normal(gen, 1.0, B, S, H)


def step(forward, p, x, mask, cy, ch):
    leaves = {**{k: t.detach().requires_grad_() for k, t in p.items()}, "x": x.detach().requires_grad_()}
    y, h, r = forward(leaves, leaves["x"], mask)
    loss = (y * cy).sum() + (h * ch).sum() + 50.0 * r[3] + 5.0 * r[4]
    grads = torch.autograd.grad(loss, list(leaves.values()))
    return dict(y=y.detach(), h=h.detach(), balance=r[3].detach(), zed=r[4].detach(), **{"d" + k: g for k, g in zip(leaves, grads)})


# Five operators after one another, each with sums of at most 272 products off by 2 * 272 steps of 2^-24 of their magnitudes, which with
# signs that cancel are up to sqrt(272) = 17 times the result's norm at worst and about 1 for the norms compared here; the
# gradients pass through as many again, and the norms' slopes are below 4.
TOLERANCE = 10 * 2 * 272 * 2.0 ** -24 * 4


def test_training_step():
    case = training_case(7)
    got = step(own_layer, *case)
    want = step(plain_layer, {k: t.double() for k, t in case[0].items()}, *(t if t.dtype == torch.bool else t.double() for t in case[1:]))
    for name, t in got.items():
        far = float((t.double() - want[name]).norm() / want[name].norm())
        assert far <= TOLERANCE, "%s: %.3g" % (name, far)


def test_captured_training_step():
    """Both passes of the whole layer in one graph, replayed on fresh tokens and weights."""
    p, x, mask, cy, ch = training_case(8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(own_layer, p, x, mask, cy, ch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        leaves = {**{k: t.detach().requires_grad_() for k, t in p.items()}, "x": x.detach().requires_grad_()}
        y, h, r = own_layer(leaves, leaves["x"], mask)
        grads = torch.autograd.grad([y, h, r[3], r[4]], list(leaves.values()), [cy, ch, torch.full_like(r[3].detach(), 50.0), torch.full_like(r[4].detach(), 5.0)])
    for rep in range(4):
        fp, fx, fmask, fcy, fch = training_case(30 + rep)
        for a, b in ((x, fx), (mask, fmask), (cy, fcy), (ch, fch)):
            a.copy_(b)
        for k, t in fp.items():
            p[k].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        fl = {**{k: t.detach().requires_grad_() for k, t in fp.items()}, "x": fx.detach().requires_grad_()}
        ey, eh, er = own_layer(fl, fl["x"], fmask)
        want = torch.autograd.grad([ey, eh, er[3], er[4]], list(fl.values()), [fcy, fch, torch.full_like(er[3].detach(), 50.0), torch.full_like(er[4].detach(), 5.0)])
        assert torch.equal(r[3].detach(), er[3].detach()) and torch.equal(r[1], er[1])
        for name, a, b in zip(fl, grads, want):
            far = float((a - b).norm() / b.norm())
            assert far <= TOLERANCE, "%s, replay %d: %.3g" % (name, rep, far)
        del fl, ey, eh, er, want


# ------------------------------------------------------------------ serving
def serving_case(T, seed, width=256, inner=192, adapters=5, rank=16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b = torch.bfloat16

    def low_rank(n, k):
        return fops.Adapters(normal(gen, k ** -0.5, adapters, rank, k, dtype=b), normal(gen, 0.3 * rank ** -0.5, adapters, n, rank, dtype=b),
                             0.5 + torch.rand(adapters, device="cuda", generator=gen))

    w = dict(norm=normal(gen, 0.2, width, mean=1.0, dtype=b), post=normal(gen, 0.2, width, mean=1.0, dtype=b),
             next=normal(gen, 0.2, width, mean=1.0, dtype=b), q13=fops.quantize_mxfp4(normal(gen, 0.05, 2 * inner, width)),
             q2=fops.quantize_mxfp4(normal(gen, 0.05, width, inner)), a13=low_rank(2 * inner, width), a2=low_rank(width, inner))
    x = normal(gen, 1.0, T, width, dtype=b)
    ids = torch.randint(-1, adapters, (T,), device="cuda", generator=gen, dtype=torch.int32)
    return w, x, ids


def serve(w, x, ids):
    h = ops.block_norm(x, w["norm"])
    g, u = fops.mxfp4_linear(h, w["q13"], w["a13"], ids).chunk(2, -1)
    inner = torch.nn.functional.silu(g) * u
    out = fops.mxfp4_linear(inner, w["q2"], w["a2"], ids)
    y, nxt = ops.block_join(x, out, w["post"], None, w["next"])
    return h, inner, out, y, nxt


@pytest.mark.parametrize("T", [1, 16, 300, 4100])
def test_serving_step(T):
    """Every operator's result from what the one before it gave."""
    w, x, ids = serving_case(T, 40 + T)
    with torch.no_grad():
        h, inner, out, y, nxt = serve(w, x, ids)
    layer_case.check(h, *layer_case.join(x, next_weight=w["norm"])["h"], "h")
    plain = fops.mxfp4_linear(inner, w["q2"])
    layer_case.check(out, *layer_case.adapters(plain, inner, *w["a2"], ids), "out")
    want = layer_case.join(x, out, w["post"], None, w["next"])
    layer_case.check(y, *want["y"], "y")
    layer_case.check(nxt, *want["h"], "next")


@pytest.mark.parametrize("T", [4, 300])
def test_captured_serving_step(T):
    w, x, ids = serving_case(T, 50)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            serve(w, x, ids)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = serve(w, x, ids)
        for rep in range(4):
            _, fx, fids = serving_case(T, 60 + rep)
            x.copy_(fx), ids.copy_(fids)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, serve(w, fx, fids)):
                assert torch.equal(a, b), "replay %d" % rep
