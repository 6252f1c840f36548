"""What the operators around a layer's blocks refuse, and the sizes they report: before anything is enqueued, so without a GPU.
And the tests' own definitions, against differences."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

from flash_distributed_moe_amd import _lib, flashFfnOp as fops, flashLayerOp as ops
from tests import layer_case

BAD = _lib.HIP_ERROR_INVALID_VALUE


def differences(f, x, dx=1e-5):
    """The gradient of the scalar f at x by central differences, in float64."""
    out = torch.zeros_like(x)
    for i in range(x.numel()):
        step = torch.zeros_like(x).reshape(-1)
        step[i] = dx
        step = step.reshape(x.shape)
        out.view(-1)[i] = (f(x + step) - f(x - step)) / (2 * dx)
    return out


# ------------------------------------------------------------------ the router's choice
def route_desc(**kw):
    d = _lib.RouteDesc(16, 4, _lib.F32, 1)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def route(d=None, logits=0x1000, ld=16, mask=None, tokens=100, weights=0x2000, experts=0x3000, counts=0x4000, balance=0x5000, zed=0x6000,
          kept=0x7000, work=0x8000):
    return _lib.load().flashMoeRoute(ctypes.byref(d or route_desc()), logits, ld, mask, tokens, weights, experts, counts, balance, zed, kept,
                                     work, None)


def route_backward(d=None, logits=0x1000, ld=16, mask=None, tokens=100, weights=0x2000, experts=0x3000, kept=0x4000, dw=0x6000, db=0x7000,
                   dz=0x8000, out=0x9000, ldd=16):
    return _lib.load().flashMoeRouteBackward(ctypes.byref(d or route_desc()), logits, ld, mask, tokens, weights, experts, kept, dw, db, dz, out,
                                             ldd, None)


@pytest.mark.parametrize("kw", [dict(experts=0), dict(experts=257), dict(top_k=0), dict(top_k=17), dict(experts=64, top_k=33), dict(dtype=2)])
def test_bad_routers(kw, capfd):
    d = route_desc(**kw)
    n = ctypes.c_size_t(0)
    assert _lib.load().flashMoeRouteBytes(ctypes.byref(d), 4, ctypes.byref(n)) == BAD
    assert route(d=d) == BAD and route_backward(d=d) == BAD
    assert capfd.readouterr().out.count("[MOE ERROR:") == 3


@pytest.mark.parametrize("kw", [dict(logits=None), dict(logits=0x1002), dict(ld=15), dict(ld=(1 << 20) + 1), dict(tokens=-1), dict(tokens=(1 << 28) + 1),
                                dict(weights=None), dict(experts=None), dict(counts=None), dict(kept=0x5002), dict(balance=None), dict(zed=None),
                                dict(work=None), dict(work=0x8001)])
def test_route_refuses(kw, capfd):
    assert route(**kw) == BAD
    assert "[MOE ERROR:" in capfd.readouterr().out


@pytest.mark.parametrize("kw", [dict(logits=None), dict(ld=3), dict(out=None), dict(out=0x9001), dict(ldd=15), dict(weights=None), dict(experts=None), dict(kept=None),
                                dict(kept=0x4002), dict(dw=0x6001), dict(dz=0x8002), dict(tokens=-1)])
def test_route_backward_refuses(kw, capfd):
    assert route_backward(**kw) == BAD
    assert "[MOE ERROR:" in capfd.readouterr().out


def test_route_workspace():
    def size(tokens):
        n = ctypes.c_size_t(0)
        assert _lib.load().flashMoeRouteBytes(ctypes.byref(route_desc(experts=256)), tokens, ctypes.byref(n)) == 0
        return n.value

    assert size(0) == size(1) == size(64) == 0
    for tokens in (65, 100, 4096, 6000, 6001, 1 << 28):
        rows = 16 if tokens <= 6000 else 64
        assert size(tokens) == min(256, -(-tokens // rows)) * 2 * 257 * 4
    assert _lib.load().flashMoeRouteBytes(ctypes.byref(route_desc()), 1, None) == BAD
    assert route_backward(tokens=0, logits=None, out=None) == 0


@pytest.mark.parametrize("call,message", [
    (lambda x: ops.route(x, 2), "CUDA tensor"), (lambda x: ops.route(None, 2), "tensor"), (lambda x: ops.route(x, "2"), "whole number"),
    (lambda x: ops.route(x, 2, mask=3), "mask"), (lambda x: ops.route([1.0], 1), "tensor"), (lambda x: ops.route(x.requires_grad_(), 2), "CUDA tensor"),
])
def test_route_of_other_arguments(call, message):
    with pytest.raises(RuntimeError, match=message):
        call(torch.zeros(3, 8))


def test_route_refuses_tangents():
    with fwd.dual_level():
        x = fwd.make_dual(torch.zeros(2, 8), torch.ones(2, 8))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.route(x, 2)


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_definition(renormalize):
    """The restatement's gradient against differences of its outputs, with padding and experts that are none."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(6, 9, generator=gen, dtype=torch.float64)
    x[1, 3:5] = float("-inf")
    x[2] = float("-inf")
    mask = torch.tensor([True, True, True, False, True, True])
    dw, db, dz = torch.randn(6, 3, generator=gen, dtype=torch.float64), torch.tensor(0.7), torch.tensor(0.4)
    layer_case.HALF.setdefault(torch.float64, 0.0)
    want = layer_case.route(x, 3, renormalize, mask, dw, db, dz)["dlogits"][0]

    def loss(v):
        r = layer_case.route(v, 3, renormalize, mask)
        return float((r["weights"][0] * dw).sum() + db * r["balance_loss"][0] + dz * r["z_loss"][0])

    got = differences(loss, x).nan_to_num(0.0)
    assert torch.allclose(want, got, rtol=0, atol=1e-8)
    # and the choice: the first of equals
    r = layer_case.route(torch.tensor([[1.0, 2.0, 2.0, 0.0], [0.0, 0.0, 0.0, 0.0]]), 3, renormalize)
    assert r["experts"].tolist() == [[1, 2, 0], [0, 1, 2]] and r["counts"].tolist() == [2, 2, 2, 0]


# ------------------------------------------------------------------ the norms around a block
def norm_desc(**kw):
    d = _lib.NormDesc(64, _lib.BF16, _lib.GATE_CHANNEL, 1, 1e-6, 1.0, 1.0, 0x1000, 0x2000, 0x3000)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def norm(d=None, x=0x10000, ldx=64, branch=0x20000, ldb=64, tokens=6, y=0x30000, h=0x40000, kept=0x50000):
    return _lib.load().flashMoeBlockNorm(ctypes.byref(d or norm_desc()), x, ldx, branch, ldb, tokens, y, h, kept, None)


def norm_backward(d=None, x=0x10000, ldx=64, branch=0x20000, ldb=64, dy=0x30000, lddy=64, dh=0x40000, lddh=64, tokens=6, kept=0x50000,
                  work=0x60000, dx=0x70000, dbranch=0x80000, dpost=0x90000, dgate=0xA0000, dnext=0xB0000):
    return _lib.load().flashMoeBlockNormBackward(ctypes.byref(d or norm_desc()), x, ldx, branch, ldb, dy, lddy, dh, lddh, tokens, kept, work, dx,
                                                 dbranch, dpost, dgate, dnext, None)


@pytest.mark.parametrize("kw", [dict(hidden=0), dict(hidden=60), dict(hidden=8200), dict(dtype=2), dict(gate=5), dict(gate=-1), dict(gate=2, shared=4),
                                dict(gate=2, shared=0), dict(eps=-1.0), dict(eps=float("nan")), dict(gate_values=None), dict(gate=0),
                                dict(gate_values=0x2008), dict(gate=3, gate_values=0x2001), dict(post_weight=0x1002), dict(next_weight=0x3008)])
def test_bad_norms(kw, capfd):
    assert norm(d=norm_desc(**kw)) == BAD and norm_backward(d=norm_desc(**kw)) == BAD
    assert _lib.load().flashMoeBlockNormBytes(ctypes.byref(norm_desc(**kw)), 6, ctypes.byref(ctypes.c_size_t(0))) == BAD
    assert capfd.readouterr().out.count("[MOE ERROR:") == 3


ALONE = dict(post_weight=None, gate=0, gate_values=None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(x=0x10008), dict(ldx=56), dict(ldx=68), dict(ldx=(1 << 20) + 8), dict(ldb=60), dict(branch=0x20002),
                                dict(tokens=-1), dict(tokens=(1 << 30) + 1), dict(y=None), dict(y=0x30004), dict(h=None), dict(kept=0x50002),
                                dict(branch=None), dict(branch=None, d=norm_desc(**ALONE)),
                                dict(branch=None, y=None, d=norm_desc(**ALONE, next_weight=None))])
def test_norm_refuses(kw, capfd):
    assert norm(**kw) == BAD
    assert "[MOE ERROR:" in capfd.readouterr().out


@pytest.mark.parametrize("kw", [dict(x=None), dict(ldx=60), dict(branch=None), dict(ldb=8), dict(dy=0x30002), dict(lddy=60), dict(lddh=72 + 4),
                                dict(kept=None), dict(work=None), dict(dx=0x70002), dict(dbranch=0x80008), dict(dpost=0x90001),
                                dict(d=norm_desc(post_weight=None)), dict(d=norm_desc(gate=0, gate_values=None)), dict(d=norm_desc(next_weight=None)),
                                dict(d=norm_desc(gate=4), dgate=0xA0008), dict(tokens=-1)])
def test_norm_backward_refuses(kw, capfd):
    assert norm_backward(**kw) == BAD
    assert "[MOE ERROR:" in capfd.readouterr().out


def test_no_tokens_need_no_rows():
    assert norm(tokens=0, x=None, branch=None, y=None, h=None, kept=None) == 0
    assert norm_backward(tokens=0, x=None, branch=None, dy=None, dh=None, kept=None, work=None, dx=None, dbranch=None, dpost=None, dgate=None,
                         dnext=None) == 0


def test_norm_workspace():
    """Column sums of at most about a thousand workgroups, whatever the groups."""
    def size(tokens, **kw):
        n = ctypes.c_size_t(0)
        assert _lib.load().flashMoeBlockNormBytes(ctypes.byref(norm_desc(**kw)), tokens, ctypes.byref(n)) == 0
        return n.value

    for tokens in (0, 1, 1000, 1 << 20, 1 << 30):
        for hidden in (8, 1024, 8192):
            assert 0 < size(tokens, hidden=hidden) <= 2 * 512 * hidden * 4
    for count, shared in ((1, 7), (3, 5), (700, 3), (2, 100000), (513, 513), (1 << 20, 1), (1 << 10, 1 << 20)):
        assert 0 < size(count * shared, gate=2, shared=shared) <= 3 * 1100 * 64 * 4


@pytest.mark.parametrize("call,message", [
    (lambda x, w: ops.block_norm(x, w), "CUDA tensor"), (lambda x, w: ops.block_norm(x, None), "must be tensors"),
    (lambda x, w: ops.block_norm(None, w), "must be tensors"), (lambda x, w: ops.block_norm(x, w, eps="1"), "eps a number"),
    (lambda x, w: ops.block_join(x, None), "must be tensors"), (lambda x, w: ops.block_join(x, x, gate=1.0), "gate"),
    (lambda x, w: ops.block_join(x, x, w, None, w), "CUDA tensor"), (lambda x, w: ops.block_join(x.requires_grad_(), x), "CUDA tensor"),
    (lambda x, w: ops.block_join(x, x, residual_scale=w), "numbers"),
])
def test_norms_of_other_arguments(call, message):
    with pytest.raises(RuntimeError, match=message):
        call(torch.zeros(3, 8), torch.ones(8))


@pytest.mark.parametrize("which", range(5))
def test_norms_refuse_tangents(which):
    args = [torch.zeros(2, 8), torch.zeros(2, 8), torch.ones(8), torch.ones(8), torch.ones(8)]
    with fwd.dual_level():
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.block_join(*args)


@pytest.mark.parametrize("gate", [None, (8,), (2, 1, 8), (2, 3, 1), (2, 3, 8)])
@pytest.mark.parametrize("post,nxt", [(True, True), (False, True), (True, False)])
def test_join_definition(gate, post, nxt):
    """The restatement's gradients against differences, and against autograd."""
    gen = torch.Generator().manual_seed(4)
    draw = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    layer_case.HALF.setdefault(torch.float64, 0.0)
    given = dict(x=draw(2, 3, 8), branch=draw(2, 3, 8), post=draw(8) if post else None, gate=draw(*gate) if gate else None,
                 next_weight=draw(8) if nxt else None)
    dy, dh = draw(2, 3, 8), draw(2, 3, 8) if nxt else None
    more = dict(alpha=0.7, beta=1.3, eps=1e-3)
    want = layer_case.join(**given, **more, dy=dy, dh=dh)
    for name, t in given.items():
        if t is not None:
            def loss(v):
                r = layer_case.join(**{**given, name: v}, **more)
                return float((r["y"][0] * dy).sum() + ((r["h"][0] * dh).sum() if nxt else 0))
            assert torch.allclose(want[name][0], differences(loss, t), rtol=0, atol=1e-7), name
    alone = layer_case.join(given["x"], next_weight=draw(8), eps=0.0, dh=dy)
    assert torch.allclose((alone["x"][0] * given["x"]).sum(-1), torch.zeros(2, 3, dtype=torch.float64), atol=1e-12)  # a norm has no slope along itself


# ------------------------------------------------------------------ adapters beside a projection
def adapter_desc(**kw):
    d = _lib.AdapterDesc(4, 16, 64, 128, 0x1000, 0x2000, 0x3000)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def add(d=None, x=0x10000, ldx=128, y=0x20000, ldy=64, ids=0x30000, rows=5, out=0x40000, ldo=64, work=0x50000):
    return _lib.load().flashMoeAdapterAdd(ctypes.byref(d or adapter_desc()), x, ldx, y, ldy, ids, rows, out, ldo, work, None)


def adapter_size(rows, **kw):
    n = ctypes.c_size_t(0)
    rc = _lib.load().flashMoeAdapterBytes(ctypes.byref(adapter_desc(**kw)), rows, ctypes.byref(n))
    return rc, n.value


@pytest.mark.parametrize("kw", [dict(adapters=0), dict(adapters=1001), dict(rank=0), dict(rank=12), dict(rank=136), dict(n=0), dict(n=60), dict(k=4),
                                dict(n=(1 << 20) + 8)])
def test_bad_adapters(kw, capfd):
    assert add(d=adapter_desc(**kw)) == BAD and adapter_size(5, **kw)[0] == BAD
    assert capfd.readouterr().out.count("[MOE ERROR:") == 2


@pytest.mark.parametrize("kw", [dict(x=None), dict(x=0x10008), dict(ldx=120), dict(ldx=132), dict(y=None), dict(ldy=56), dict(out=None), dict(out=0x40004),
                                dict(ldo=68), dict(ldo=(1 << 20) + 8), dict(out=0x20000, ldo=72), dict(ids=None), dict(ids=0x30002), dict(rows=-1),
                                dict(rows=(1 << 26) + 1), dict(work=None), dict(work=0x50008), dict(d=adapter_desc(down=None)),
                                dict(d=adapter_desc(up=0x2008)), dict(d=adapter_desc(scales=None))])
def test_adapters_refuse(kw, capfd):
    assert add(**kw) == BAD
    assert "[MOE ERROR:" in capfd.readouterr().out


def test_adapter_workspace():
    assert adapter_size(0) == (0, 0) and add(rows=0, x=None, y=None, out=None, ids=None, work=None) == 0
    assert 5 * 16 * 4 <= adapter_size(5)[1] < 5 * 16 * 4 + 256
    # row by row: u alone
    assert 700 * 16 * 4 <= adapter_size(700, n=2048, k=4096)[1] < 700 * 16 * 4 + 256
    for rows, adapters in ((900, 4), (900, 1000), (2000, 4), (4097, 1000), (100000, 1000), (1 << 26, 1000)):
        rc, size = adapter_size(rows, adapters=adapters, n=2048, k=4096)
        tall = rows >= 1195 and rows >= 12 * adapters
        tiles = -(-rows // (64 if tall else 16)) + min(rows, adapters + 2)
        # u at least once, the order of the rows, and 16 bytes a tile and one more
        assert rc == 0 and rows * 16 * 4 + rows * 4 + (tiles + 1) * 16 <= size < rows * 16 * 4 * 8 + rows * 4 + (tiles + 1) * 16 + 1024


@pytest.mark.parametrize("call,message", [
    (lambda y, x, a, i: fops.add_adapters(y, x, a, i), "CUDA tensor"), (lambda y, x, a, i: fops.add_adapters(y, x, None, i), "must be tensors"),
    (lambda y, x, a, i: fops.add_adapters(None, x, a, i), "must be tensors"), (lambda y, x, a, i: fops.add_adapters(y, x, a, 3), "must be tensors"),
    (lambda y, x, a, i: fops.add_adapters(y, x, a, i, out=1), "must be tensors"),
    (lambda y, x, a, i: fops.add_adapters(y, x.requires_grad_(), a, i), "no backward pass"),
    (lambda y, x, a, i: fops.mxfp4_linear(x, None, a), "belong together"),
])
def test_adapters_of_other_arguments(call, message):
    b = torch.bfloat16
    a = fops.Adapters(torch.zeros(2, 8, 16, dtype=b), torch.zeros(2, 24, 8, dtype=b), torch.zeros(2))
    with pytest.raises(RuntimeError, match=message):
        call(torch.zeros(3, 24, dtype=b), torch.zeros(3, 16, dtype=b), a, torch.zeros(3, dtype=torch.int32))


def test_adapters_refuse_tangents():
    b = torch.bfloat16
    a = fops.Adapters(torch.zeros(2, 8, 16, dtype=b), torch.zeros(2, 24, 8, dtype=b), torch.zeros(2))
    with fwd.dual_level():
        x = fwd.make_dual(torch.zeros(3, 16, dtype=b), torch.ones(3, 16, dtype=b))
        with pytest.raises(RuntimeError, match="forward-mode"):
            fops.add_adapters(torch.zeros(3, 24, dtype=b), x, a, torch.zeros(3, dtype=torch.int32))
