"""What the operators around a layer's blocks refuse, and the sizes they report: before anything is enqueued, so without a GPU.
And the tests' own definitions, against differences."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

from flash_distributed_moe_amd import _lib, flashLayerOp as ops
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


def route(d=None, logits=0x1000, ld=16, mask=None, tokens=100, weights=0x2000, experts=0x3000, counts=0x4000, totals=0x5000, balance=0x6000,
          zed=0x7000, work=0x8000):
    return _lib.load().flashMoeRoute(ctypes.byref(d or route_desc()), logits, ld, mask, tokens, weights, experts, counts, totals, balance, zed,
                                     work, None)


def route_backward(d=None, logits=0x1000, ld=16, mask=None, tokens=100, experts=0x3000, counts=0x4000, totals=0x5000, dw=0x6000, db=0x7000,
                   dz=0x8000, out=0x9000, ldd=16):
    return _lib.load().flashMoeRouteBackward(ctypes.byref(d or route_desc()), logits, ld, mask, tokens, experts, counts, totals, dw, db, dz, out,
                                             ldd, None)


@pytest.mark.parametrize("kw", [dict(experts=0), dict(experts=257), dict(top_k=0), dict(top_k=17), dict(experts=64, top_k=33), dict(dtype=2)])
def test_bad_routers(kw, capfd):
    d = route_desc(**kw)
    n = ctypes.c_size_t(0)
    assert _lib.load().flashMoeRouteBytes(ctypes.byref(d), 4, ctypes.byref(n)) == BAD
    assert route(d=d) == BAD and route_backward(d=d) == BAD
    assert capfd.readouterr().out.count("[MOE ERROR:") == 3


@pytest.mark.parametrize("kw", [dict(logits=None), dict(logits=0x1002), dict(ld=15), dict(ld=(1 << 20) + 1), dict(tokens=-1), dict(tokens=(1 << 28) + 1),
                                dict(weights=None), dict(experts=None), dict(counts=None), dict(totals=0x5002), dict(balance=None), dict(zed=None),
                                dict(work=None), dict(work=0x8001)])
def test_route_refuses(kw, capfd):
    assert route(**kw) == BAD
    assert "[MOE ERROR:" in capfd.readouterr().out


@pytest.mark.parametrize("kw", [dict(logits=None), dict(ld=3), dict(out=None), dict(out=0x9001), dict(ldd=15), dict(experts=None), dict(counts=None),
                                dict(totals=None), dict(dw=0x6001), dict(dz=0x8002), dict(tokens=-1)])
def test_route_backward_refuses(kw, capfd):
    assert route_backward(**kw) == BAD
    assert "[MOE ERROR:" in capfd.readouterr().out


def test_route_workspace():
    def size(tokens):
        n = ctypes.c_size_t(0)
        assert _lib.load().flashMoeRouteBytes(ctypes.byref(route_desc(experts=256)), tokens, ctypes.byref(n)) == 0
        return n.value

    assert size(0) == size(1) == size(64) == 0
    for tokens in (65, 100, 4096, 4097, 1 << 28):
        rows = 16 if tokens <= 4096 else 64
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
