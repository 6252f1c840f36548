"""The C entries of the operators around a layer's blocks on device memory, in the forms that the Python surface does not hand over."""
import ctypes

import pytest
import torch

from flash_distributed_moe_amd import _lib
from tests import layer_case

pytestmark = pytest.mark.gpu


def at(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def memory(bytes_):
    return torch.empty(max(1, bytes_), dtype=torch.uint8, device="cuda")


def size(f, desc, tokens):
    n = ctypes.c_size_t(0)
    assert f(ctypes.byref(desc), tokens, ctypes.byref(n)) == 0
    return n.value


CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


@pytest.mark.parametrize("dtype", sorted(CODE, key=str))
@pytest.mark.parametrize("residual,branch_scale", [(0.0, 0.0), (0.8, 1.0), (1.0, 0.5), (-2.0, 1.0)])
@pytest.mark.parametrize("T,H,gradients", [(5, 264, "h"), (700, 2048, "hy"), (33, 4104, "hy")])
def test_a_norm_without_a_branch_has_no_scales(T, H, gradients, residual, branch_scale, dtype):
    """y = x then, forward and backward, whatever the description's scales are."""
    lib = _lib.load()
    gen = torch.Generator(device="cuda").manual_seed(7000 + T)
    x, w, dh, dy = (torch.empty(s, device="cuda").normal_(generator=gen).to(dtype) for s in ((T, H), (H,), (T, H), (T, H)))
    dy = dy if "y" in gradients else None
    d = _lib.NormDesc(H, CODE[dtype], _lib.GATE_NONE, 0, 1e-5, residual, branch_scale, None, None, at(w))
    h, kept = torch.empty_like(x), torch.empty(2, T, device="cuda")
    assert lib.flashMoeBlockNorm(ctypes.byref(d), at(x), H, None, 0, T, None, at(h), at(kept), stream()) == 0
    dx, dw, work = torch.empty_like(x), torch.empty_like(w), memory(size(lib.flashMoeBlockNormBytes, d, T))
    assert lib.flashMoeBlockNormBackward(ctypes.byref(d), at(x), H, None, 0, at(dy), H, at(dh), H, T, at(kept), at(work), at(dx), None, None,
                                         None, at(dw), stream()) == 0
    want = layer_case.join(x, next_weight=w, eps=1e-5, dy=dy, dh=dh)
    for name, t in (("h", h), ("x", dx), ("next_weight", dw)):
        layer_case.check(t, *want[name], name)


@pytest.mark.parametrize("dtype", sorted(CODE, key=str))
@pytest.mark.parametrize("kind", ["none", "group", "token"])
def test_join(kind, dtype):
    """Rows apart on every side, a gate of tokens that begins on no 16 bytes, and the whole set of gradients."""
    lib = _lib.load()
    T, H, shared, ld = 60, 520, 12, 536
    gen = torch.Generator(device="cuda").manual_seed(7100)
    x, branch, dy, dh = (torch.empty(T, ld, device="cuda").normal_(generator=gen).to(dtype) for _ in range(4))
    post, nxt = (torch.empty(H, device="cuda").normal_(1.0, 0.5, generator=gen).to(dtype) for _ in range(2))
    shape = dict(none=None, group=(T // shared, H), token=(T,))[kind]
    values = None if shape is None else torch.empty(1 + shape[0] * (1 if len(shape) == 1 else H), device="cuda").normal_(generator=gen).to(dtype)
    gate = None if shape is None else (values[1:] if kind == "token" else values[:-1]).view(shape)
    d = _lib.NormDesc(H, CODE[dtype], dict(none=_lib.GATE_NONE, group=_lib.GATE_GROUP, token=_lib.GATE_TOKEN)[kind], shared, 1e-6, 0.75, 1.5,
                      at(post), at(gate), at(nxt))
    y, h = (torch.empty(T, H, dtype=dtype, device="cuda") for _ in range(2))
    kept, work = torch.empty(2, T, device="cuda"), memory(size(lib.flashMoeBlockNormBytes, d, T))
    assert lib.flashMoeBlockNorm(ctypes.byref(d), at(x), ld, at(branch), ld, T, at(y), at(h), at(kept), stream()) == 0
    dx, dbranch, dpost, dnext = (torch.empty_like(t) for t in (y, y, post, nxt))
    dgate = None if gate is None else torch.empty_like(gate)
    assert lib.flashMoeBlockNormBackward(ctypes.byref(d), at(x), ld, at(branch), ld, at(dy), ld, at(dh), ld, T, at(kept), at(work), at(dx),
                                         at(dbranch), at(dpost), at(dgate), at(dnext), stream()) == 0
    groups = T // shared
    cube = lambda t: t[:, :H].view(groups, shared, H) if t.dim() == 2 else t  # noqa: E731
    given = None if gate is None else gate.view(groups, 1, H) if kind == "group" else gate.view(groups, shared, 1)
    want = layer_case.join(cube(x), cube(branch), post, given, nxt, 0.75, 1.5, dy=cube(dy), dh=cube(dh))
    got = dict(y=y, h=h, x=dx, branch=dbranch, post=dpost, next_weight=dnext, **({} if gate is None else {"gate": dgate}))
    assert set(got) == set(want)
    for name, t in got.items():
        layer_case.check(t, *want[name], "%s, gate %s" % (name, kind))


@pytest.mark.parametrize("dtype", sorted(CODE, key=str))
@pytest.mark.parametrize("T,E,k,ld,ldd", [(37, 60, 4, 64, 72), (300, 128, 8, 131, 129), (5, 7, 7, 7, 9), (70, 200, 20, 200, 204)])
def test_route(T, E, k, ld, ldd, dtype):
    """Gradients of the logits in rows that lie apart, whose gaps stay as they are; a mask of any bytes; no kept values wanted."""
    lib = _lib.load()
    gen = torch.Generator(device="cuda").manual_seed(7200 + T)
    logits = torch.empty(T, ld, device="cuda").normal_(0.0, 2.0, generator=gen).to(dtype)
    mask = torch.randint(0, 4, (T,), device="cuda", generator=gen).mul(85).to(torch.uint8)
    d = _lib.RouteDesc(E, k, CODE[dtype], 1)
    work = memory(size(lib.flashMoeRouteBytes, d, T))
    kept = torch.empty(2 + E, dtype=torch.int32, device="cuda")

    def forward(kept):
        w, e, c = torch.empty(T, k, device="cuda"), torch.empty(T, k, dtype=torch.int32, device="cuda"), torch.empty(E, dtype=torch.int32, device="cuda")
        b, z = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
        assert lib.flashMoeRoute(ctypes.byref(d), at(logits), ld, at(mask), T, at(w), at(e), at(c), at(b), at(z), at(kept), at(work), stream()) == 0
        return w, e, c, b, z

    w, e, c, b, z = forward(kept)
    for one, other in zip((w, e, c, b, z), forward(None)):
        assert torch.equal(one, other)
    dw, db, dz = torch.empty(T, k, device="cuda").normal_(generator=gen), torch.tensor(0.3, device="cuda"), torch.tensor(-0.2, device="cuda")
    out = torch.full((T, ldd), 77.0, dtype=dtype, device="cuda")
    assert lib.flashMoeRouteBackward(ctypes.byref(d), at(logits), ld, at(mask), T, at(w), at(e), at(kept), at(dw), at(db), at(dz), at(out), ldd,
                                     stream()) == 0
    want = layer_case.route(logits[:, :E], k, True, mask != 0, dw, db, dz)
    assert torch.equal(e.long(), want["experts"]) and torch.equal(c.long(), want["counts"]) and torch.equal(kept[2:], c)
    for name, t in (("weights", w), ("balance_loss", b), ("z_loss", z), ("dlogits", out[:, :E])):
        layer_case.check(t, *want[name], name)
    assert (out[:, E:] == 77.0).all()


@pytest.mark.parametrize("T,adapters", [(9, 3), (300, 40), (2000, 5)])
def test_adapters(T, adapters):
    """Rows apart on every side, in place and not; what lies between the rows stays as it is."""
    lib = _lib.load()
    N, K, r = 1160, 2056, 64
    gen = torch.Generator(device="cuda").manual_seed(7300 + T)

    def normal(sigma, *shape):
        return torch.empty(shape, device="cuda").normal_(0.0, sigma, generator=gen).bfloat16()

    x, y = normal(1.0, T, K + 8), normal(1.0, T, N + 16)
    down, up, scales = normal(K ** -0.5, adapters, r, K), normal(r ** -0.5, adapters, N, r), torch.rand(adapters, device="cuda", generator=gen)
    ids = torch.randint(-1, adapters, (T,), device="cuda", generator=gen, dtype=torch.int32)
    d = _lib.AdapterDesc(adapters, r, N, K, at(down), at(up), at(scales))
    work = memory(size(lib.flashMoeAdapterBytes, d, T))
    out = torch.full((T, N + 24), 77.0, dtype=torch.bfloat16, device="cuda")
    assert lib.flashMoeAdapterAdd(ctypes.byref(d), at(x), K + 8, at(y), N + 16, at(ids), T, at(out), N + 24, at(work), stream()) == 0
    layer_case.check(out[:, :N], *layer_case.adapters(y[:, :N], x[:, :K], down, up, scales, ids), "out")
    assert (out[:, N:] == 77.0).all()
    gaps = y[:, N:].clone()
    assert lib.flashMoeAdapterAdd(ctypes.byref(d), at(x), K + 8, at(y), N + 16, at(ids), T, at(y), N + 16, at(work), stream()) == 0
    assert torch.equal(y[:, :N], out[:, :N]) and torch.equal(y[:, N:], gaps)
