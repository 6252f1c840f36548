"""What the dense block and MXFP4 refuse, and the sizes they report: before anything is enqueued, so
without a GPU."""
import ctypes

import pytest
import torch

from flash_distributed_moe_amd import _lib, flashFfnOp as ops
from tests import ffn_case

BAD = _lib.HIP_ERROR_INVALID_VALUE


def desc(**kw):
    d = _lib.FfnDesc(64, 32, _lib.BF16, _lib.ACT_SILU, _lib.FFN_ROW_MAJOR, 0x1000, 0x2000, 0x3000, 0x4000)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def sizes(d, tokens):
    n = [ctypes.c_size_t(0) for _ in range(3)]
    rc = _lib.load().flashMoeFfnBytes(ctypes.byref(d), tokens, *(ctypes.byref(v) for v in n))
    return rc, [v.value for v in n]


def test_sizes():
    rc, (saved, forward, backward) = sizes(desc(), 100)
    assert rc == 0
    # kept: both projections in float32 and h; a forward pass alone needs h, a backward pass the projections' gradients
    assert 100 * 32 * (8 + 2) <= saved < 100 * 32 * 10 + 1024
    assert forward >= 100 * 32 * 2 and backward >= 100 * 64 * 2
    assert sizes(desc(), 0)[0] == 0
    # more than 2^32 bytes
    rc, (saved, _, _) = sizes(desc(hidden=4096, intermediate=12288), 1 << 20)
    assert rc == 0 and saved >= (1 << 20) * 12288 * 10


def test_workspaces_of_shared_sums():
    def saving(d, tokens):
        n = ctypes.c_size_t(0)
        assert _lib.load().flashMoeFfnSavingBytes(ctypes.byref(d), tokens, ctypes.byref(n)) == 0
        return n.value

    for weights in (0, 1):
        few = desc(hidden=384, intermediate=7680, weights=weights)  # 67 x 384 results of 7680 products each
        assert saving(few, 67) >= 2 * 67 * 384 * 4
        assert sizes(few, 67)[1][1] >= 67 * 7680 * 2 + saving(few, 67)
        assert saving(few, 0) == 0
    assert saving(desc(hidden=4096, intermediate=12288), 8192) == 0
    assert saving(desc(), 100) == 0
    assert sizes(desc(hidden=4096, intermediate=12288), 8192)[1][2] < 8192 * (2 * 12288 + 64) * 2 + 1024
    assert _lib.load().flashMoeFfnSavingBytes(ctypes.byref(desc()), 1, None) == BAD
    assert _lib.load().flashMoeFfnSavingBytes(ctypes.byref(desc()), -1, ctypes.byref(ctypes.c_size_t(0))) == BAD


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(dtype=-1), dict(activation=2), dict(weights=2), dict(hidden=0), dict(hidden=60),
                                dict(hidden=(1 << 20) + 8), dict(intermediate=4), dict(intermediate=(1 << 19) + 8),
                                dict(weights=1, hidden=72), dict(weights=1, intermediate=40), dict(weights=1, dtype=0)])
def test_bad_descriptions(kw, capfd):
    assert sizes(desc(**kw), 4)[0] == BAD
    assert "[MOE ERROR:" in capfd.readouterr().out


def test_negative_batches_and_null_descriptions():
    assert sizes(desc(), -1)[0] == BAD
    assert _lib.load().flashMoeFfnBytes(None, 1, None, None, None) == BAD


def forward(d=None, x=0x10000, ldx=64, y=0x20000, ldy=64, tokens=4, saved=None, work=0x30000):
    return _lib.load().flashMoeFfnForward(ctypes.byref(d or desc()), x, ldx, y, ldy, tokens, saved, work, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(y=None), dict(x=0x10008), dict(y=0x20002), dict(ldx=63), dict(ldx=68), dict(ldy=8),
                                dict(ldx=(1 << 20) + 8), dict(work=None), dict(work=0x30004), dict(saved=0x40001),
                                dict(d=desc(w13=None)), dict(d=desc(w2=None)), dict(d=desc(w2=0x2004)),
                                dict(d=desc(weights=1, w2_scales=None)), dict(d=desc(weights=1), saved=0x40000)])
def test_forward_refuses(kw, capfd):
    assert forward(**kw) == BAD
    assert "[MOE ERROR:" in capfd.readouterr().out


def test_no_tokens_needs_no_pointers():
    assert forward(x=None, y=None, work=None, tokens=0) == 0


def backward(d=None, x=0x10000, ldx=64, dy=0x20000, lddy=64, tokens=4, saved=0x30000, work=0x40000, dx=0x50000, lddx=64, dw13=0x60000,
             dw2=0x70000):
    return _lib.load().flashMoeFfnBackward(ctypes.byref(d or desc()), x, ldx, dy, lddy, tokens, saved, work, dx, lddx, dw13, dw2, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(dy=None), dict(dy=0x20008), dict(lddy=60), dict(saved=None), dict(work=None),
                                dict(dx=0x50004), dict(lddx=56), dict(dw13=0x60002), dict(dw2=0x70008), dict(d=desc(weights=1)),
                                dict(tokens=-1)])
def test_backward_refuses(kw, capfd):
    assert backward(**kw) == BAD
    assert "[MOE ERROR:" in capfd.readouterr().out


def test_backward_without_results_is_nothing():
    assert backward(dx=None, dw13=None, dw2=None) == 0


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(x=None), dict(x=0x1008), dict(ldx=32), dict(ldx=68), dict(k=48), dict(k=0), dict(rows=-1),
                                dict(codes=None), dict(scales=None), dict(codes=0x2008)])
def test_conversions_refuse(kw, capfd):
    a = dict(dtype=_lib.BF16, x=0x1000, ldx=64, rows=3, k=64, codes=0x2000, scales=0x3000)
    a.update(kw)
    lib = _lib.load()
    assert lib.flashMoeMxfp4Quantize(a["dtype"], a["x"], a["ldx"], a["rows"], a["k"], a["codes"], a["scales"], None) == BAD
    assert lib.flashMoeMxfp4Dequantize(a["dtype"], a["codes"], a["scales"], a["rows"], a["k"], a["x"], a["ldx"], None) == BAD
    assert capfd.readouterr().out.count("[MOE ERROR:") == 2


@pytest.mark.parametrize("kw", [dict(fmt=0), dict(fmt=3), dict(x=None), dict(x=0x1004), dict(ldx=60), dict(k=80), dict(n=-1), dict(rows=-1),
                                dict(codes=None), dict(codes=0x2004), dict(scales=None), dict(y=None), dict(y=0x5002), dict(ldy=7),
                                dict(ldy=12), dict(n=7, ldy=7, y=0x5001), dict(fmt=2, ldx=128), dict(fmt=2, x_scales=None)])
def test_product_refuses(kw, capfd):
    a = dict(fmt=_lib.BF16, x=0x1000, x_scales=0x4000, ldx=64, rows=3, codes=0x2000, scales=0x3000, n=8, k=64, y=0x5000, ldy=8)
    a.update(kw)
    lib = _lib.load()
    work = 0x6000
    assert lib.flashMoeMxfp4Linear(a["fmt"], a["x"], a["x_scales"], a["ldx"], a["rows"], a["codes"], a["scales"], a["n"], a["k"], a["y"],
                                   a["ldy"], work, None) == BAD
    assert "[MOE ERROR:" in capfd.readouterr().out


def test_python_surface_refuses():
    x, w13, w2 = torch.zeros(2, 64), torch.zeros(64, 64), torch.zeros(64, 32)
    q = ops.Mxfp4(torch.zeros(64, 32, dtype=torch.uint8), torch.zeros(64, 2, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.gated_ffn(x, w13, w2)
    with pytest.raises(RuntimeError, match="activation must be one of"):
        ops.gated_ffn(x, w13, w2, activation="relu")
    with pytest.raises(RuntimeError, match="both weights must be MXFP4"):
        ops.gated_ffn(x, q, w2)
    with pytest.raises(RuntimeError, match="no backward pass"):
        ops.gated_ffn(x.requires_grad_(), q, q)
    with pytest.raises(RuntimeError, match="no backward pass"):
        ops.mxfp4_linear(x, q)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.quantize_mxfp4(x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.dequantize_mxfp4(q)
    with pytest.raises(RuntimeError, match="quantize must be"):
        ops.FlashGatedFfn(None, quantize="int4")


def test_definitions_agree():
    """The restatement of the format against each value's own nearest neighbour, and of the gradients against autograd."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(40, 96, generator=gen, dtype=torch.float64) * torch.exp2(torch.randint(-20, 20, (40, 1), generator=gen).double())
    codes, scales = ffn_case.mx_encode(x)
    values = ffn_case.mx_values(codes, scales)
    scale = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    most = x.abs().reshape(40, 3, 32).amax(-1).repeat_interleave(32, -1) / scale
    assert ((most >= 4) & (most < 8)).all()
    grid = torch.tensor(ffn_case.GRID, dtype=torch.float64)
    nearest = ((x.abs() / scale)[..., None] - grid).abs().amin(-1)
    assert torch.allclose((values.abs() - x.abs()).abs() / scale, nearest, rtol=0, atol=1e-12)
    assert ((values == 0) | (values.sign() == x.sign())).all()
    for act in ("silu", "gelu_tanh"):
        x, w13, w2, dy = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((5, 16), (24, 16), (16, 12), (5, 16)))
        leaves = [t.clone().requires_grad_() for t in (x, w13, w2)]
        g, u = (leaves[0] @ leaves[1].t()).chunk(2, -1)
        a = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g, approximate="tanh")
        y = (a * u) @ leaves[2].t()
        grads = torch.autograd.grad(y, leaves, dy)
        ffn_case.HALF[torch.float64] = 0.0
        got = ffn_case.block(x, w13, w2, act, dy)
        for name, t in zip(("y", "dx", "dw13", "dw2"), (y.detach(), *grads)):
            assert torch.allclose(got[name][0], t, rtol=1e-10, atol=1e-10)
