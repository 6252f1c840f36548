"""Calls of the dense block and of MXFP4 products keep to the workspaces they ask for, whatever the scales' addresses:
the plans of thousands of calls on the CPU (tests/cpp/ffnWorkspaceTest.cpp), a few of them on the GPU with bytes behind
the workspace that must stay as they are."""
import ctypes
import os
import subprocess

import pytest
import torch

from flash_distributed_moe_amd import _lib
from tests import ffn_case

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GUARD = 4096


def test_plans_fit_their_workspaces():
    exe = os.path.join(ROOT, "tests", "cpp", "bin", "ffnWorkspaceTest")
    if not os.path.exists(exe):
        pytest.fail("%s is not built: run `make -C tests/cpp` (or __graft_entry__.build())" % exe)
    p = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert p.returncode == 0 and "4 tests, 0 failed" in p.stdout, p.stdout[-2000:]


def normal(*shape, sigma=1.0, seed=0, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(3000 + seed)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, sigma, generator=gen)


def guarded(size):
    return torch.full((size + GUARD,), 0xA5, dtype=torch.uint8, device="cuda")


def at_byte(t, offset):
    """A copy of t that begins `offset` bytes behind a multiple of 16."""
    room = torch.empty(t.numel() + 16, dtype=torch.uint8, device="cuda")
    room[offset:offset + t.numel()] = t.reshape(-1)
    return room[offset:offset + t.numel()].view(t.shape)


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,I", [(1, 1280, 17408), (16, 2048, 18432), (8, 16416, 4096), (32, 17408, 1024)])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_block_on_scales_at_odd_addresses(T, H, I, offset):
    from flash_distributed_moe_amd import flashFfnOp as ops

    lib = _lib.load()
    x = normal(T, H, seed=1)
    w13, w2 = ops.quantize_mxfp4(normal(2 * I, H, sigma=H ** -0.5, seed=2)), ops.quantize_mxfp4(normal(H, I, sigma=I ** -0.5, seed=3))
    s13, s2 = at_byte(w13.scales, offset), at_byte(w2.scales, 2 * offset + 1 if offset else 0)
    d = _lib.FfnDesc(H, I, _lib.BF16, _lib.ACT_SILU, _lib.FFN_MXFP4, w13.codes.data_ptr(), w2.codes.data_ptr(), s13.data_ptr(), s2.data_ptr())
    n = ctypes.c_size_t(0)
    assert lib.flashMoeFfnBytes(ctypes.byref(d), T, None, ctypes.byref(n), None) == 0
    work, y = guarded(n.value), torch.empty_like(x)
    assert lib.flashMoeFfnForward(ctypes.byref(d), x.data_ptr(), H, y.data_ptr(), H, T, None, work.data_ptr(), stream()) == 0
    torch.cuda.synchronize()
    assert (work[n.value:] == 0xA5).all()
    v13, v2 = (ffn_case.mx_values(*w).to(torch.bfloat16) for w in (w13, w2))
    ffn_case.check(y, *ffn_case.block(x, v13, v2, "silu")["y"], "T=%d H=%d I=%d" % (T, H, I))
    assert torch.equal(ops.gated_ffn(x, ops.Mxfp4(w13.codes, s13), ops.Mxfp4(w2.codes, s2)), y)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(5, 300, 4096), (5, 300, 17408), (40, 37, 5120), (93, 200, 7520)])
@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_products_on_scales_at_odd_addresses(M, N, K, both, offset):
    from flash_distributed_moe_amd import flashFfnOp as ops

    lib = _lib.load()
    w = ops.quantize_mxfp4(normal(N, K, sigma=0.02, seed=4))
    x = normal(M, K, seed=5)
    scales = at_byte(w.scales, offset)
    if both:
        x = ops.quantize_mxfp4(x)
        x_scales = at_byte(x.scales, 3 - offset)
    value = ffn_case.mx_values(*x) if both else x.double()
    n = ctypes.c_size_t(0)
    fmt = _lib.MXFP4 if both else _lib.BF16
    assert lib.flashMoeMxfp4LinearBytes(fmt, M, N, K, ctypes.byref(n)) == 0
    work = guarded(n.value)
    y = torch.full((M + 1, N), 7.0, dtype=torch.bfloat16, device="cuda")
    assert lib.flashMoeMxfp4Linear(fmt, (x.codes if both else x).data_ptr(), x_scales.data_ptr() if both else None, K, M, w.codes.data_ptr(),
                                   scales.data_ptr(), N, K, y.data_ptr(), N, work.data_ptr(), stream()) == 0
    torch.cuda.synchronize()
    assert (work[n.value:] == 0xA5).all() and (y[M] == 7).all()
    # every product is exact in float32; a sum of K is off by at most 2 K 2^-24 of the magnitudes, the result by 2^-8 of itself
    want, weights = value @ ffn_case.mx_values(*w).t(), ffn_case.mx_values(*w)
    far = 2.0 * K * 2.0 ** -24 * (value.abs() @ weights.abs().t())
    ffn_case.check(y[:M], want, far + 2.0 ** -8 * (want.abs() + far), "product")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,I", [(67, 384, 7680), (2100, 200, 3000), (50, 4360, 72), (8200, 72, 40)])
@pytest.mark.parametrize("want", [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)])
def test_backward_writes_nothing_behind_its_workspace(T, H, I, want, dtype):
    """Workspace, what the forward pass saved, and all three gradients, each with a guard behind it."""
    lib = _lib.load()
    size = torch.empty((), dtype=dtype).element_size()
    x, dy = normal(T, H, seed=6, dtype=dtype), normal(T, H, seed=7, dtype=dtype)
    w13, w2 = normal(2 * I, H, sigma=H ** -0.5, seed=8, dtype=dtype), normal(H, I, sigma=I ** -0.5, seed=9, dtype=dtype)
    d = _lib.FfnDesc(H, I, _lib.BF16 if size == 2 else _lib.F32, _lib.ACT_SILU, _lib.FFN_ROW_MAJOR, w13.data_ptr(), w2.data_ptr(), None, None)
    saved, back, fore = (ctypes.c_size_t(0) for _ in range(3))
    assert lib.flashMoeFfnBytes(ctypes.byref(d), T, ctypes.byref(saved), None, ctypes.byref(back)) == 0
    assert lib.flashMoeFfnSavingBytes(ctypes.byref(d), T, ctypes.byref(fore)) == 0
    keep, room, work = guarded(saved.value), guarded(fore.value), guarded(back.value)
    y = torch.empty_like(x)
    assert lib.flashMoeFfnForward(ctypes.byref(d), x.data_ptr(), H, y.data_ptr(), H, T, keep.data_ptr(), room.data_ptr(), stream()) == 0
    outs = [guarded(n * size) for n in (T * H, 2 * I * H, H * I)]
    at = [o.data_ptr() if wanted else None for o, wanted in zip(outs, want)]
    kept = keep.clone()
    assert lib.flashMoeFfnBackward(ctypes.byref(d), x.data_ptr(), H, dy.data_ptr(), H, T, keep.data_ptr(), work.data_ptr(), at[0], H, at[1],
                                   at[2], stream()) == 0
    torch.cuda.synchronize()
    assert torch.equal(keep, kept) and (keep[saved.value:] == 0xA5).all()
    assert (room[fore.value:] == 0xA5).all() and (work[back.value:] == 0xA5).all()
    values = ffn_case.block(x, w13, w2, "silu", dy)
    for o, wanted, name in zip(outs, want, ("dx", "dw13", "dw2")):
        n = o.numel() - GUARD
        assert (o[n:] == 0xA5).all() and (wanted or (o == 0xA5).all())
        if wanted:
            ffn_case.check(o[:n].view(dtype), *values[name], name)
