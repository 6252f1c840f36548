"""Calls of the dense block and of MXFP4 that would give an answer that is not the caller's: refused, before anything about
the tensors' device is looked at, so without a GPU."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

from flash_distributed_moe_amd import _lib, flashFfnOp as ops


def operands():
    return torch.zeros(2, 64), torch.zeros(64, 64), torch.zeros(64, 32)


def packed():
    return ops.Mxfp4(torch.zeros(64, 32, dtype=torch.uint8), torch.zeros(64, 2, dtype=torch.uint8))


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_is_refused(which, leaf):
    """A dual tensor has no requires_grad: its tangent would be dropped without a word."""
    args = list(operands())
    with fwd.dual_level():
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        if leaf:
            args[(which + 1) % 3].requires_grad_()
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.gated_ffn(*args)


def test_forward_mode_is_refused_with_mxfp4_weights():
    q = packed()
    with fwd.dual_level():
        x = fwd.make_dual(torch.zeros(2, 64), torch.ones(2, 64))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.mxfp4_linear(x, q)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.gated_ffn(x, q, q)
        # detached values, and dual tensors that are not differentiated, are ordinary ones: the next check speaks
        with fwd._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="CUDA tensor"):
            ops.gated_ffn(x, *operands()[1:])


def test_the_extension_takes_no_saved_results():
    """What a forward pass keeps is the autograd node's: no call takes it from its caller or hands it out."""
    bound = [name for name in dir(ops.flashMoeLauncher) if "ffn" in name or "mxfp4" in name]
    assert sorted(bound) == ["gated_ffn", "gated_ffn_mxfp4", "mxfp4_dequantize", "mxfp4_linear", "mxfp4_quantize"]


@pytest.mark.parametrize("call", [
    lambda x, w13, w2, q: ops.mxfp4_linear(x, w13),
    lambda x, w13, w2, q: ops.mxfp4_linear(None, q),
    lambda x, w13, w2, q: ops.mxfp4_linear([1.0], q),
    lambda x, w13, w2, q: ops.mxfp4_linear(x, None),
    lambda x, w13, w2, q: ops.dequantize_mxfp4(x),
    lambda x, w13, w2, q: ops.dequantize_mxfp4(q, "bfloat16"),
    lambda x, w13, w2, q: ops.quantize_mxfp4(q),
    lambda x, w13, w2, q: ops.quantize_mxfp4(None),
    lambda x, w13, w2, q: ops.gated_ffn(None, w13, w2),
    lambda x, w13, w2, q: ops.gated_ffn(x, None, w2),
    lambda x, w13, w2, q: ops.gated_ffn(x, w13, 3.0),
    lambda x, w13, w2, q: ops.gated_ffn(q, q, q),
    lambda x, w13, w2, q: ops.gated_ffn(x, ops.Mxfp4(q.codes, None), q),
    lambda x, w13, w2, q: ops.mxfp4_linear(ops.Mxfp4(None, None), q),
    lambda x, w13, w2, q: ops.dequantize_mxfp4(ops.Mxfp4(1, 2)),
    lambda x, w13, w2, q: ops.gated_ffn(x, w13, w2, activation=["silu"]),
])
def test_arguments_of_another_kind(call):
    """Wrong arguments raise RuntimeError, as the documentation says, whatever they are instead."""
    with pytest.raises(RuntimeError):
        call(*operands(), packed())


HUGE = [(1 << 30) + 1, (1 << 31) - 64, (1 << 31) - 1]


@pytest.mark.parametrize("n", HUGE)
def test_batches_beyond_what_a_launch_counts(n, capfd):
    """Sizes whose tiles would be counted beyond 32 bits, among them a sum over tokens that would have come out as zeros."""
    lib = _lib.load()
    d = _lib.FfnDesc(8, 8, _lib.BF16, _lib.ACT_SILU, _lib.FFN_ROW_MAJOR, 0x1000, 0x2000, None, None)
    size = ctypes.c_size_t(0)
    bad = _lib.HIP_ERROR_INVALID_VALUE
    assert lib.flashMoeFfnBytes(ctypes.byref(d), n, ctypes.byref(size), None, None) == bad
    assert lib.flashMoeFfnForward(ctypes.byref(d), 0x10000, 8, 0x20000, 8, n, None, 0x30000, None) == bad
    assert lib.flashMoeFfnBackward(ctypes.byref(d), 0x10000, 8, 0x20000, 8, n, 0x30000, None, None, 8, None, 0x40000, None) == bad
    for fmt in (_lib.BF16, _lib.MXFP4):
        for rows, columns in ((n, 8), (1, n)):
            assert lib.flashMoeMxfp4LinearBytes(fmt, rows, columns, 32, ctypes.byref(size)) == bad
            assert lib.flashMoeMxfp4Linear(fmt, 0x10000, 0x1000, 32, rows, 0x20000, 0x2000, columns, 32, 0x30000, columns, 0x40000, None) == bad
    assert lib.flashMoeMxfp4Quantize(_lib.BF16, 0x10000, 64, n, 64, 0x20000, 0x30000, None) == bad
    assert lib.flashMoeMxfp4Dequantize(_lib.BF16, 0x10000, 0x20000, n, 64, 0x30000, 64, None) == bad
    assert "[MOE" in capfd.readouterr().out
