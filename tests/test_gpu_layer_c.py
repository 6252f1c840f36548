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
