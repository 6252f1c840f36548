"""The dense gated feed-forward block and MXFP4 weights, beside the sparse layer.

The models whose mixture-of-experts layer `flashMoeOp.FlashMoeBlockWrapper` runs also have dense
blocks and shared experts of the same form, y = (act(x Wg^T) * (x Wu^T)) Wd^T, on the weight
layouts of one expert (w13 [2I, H]: gate rows, then up rows; w2 [H, I]). `gated_ffn` is that block,
differentiable; `FlashGatedFfn` a module of it over the weights of a block it is given.

MXFP4 keeps 32 consecutive values of a row in 16 bytes and a scale byte (the Open Compute
microscaling format): `quantize_mxfp4`, `dequantize_mxfp4`, `mxfp4_linear` for a product with such
weights, and `gated_ffn` takes them in place of both weights (no gradients).

There is no fallback: everything runs on the compiled `flashMoeLauncher` extension, on the current
stream of the tensors' device, and can be captured into a HIP graph. Wrong arguments raise
RuntimeError, and so do inputs that carry a forward-mode tangent. (The reference has none of these operators; its wrapper,
test/singleGPU/python/flashMoeOp.py:7-38, covers the sparse block only.)
"""
import os
import sys
from typing import NamedTuple

import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if _ROOT not in sys.path:
    sys.path.insert(0, _ROOT)
try:
    import flashMoeLauncher
except ImportError as e:  # no fallback: say how to build it
    raise ImportError("the flashMoeLauncher extension is not built; run "
                      "`python -m flash_distributed_moe_amd.build` (%s)" % e)

ACTIVATIONS = {"silu": flashMoeLauncher.ACT_SILU, "gelu_tanh": flashMoeLauncher.ACT_GELU_TANH}


class Mxfp4(NamedTuple):
    """A tensor [..., K] in MXFP4: codes uint8 [..., K/2] (the even value in the low half of its
    byte) and scales uint8 [..., K/32] (b stands for 2^(b-127), 255 for NaN)."""

    codes: torch.Tensor
    scales: torch.Tensor


# what reading an attribute of a stranger or handing it to the extension raises
_STRANGERS = (AttributeError, TypeError)


def _stranger(wanted, *args):
    return RuntimeError("%s: not %s" % (wanted, ", ".join(type(a).__name__ for a in args)))


def quantize_mxfp4(x):
    """x [..., K] (float32 or bfloat16, K a multiple of 32) as Mxfp4. Not differentiable."""
    try:
        return Mxfp4(*flashMoeLauncher.mxfp4_quantize(x.detach()))
    except _STRANGERS:
        raise _stranger("x must be a tensor", x) from None


def dequantize_mxfp4(q, dtype=torch.bfloat16):
    """The values of q, which both dtypes hold exactly."""
    try:
        return flashMoeLauncher.mxfp4_dequantize(q.codes, q.scales, dtype)
    except _STRANGERS:
        raise _stranger("q must be Mxfp4 and dtype a torch.dtype", q, dtype) from None


class Adapters(NamedTuple):
    """Low-rank adapters of one projection [N, K]: down bfloat16 [adapters, r, K], up bfloat16 [adapters, N, r], scales float32
    [adapters]. Adapter i adds scales[i] * up[i] @ down[i] to the projection's weights. r is a multiple of 8, up to 128
    (shorter adapters are filled up with zeros), and there are up to 1000 of them."""

    down: torch.Tensor
    up: torch.Tensor
    scales: torch.Tensor


def add_adapters(y, x, adapters, ids, out=None):
    """y [..., N] + scales[i] * (x [..., K] down[i]^T) up[i]^T, i = ids[...] (int32) being each row's adapter, for y that
    a projection of x gave: one call for the rows of many requests, in any order.

    All bfloat16, rounded once. Sums are float32, and so is what goes from the first product to the second while rows are
    few; of many rows it is two bfloat16 parts, which leave out 2^-16 of it, so that a row's last bits may depend on how many the call has.
    A row whose id is negative has no adapter and keeps y; a row whose id names no adapter becomes NaN (ids are not read on the
    host). The result is new, or out, which may be y and overlaps nothing else. K and N multiples of 8. Not differentiable."""
    try:
        return flashMoeLauncher.add_adapters(y, x, adapters.down, adapters.up, adapters.scales, ids, out)
    except _STRANGERS:
        raise _stranger("y, x, ids and out must be tensors, adapters Adapters", y, x, adapters, ids, out) from None


def mxfp4_linear(x, weight, adapters=None, ids=None):
    """x [..., K] (bfloat16, or Mxfp4) times the transpose of weight (Mxfp4 [N, K]): bfloat16 [..., N],
    summed in float32. With adapters and ids what `add_adapters` adds to that, for bfloat16 x. Not differentiable."""
    if (adapters is None) != (ids is None):
        raise RuntimeError("adapters and ids belong together")
    if adapters is not None:
        if isinstance(x, Mxfp4):
            raise RuntimeError("adapters take bfloat16 x")
        y = mxfp4_linear(x, weight)
        return add_adapters(y, x, adapters, ids, out=y)
    try:
        if isinstance(x, Mxfp4):
            return flashMoeLauncher.mxfp4_linear(x.codes, x.scales, weight.codes, weight.scales)
        _refuse_grad(x)
        return flashMoeLauncher.mxfp4_linear(x, None, weight.codes, weight.scales)
    except _STRANGERS:
        raise _stranger("x must be a tensor or Mxfp4, weight Mxfp4", x, weight) from None


def _refuse_grad(x):
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("products with MXFP4 weights have no backward pass: detach x or use torch.no_grad()")


def gated_ffn(x, w13, w2, activation="silu"):
    """(act(x Wg^T) * (x Wu^T)) Wd^T for x [..., H], w13 [2I, H] (gate rows, then up rows) and w2 [H, I].

    float32 or bfloat16 throughout, H and I multiples of 8; or x bfloat16 and both weights Mxfp4,
    H and I multiples of 32. activation: "silu" or "gelu_tanh". Weights are contiguous; rows of x
    may lie apart. Gradients (once) for x and row-major weights; a pass that needs them keeps the two
    projections in float32 and h until its backward pass. A step that is captured into a HIP graph wants no
    eager graph of the same parameters alive: the call raises then."""
    if not isinstance(activation, str) or activation not in ACTIVATIONS:
        raise RuntimeError("activation must be one of %s" % ", ".join(sorted(ACTIVATIONS)))
    act = ACTIVATIONS[activation]
    try:
        if isinstance(w13, Mxfp4) or isinstance(w2, Mxfp4):
            if not (isinstance(w13, Mxfp4) and isinstance(w2, Mxfp4)):
                raise RuntimeError("both weights must be MXFP4, or neither")
            _refuse_grad(x)
            return flashMoeLauncher.gated_ffn_mxfp4(x, w13.codes, w2.codes, w13.scales, w2.scales, act)
        return flashMoeLauncher.gated_ffn(x, w13, w2, act)
    except _STRANGERS:
        raise _stranger("x must be a tensor, the weights tensors or Mxfp4", x, w13, w2) from None


def _activation_of(act_fn):
    """Which of ACTIVATIONS a block's activation is, by its values; of gates alone, or of gates and up projections side by
    side (a vector of gates and ones tells)."""
    g = torch.linspace(-6.0, 6.0, 97, dtype=torch.float32, device="cpu")
    try:
        with torch.no_grad():
            a = act_fn(torch.cat((g, torch.ones_like(g))))[..., :97]
        known = {"silu": torch.nn.functional.silu(g), "gelu_tanh": torch.nn.functional.gelu(g, approximate="tanh")}
        for name, values in known.items():
            if torch.allclose(a.float().cpu(), values, rtol=0, atol=1e-4):  # exact GELU is 5e-4 off its tanh form
                return name
    except Exception:  # whatever a stranger's code raises for these arguments
        pass
    raise RuntimeError("the block's act_fn is neither SiLU nor GELU's tanh form: pass activation to say which to use")


class FlashGatedFfn(torch.nn.Module):
    """`gated_ffn` over the weights of a dense block or shared expert: a module with
    `gate_up_proj.weight` [2I, H] and `down_proj.weight` [H, I], without biases. The parameters stay the block's own.
    activation: by default what the block's `act_fn` is, SiLU if it has none. quantize="mxfp4" converts the weights
    once, into buffers of this module (the block is not kept)."""

    def __init__(self, block, activation=None, quantize=None):
        super().__init__()
        if activation is not None and activation not in ACTIVATIONS:
            raise RuntimeError("activation must be one of %s" % ", ".join(sorted(ACTIVATIONS)))
        if quantize not in (None, "mxfp4"):
            raise RuntimeError('quantize must be None or "mxfp4"')
        for name in ("gate_up_proj", "down_proj"):
            if getattr(getattr(block, name), "bias", None) is not None:
                raise RuntimeError("%s has a bias, which gated_ffn does not add" % name)
        if activation is None:
            act_fn = getattr(block, "act_fn", None)
            activation = "silu" if act_fn is None else _activation_of(act_fn)
        self.activation, self.quantize = activation, quantize
        w13, w2 = block.gate_up_proj.weight, block.down_proj.weight
        if quantize is None:
            self.w13, self.w2 = w13, w2
        else:
            for name, w in (("w13", w13), ("w2", w2)):
                q = quantize_mxfp4(w)
                self.register_buffer(name + "_codes", q.codes)
                self.register_buffer(name + "_scales", q.scales)

    def forward(self, x):
        if self.quantize is None:
            return gated_ffn(x, self.w13, self.w2, self.activation)
        return gated_ffn(x, Mxfp4(self.w13_codes, self.w13_scales), Mxfp4(self.w2_codes, self.w2_scales), self.activation)
