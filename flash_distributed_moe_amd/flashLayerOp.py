"""What stands around the blocks of a layer: the router's choice with its losses, and the norms before and
after a block.

The sparse layer of `flashMoeOp.FlashMoeBlockWrapper` routes inside its kernel; a model that trains, or
that watches how its experts are used, needs the choice by itself, with the counts and losses that
go with it: `route`. Around that layer and around the dense block of `flashFfnOp` stand `block_norm`, in front of
a block, and `block_join`, behind it. (The reference's layer has neither losses nor norms nor gradients,
test/singleGPU/cpp/moe/reference/refFullMoe.h:9-70.)

There is no fallback: everything runs on the compiled `flashMoeLauncher` extension, on the current
stream of the tensors' device, and can be captured into a HIP graph (with its backward pass as long as no eager
graph of the same parameters is alive: the call raises then). Wrong arguments raise RuntimeError, and so do
inputs that carry a forward-mode tangent; gradients are differentiated once.
"""
from typing import NamedTuple

import torch

from .flashFfnOp import _STRANGERS, _stranger, flashMoeLauncher


class Routing(NamedTuple):
    """What `route` returns, for logits [..., E] and k winners a token."""

    weights: torch.Tensor       # float32 [..., k], differentiable
    experts: torch.Tensor       # int32 [..., k], -1 where no candidate was left
    counts: torch.Tensor        # int32 [E]: slots that each expert won
    balance_loss: torch.Tensor  # float32 scalar, differentiable: 1 if all experts are used and liked evenly
    z_loss: torch.Tensor        # float32 scalar, differentiable


def route(logits, top_k, renormalize=True, mask=None):
    """The top_k largest of each token's logits [..., E] (float32 or bfloat16), as `Routing`.

    Winners come largest first, the lowest expert of equals, as the sparse layer picks them. A logit is a candidate if
    it is greater than its type's lowest value (NaN and -inf are none); mask [...] (bool) leaves out the tokens where
    it is False. With p the softmax over a token's candidates, weights are p of the winners, divided by their
    sum if renormalize; balance_loss is E sum_e (counts_e / slots won) (mean_t p_te) and z_loss the mean squared
    logarithm of the sum of exp(logits), both over the tokens that have a candidate. Gradients reach the logits from weights and both
    losses; the choice and the counts are constants. E up to 256, top_k up to min(E, 32).
    (The sparse layer routes by itself and takes no choice from outside: beside it this call gives the counts, losses and
    their gradient.)"""
    try:
        return Routing(*flashMoeLauncher.route(logits, top_k, bool(renormalize), mask))
    except _STRANGERS:
        raise _stranger("logits must be a tensor, top_k a whole number, mask a tensor or None", logits, top_k, mask) from None


def block_norm(x, weight, eps=1e-6):
    """The norm in front of a block: x / sqrt(mean x^2 + eps) * weight for x [..., H] (float32 or bfloat16) and weight [H] of
    x's dtype. H a multiple of 8, up to 8192. Squares are summed in float32: where they overflow (values from 1.8 10^19 / sqrt(H) on) the
    row becomes zeros. Differentiable in x and weight."""
    try:
        return flashMoeLauncher.block_norm(x, None, None, None, _present(weight), 1.0, 1.0, eps)[0]
    except _STRANGERS:
        raise _stranger("x and weight must be tensors, eps a number", x, weight, eps) from None


def block_join(x, branch, post_weight=None, gate=None, next_weight=None, residual_scale=1.0, branch_scale=1.0, eps=1e-6):
    """A block's output joins the residual stream: y = residual_scale * x + branch_scale * gate * z, where z is the
    branch, or with post_weight [H] its norm branch / sqrt(mean branch^2 + eps) * post_weight. With next_weight [H] the result is
    (y, h), h = y / sqrt(mean y^2 + eps) * next_weight being what the next block takes (of y before it is rounded).

    x and branch [..., H] share shape and dtype (float32 or bfloat16), rows may lie apart; H a multiple of 8, up to 8192.
    gate: [H], or x's leading dimensions up to some one, ones from there and H ([B, 1, H]: one for each sequence), or one value a
    token ([..., 1]). All of x's dtype. Everything of a row is float32 until y and h are rounded (squares too, as in
    `block_norm`). Differentiable in all tensors; the scales and eps are numbers."""
    try:
        out = flashMoeLauncher.block_norm(x, _present(branch), post_weight, gate, next_weight, residual_scale, branch_scale, eps)
    except _STRANGERS:
        raise _stranger("x and branch must be tensors, weights and gate tensors or None, the rest numbers", x, branch, post_weight, gate,
                        next_weight, residual_scale, branch_scale, eps) from None
    return out[0] if next_weight is None else tuple(out)


def _present(t):
    if t is None:
        raise TypeError("None")
    return t
