"""The norms around a block: behind the operator with its gate (`gated_rms_norm`), and between two blocks with the residual sum (`residual_rms_norm`).
One pass over each tensor, forward and backward, in hand-written sm_100a kernels (`csrc/kda_norm.cu`); bfloat16 and float32 tensors, no fallback."""
from __future__ import annotations

from . import _lib

_ACTIVATIONS = {"sigmoid": 0, "silu": 1, "swish": 1}


def _native():
    return _lib._native or _lib.native()


def gated_rms_norm(x, gate, weight=None, eps=1e-6, activation="sigmoid"):
    """y = x / sqrt(mean(x^2) + eps) * weight * act(gate) over the last dimension (up to 8192 columns), act = "sigmoid", or "silu" ("swish"): z sigmoid(z).

    x and gate [..., D] in bfloat16 or float32 each, weight [D] or None.  y has x's type; with float32 x the activation is good to float32's rounding, with bfloat16 x
    fast exponentials are taken (4e-6 at most).  Differentiable with respect to all three; sums over rows are taken in float32 and in a fixed order."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"kda_b200: activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    return _native().gated_norm(x, gate, weight, eps, _ACTIVATIONS[activation])


def residual_rms_norm(x, residual, weight, scale=None, post_weight=None, eps=1e-6):
    """What stands between two blocks: returns (y, r) with r = residual + scale * b and y = r / sqrt(mean(r^2) + eps) * weight, where b is the block's output x or,
    with `post_weight` [D], x / sqrt(mean(x^2) + eps) * post_weight.

    x, residual [..., D] (up to 8192 columns) in bfloat16 or float32 each; weight, post_weight [D]; scale a number (None: 1) or [D].  y has x's type, r
    residual's; y is computed from r before its rounding.  Differentiable with respect to every tensor."""
    return _native().residual_norm(x, residual, weight, scale, post_weight, eps)
