"""kda_b200 — Kimi Delta Attention for NVIDIA B200 (sm_100a).

`chunk_kda` and `fused_recurrent_kda` keep the operator API of flash-linear-attention's KDA ops and run
hand-written CUDA kernels through the C ABI in include/kda_b200.h (libkda_b200.so, built in-tree by
`python -m kda_b200.build`).  `chunk_gated_delta` and `fused_recurrent_gated_delta` are the rule with one decay per head;
`gated_rms_norm` and `residual_rms_norm` the norms around a block.  No Triton, no backend dispatch, no CPU fallback."""
from .delta import chunk_gated_delta, fused_recurrent_gated_delta, fused_recurrent_gated_delta_fwd  # noqa: F401
from .norms import gated_rms_norm, residual_rms_norm  # noqa: F401
from .ops import chunk_kda, fused_kda_gate, fused_recurrent_kda, fused_recurrent_kda_fwd  # noqa: F401

__all__ = ["chunk_gated_delta", "chunk_kda", "fused_kda_gate", "fused_recurrent_gated_delta", "fused_recurrent_gated_delta_fwd", "fused_recurrent_kda",
           "fused_recurrent_kda_fwd", "gated_rms_norm", "residual_rms_norm"]
__version__ = "0.1.0"
