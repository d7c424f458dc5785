"""The gated delta rule with one decay per token and head, beside `chunk_kda` / `fused_recurrent_kda`, whose decay is per key channel:

    S_t = exp(g_t) (I - beta_t k_t k_t^T) S_{t-1} + beta_t k_t v_t^T,      o_t = scale S_t^T q_t

g is [B, T, HV], and with it `dt_bias` [HV].  The token-by-token operators otherwise take what theirs of the per-channel rule take; the chunked one takes a log-decay
and a beta that are activated already (no raw gate and logits, no intermediate states), and checks its arguments as `chunk_kda` does.  Everything below the Python
signature runs in hand-written sm_100a kernels (`csrc/delta*.cu`, `csrc/kda_decode_bulk.cu`), and there is no fallback."""
from __future__ import annotations

import torch

from . import _lib, ops

SCAN_SLICES = 0      # CTAs per (sequence, head) of the walks: 0 = automatic; 1, 2 or 4 force a layout (tests, measurements)


def _native():
    return _lib._native or _lib.native()


def fused_recurrent_gated_delta_fwd(q, k, v, g, beta, A_log=None, dt_bias=None, initial_state=None, scale=None, output_final_state=False, inplace_final_state=True,
                                    cu_seqlens=None, ssm_state_indices=None, num_accepted_tokens=None, use_qk_l2norm_in_kernel=False, use_gate_in_kernel=False,
                                    use_beta_sigmoid_in_kernel=False, lower_bound=None, out=None, transpose_state_layout=False):
    """Decode step, forward only: `fused_recurrent_kda_fwd` with one decay per token and head.

    q, k [B,T,H,K]; v [B,T,HV,V]; g, beta [B,T,HV] in bfloat16 or float32 (raw layer outputs with `use_gate_in_kernel`, `use_beta_sigmoid_in_kernel`; then
    g = -exp(A_log) softplus(g + dt_bias) with A_log, dt_bias [HV], or lower_bound sigmoid(exp(A_log) (g + dt_bias)); to float32's rounding: states carry about 1e-7 of
    their norm).  K in {32, 64, 128, 256}, V a multiple of 32.
    With `inplace_final_state` states are written over `initial_state`, a float32 [slots, HV, K, V] pool where `ssm_state_indices` [N] or [N, T] names the slot of
    every token: a sequence starts from the slot of its first token (with `num_accepted_tokens` [N] of its last accepted one) and the state behind token t lands
    in that token's slot.  Slots are read as 32-bit numbers; no two sequences may name the same one.  A sequence whose starting slot lies outside the pool (-1: a padded entry) or whose accepted count
    names no column gets zeros for its rows of o and touches no state; a later token's slot outside the pool is left out.  With cu_seqlens, rows of o (of `out` too) in
    front of the first sequence and behind the last one become zeros.  Returns (o, states)."""
    return _native().delta_recurrent_fwd(
        q, k, v, g, beta, A_log, dt_bias, initial_state, scale, output_final_state, inplace_final_state, cu_seqlens, ssm_state_indices, num_accepted_tokens,
        use_qk_l2norm_in_kernel, use_gate_in_kernel, use_beta_sigmoid_in_kernel, lower_bound, out, transpose_state_layout)


def fused_recurrent_gated_delta(q, k, v, g, beta, A_log=None, dt_bias=None, scale=None, initial_state=None, output_final_state=False, use_qk_l2norm_in_kernel=False,
                                use_gate_in_kernel=False, use_beta_sigmoid_in_kernel=False, lower_bound=None, cu_seqlens=None, transpose_state_layout=False):
    """Token by token, forward only: `fused_recurrent_kda` with one decay per token and head (arguments as in `fused_recurrent_gated_delta_fwd`).
    initial_state [N,HV,K,V] float32 is left as it is.  Returns (o, final_state or None)."""
    if cu_seqlens is not None and initial_state is not None and initial_state.shape[0] != len(cu_seqlens) - 1:
        raise ValueError(f"The number of initial states is expected to be equal to the number of input sequences, i.e., {len(cu_seqlens) - 1} rather than "
                         f"{initial_state.shape[0]}.")
    return fused_recurrent_gated_delta_fwd(
        q, k, v, g, beta, A_log=A_log, dt_bias=dt_bias, initial_state=initial_state, scale=scale, output_final_state=output_final_state, inplace_final_state=False,
        cu_seqlens=cu_seqlens, use_qk_l2norm_in_kernel=use_qk_l2norm_in_kernel, use_gate_in_kernel=use_gate_in_kernel,
        use_beta_sigmoid_in_kernel=use_beta_sigmoid_in_kernel, lower_bound=lower_bound, transpose_state_layout=transpose_state_layout)


def _no_second_derivative(grads):
    if torch.is_grad_enabled():      # a backward with create_graph=True: the kernels' gradients carry no graph
        raise NotImplementedError("kda_b200: chunk_gated_delta has no second derivative (create_graph=True)")


def _float32_packed(q, k, v, g, beta, cu_seqlens, call):
    """A packed float32 call with gradients.  The kernels behind chunk_kda take the offsets as they are and leave rows of no sequence unwritten; here offsets stay
    inside the tensors, and these rows are cut off on the way in and on the way out, so that they are zero in o and in the gradients."""
    cu = cu_seqlens.to(q.device).clamp(0, q.shape[1]).cummax(0).values
    row = torch.arange(q.shape[1], device=q.device)
    inside = (row >= cu[0]) & (row < cu[-1])
    cut = lambda t: torch.where(inside.view(1, -1, *[1] * (t.dim() - 2)), t, 0)      # noqa: E731
    o, ht = call(*(cut(t) for t in (q, k, v, g, beta)), cu)
    return cut(o), ht


@torch.compiler.disable
def chunk_gated_delta(q, k, v, g, beta, scale=None, initial_state=None, output_final_state=False, use_qk_l2norm_in_kernel=False, cu_seqlens=None,
                      transpose_state_layout=False):
    """Whole sequences (prefill, training): `chunk_kda` with one decay per token and head.

    q, k [B,T,H,K]; v [B,T,HV,V]; g [B,T,HV] log-space decay (<= 0; -inf forgets the state) and beta [B,T,HV], in bfloat16 or float32; initial_state [N,HV,K,V]
    float32; cu_seqlens [N+1] with B == 1.  HV is a multiple of H (value head h reads q/k head h // (HV // H)).  Returns (o, final_state or None), differentiable
    with respect to q, k, v, g, beta and initial_state; gradients come in the types of their tensors.  Rows in front of the first sequence of cu_seqlens and behind
    the last one are zero, in o and in the gradients.  `transpose_state_layout`: states are [.., V, K] (turned by a copy in front of and behind the kernels).

    bfloat16 with K, V up to 128 takes the chunked tensor-core kernels (columns in multiples of 8 as they are, others zero-padded); final states and dh0 carry about
    1e-5 of their norm, which single bfloat16 operands would not give; the other gradients 3e-3, those of q and k per value head where heads are grouped.  bfloat16 with K = 256 runs forward only, token by token.  float32 runs token by
    token: forward for K in {32, 64, 128, 256}; with gradients (K, V in {32, 64, 128}) through `chunk_kda`, the decay spread over the key channels."""
    r = _native().chunk_delta(q, k, v, g, beta, initial_state, scale, output_final_state, cu_seqlens, use_qk_l2norm_in_kernel, transpose_state_layout, SCAN_SLICES)
    if r is not None:
        return r
    K, V = q.shape[-1], v.shape[-1]
    if scale is None:
        scale = K ** -0.5
    grads = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_state))
    if q.dtype == torch.float32 and grads:
        def per_channel(q, k, v, g, beta, cu):
            o, ht = ops.chunk_kda(q, k, v, g.unsqueeze(-1).expand(*g.shape, K), beta, scale=scale, initial_state=initial_state, output_final_state=output_final_state,
                                  use_qk_l2norm_in_kernel=use_qk_l2norm_in_kernel, cu_seqlens=cu, transpose_state_layout=transpose_state_layout)
            o.grad_fn.register_prehook(_no_second_derivative)      # (of the one node that o and ht come from)
            return o, ht
        return per_channel(q, k, v, g, beta, None) if cu_seqlens is None else _float32_packed(q, k, v, g, beta, cu_seqlens, per_channel)
    if q.dtype == torch.float32 or K > 128 or V > 128:
        if grads or (q.dtype != torch.float32 and K != 256):
            raise NotImplementedError(f"kda_b200: the bf16 chunked kernels are built for head sizes up to 128, got K={K}, V={V} (K = 256 runs forward-only)")
        return fused_recurrent_gated_delta(q, k, v, g, beta, scale=scale, initial_state=initial_state, output_final_state=output_final_state,
                                           use_qk_l2norm_in_kernel=use_qk_l2norm_in_kernel, cu_seqlens=cu_seqlens, transpose_state_layout=transpose_state_layout)
    # heads whose columns are no multiple of eight: zero columns change neither o nor the states' real part, nor any gradient
    pk, pv = -K % 8, -V % 8
    tr = (lambda t: t.transpose(-1, -2)) if transpose_state_layout else (lambda t: t)
    pad = torch.nn.functional.pad
    h0 = pad(tr(initial_state), (0, pv, 0, pk)) if initial_state is not None else None
    o, ht = _native().chunk_delta(pad(q, (0, pk)), pad(k, (0, pk)), pad(v, (0, pv)), g, beta, h0, scale, output_final_state, cu_seqlens, use_qk_l2norm_in_kernel, False,
                                  SCAN_SLICES)
    return o[..., :V], (tr(ht[..., :K, :V]) if ht is not None else None)
