"""Derivatives that the gated delta rule does not have are refused on every path of a call, not dropped: forward-mode tangents, and gradients of gradients."""
import pytest
import torch
from torch.autograd import forward_ad

from test_gated_delta_gpu import leave_no_memory, make      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAMES = ("q", "k", "v", "g", "beta", "h0")


def inputs(K, V, dtype):
    return {n: t.cuda() for n, t in make(1, 40, 1, 2, K, V, seed=K, dtype=dtype).items()}


@pytest.mark.parametrize("K,V,dtype", [(64, 64, BF), (20, 12, BF), (256, 64, BF), (64, 64, F32), (256, 32, F32)])
@pytest.mark.parametrize("which", NAMES)
def test_a_tangent_is_refused(K, V, dtype, which):
    from kda_b200 import chunk_gated_delta, fused_recurrent_gated_delta
    x = inputs(K, V, dtype)
    with forward_ad.dual_level():
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        args = [x[n] for n in NAMES[:5]]
        with pytest.raises(NotImplementedError, match="jvp"):
            chunk_gated_delta(*args, initial_state=x["h0"])
        if K % 32 == 0:
            with pytest.raises(NotImplementedError, match="jvp"):
                fused_recurrent_gated_delta(*args, initial_state=x["h0"])


def test_inference_mode_has_none():
    from kda_b200 import chunk_gated_delta, fused_recurrent_gated_delta
    with torch.inference_mode():
        x = inputs(64, 64, BF)
        args = [x[n] for n in NAMES[:5]]
        a, b = chunk_gated_delta(*args, initial_state=x["h0"])[0], fused_recurrent_gated_delta(*args, initial_state=x["h0"])[0]
        assert float((a.double() - b.double()).norm()) <= 2.0 ** -6 * float(a.double().norm())
@pytest.mark.parametrize("tr", [False, True])
@pytest.mark.parametrize("K,V,dtype", [(64, 64, BF), (20, 12, BF), (64, 64, F32)])
@pytest.mark.parametrize("which", ["o", "ht", "both"])
def test_a_gradients_gradient_is_refused(K, V, dtype, which, tr):
    from kda_b200 import chunk_gated_delta
    x = inputs(K, V, dtype)
    x["v"].requires_grad_()
    h0 = x["h0"].transpose(-1, -2).contiguous() if tr else x["h0"]
    o, ht = chunk_gated_delta(*[x[n] for n in NAMES[:5]], initial_state=h0, output_final_state=True, transpose_state_layout=tr)
    outs = {"o": (o,), "ht": (ht,), "both": (o, ht)}[which]
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(outs, x["v"], [torch.ones_like(t) for t in outs], create_graph=True)
    o, ht = chunk_gated_delta(*[x[n] for n in NAMES[:5]], initial_state=h0, output_final_state=True, transpose_state_layout=tr)
    (dv,) = torch.autograd.grad((o, ht), x["v"], (torch.ones_like(o), torch.ones_like(ht)))      # once it is there
    assert dv.any()
