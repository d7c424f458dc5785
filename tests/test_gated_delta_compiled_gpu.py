"""A layer of the package's operators inside torch.compile: the calls run as they are, between the pieces that are compiled, with the bits of the layer that is not."""
import pytest
import torch

from test_gated_delta_gpu import leave_no_memory      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def layer(x, res, w, wo, g, beta):
    from kda_b200 import chunk_gated_delta, gated_rms_norm, residual_rms_norm
    y, r = residual_rms_norm(x, res, w[0], scale=0.5, post_weight=w[1])
    h = y.view(*y.shape[:2], 2, 64)
    o, _ = chunk_gated_delta(h, h * 0.5, h + 1, g, beta, use_qk_l2norm_in_kernel=True)
    o = gated_rms_norm(o, h, wo, activation="silu").flatten(2) * 2
    return residual_rms_norm(o, r, w[2])


@pytest.mark.parametrize("grads", [False, True])
def test_a_compiled_layer(grads):
    gen = torch.Generator(device="cuda").manual_seed(5)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")      # noqa: E731
    leaves = [randn(2, 70, 128).to(BF), randn(2, 70, 128), randn(3, 128).to(BF), randn(64).to(BF), -torch.rand(2, 70, 2, generator=gen, device="cuda"), torch.sigmoid(randn(2, 70, 2))]
    leaves = [t.requires_grad_(grads) for t in leaves]
    gy, gr = randn(2, 70, 128).to(BF), randn(2, 70, 128)
    torch._dynamo.reset()
    compiled = torch.compile(layer, backend="eager")
    for _ in range(2):
        a, b = layer(*leaves), compiled(*leaves)
        assert all(torch.equal(s, t) for s, t in zip(a, b))
        if grads:
            ga, gb = (torch.autograd.grad(t, leaves, (gy, gr)) for t in (a, b))
            assert all(torch.equal(s, t) for s, t in zip(ga, gb))
    torch._dynamo.reset()
