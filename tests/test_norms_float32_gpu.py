"""The gated norm on float32 tensors: its activation and that one's slope to float32, element by element, over all of the gate's range.

Bound, relative to each element.  sigmoid(z) = 1 / (1 + exp(-z)): the exponential 2^-22 and its argument's rest 2^-23, the sum 2^-24 and the reciprocal 2^-23; 1 - sigmoid(z) one
product more.  1 / rms(x): a sum of 128 squares in at most 16 steps of 2^-24, halved by the root, and a root of 2^-22.  Four products of 2^-24 behind them: 2^-20 together.  Where the
result is a sum of two such terms (the slope of z sigmoid(z), dx) the bound is of their absolute values.  Results below 2^-126 are no normal numbers and count as zero."""
import pytest
import torch

from test_norms_gpu import gated_ref, leave_no_memory      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -20


def off(got, ref, size):
    return float(((got.double() - ref).abs() / (size + 2.0 ** -126 / TOL)).max())


@pytest.mark.parametrize("rows", [40, 70000])      # straight from memory, and through shared memory
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_activation(rows, act):
    from kda_b200 import gated_rms_norm
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.rand(rows, 128, generator=gen, device="cuda") + 0.5).requires_grad_()
    z = (torch.linspace(-86, 86, rows * 128, device="cuda").view(128, rows).T + torch.rand(rows, 128, generator=gen, device="cuda")).contiguous().requires_grad_()
    dy = torch.rand(rows, 128, generator=gen, device="cuda") + 0.5
    y = gated_rms_norm(x, z, activation=act)
    dx, dz = torch.autograd.grad(y, (x, z), dy)
    X, Z = x.detach().double(), z.detach().double()
    s, c = 1 / (1 + torch.exp(-Z)), 1 / (1 + torch.exp(Z))
    n = X * (X.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()
    a = Z * s if act == "silu" else s
    e = off(y.detach(), n * a, (n * a).abs())
    assert e <= TOL, e
    slope, size = (s * (1 + Z * c), s * (1 + (Z * c).abs())) if act == "silu" else (s * c, s * c)
    e = off(dz, dy.double() * n * slope, (dy.double() * n * size).abs())
    assert e <= TOL, e


def test_ends_of_the_range():
    """Infinities and NaN in the gate, and what is beyond the exponential's range: sigmoid's limits."""
    from kda_b200 import gated_rms_norm
    x = torch.ones(8, 16, device="cuda")
    z = torch.tensor([float("inf"), 1e30, 200.0, 90.0, -90.0, -200.0, -1e30, float("nan")], device="cuda")[:, None].expand(8, 16).contiguous()
    z.requires_grad_()
    y = gated_rms_norm(x, z, eps=0.0)
    (dz,) = torch.autograd.grad(y, z, torch.ones_like(y))
    assert (y[:4] == 1).all() and (y[4:7].abs() < 1e-37).all() and y[7].isnan().all()
    assert (dz[:7].abs() < 1e-37).all() and dz[7].isnan().all()
    assert torch.equal(gated_rms_norm(x, torch.full_like(x, -float("inf")), eps=0.0), torch.zeros_like(x))
