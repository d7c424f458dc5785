"""The decode call with one decay per head: the decay that a state is multiplied with, and beta, to float32's rounding over the range of a layer's raw values.

Bound, relative, element by element.  exp(g): the exponential 2^-22, its argument's rest 2^-23; the product with the state 2^-24.  g = -exp(A_log) softplus(x) is itself off by
2^-21 of its value (exp(A_log) 2^-22, log1p 2^-23, products), which the exponential turns into |g| 2^-21; with a lower bound 2^-21 too, and its argument's error, 2^-22 of
|exp(A_log) x|, falls behind sigmoid.  2^-21 (1 + 2 |g|) together."""
import numpy as np
import pytest
import torch

from _abi import bulk_decode_batch
from test_gated_delta_gpu import leave_no_memory      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16


def call(x, A, bias, beta, lower, h0, tr, K, v=None):
    from kda_b200 import fused_recurrent_gated_delta
    N, HV = x.shape
    q = torch.zeros(N, 1, 1, K, device="cuda", dtype=BF)
    k = q.clone()
    k[..., 0] = 1
    v = torch.zeros(N, 1, HV, 128, device="cuda", dtype=BF) if v is None else v
    h = h0.transpose(-1, -2).contiguous() if tr else h0
    _, ht = fused_recurrent_gated_delta(q, k, v, x[:, None], beta[:, None], A_log=A, dt_bias=bias, initial_state=h, output_final_state=True, use_gate_in_kernel=True,
                                        use_beta_sigmoid_in_kernel=True, lower_bound=lower, transpose_state_layout=tr)
    return ht.transpose(-1, -2) if tr else ht


def sizes(which):
    N, HV = (6, 8) if which == "few" else bulk_decode_batch()      # few warps, and whole states in shared memory
    return N, HV


@pytest.mark.parametrize("which", ["few", "many"])
@pytest.mark.parametrize("tr", [False, True])
@pytest.mark.parametrize("lower", [None, -5.0])
@pytest.mark.parametrize("gate_dtype", [F32, BF])
def test_decay(which, tr, lower, gate_dtype):
    N, HV = sizes(which)
    gen = torch.Generator(device="cuda").manual_seed(1)
    A, bias = torch.log(torch.linspace(1.0, 16.0, HV, device="cuda")), torch.linspace(-7.0, -2.0, HV, device="cuda")
    x = (torch.linspace(-9, 5, N * HV, device="cuda").view(HV, N).T + torch.randn(N, HV, generator=gen, device="cuda")).to(gate_dtype).contiguous()
    beta = torch.full((N, HV), -1e4, device="cuda", dtype=gate_dtype)      # nothing is written
    h0 = torch.rand(N, HV, 128, 128, generator=gen, device="cuda") + 0.5
    ht = call(x, A, bias, beta, lower, h0, tr, 128)
    y, a = (x.float() + bias).double(), A.double().exp()      # (the raw value and its bias are added in float32)
    g = lower / (1 + torch.exp(-a * y)) if lower is not None else -a * torch.where(y > 30, y, torch.log1p(y.clamp(max=30).exp()))
    want = h0.double() * g.exp()[..., None, None]
    off = ((ht.double() - want).abs() / want).amax((-1, -2))
    room = 2.0 ** -21 * (1 + 2 * g.abs())
    print(float((off / room).max()))
    assert (off <= room)[want.amin((-1, -2)) > 2.0 ** -120].all()


@pytest.mark.parametrize("which", ["few", "many"])
def test_beta(which):
    """An empty state behind one token: row 0 is beta v."""
    N, HV = sizes(which)
    logits = torch.linspace(-30, 10, N * HV, device="cuda").view(N, HV)
    v = torch.ones(N, 1, HV, 128, device="cuda", dtype=BF)
    zero = torch.zeros(HV, device="cuda")
    ht = call(torch.zeros(N, HV, device="cuda"), zero, zero, logits, None, torch.zeros(N, HV, 128, 128, device="cuda"), False, 128, v)
    want = torch.sigmoid(logits.double())
    off = (ht[:, :, 0].double() - want[..., None]).abs().amax(-1) / want
    assert float(off.max()) <= 2.0 ** -21, float(off.max())
    assert not ht[:, :, 1:].any()


@pytest.mark.parametrize("which", ["few", "many"])
def test_ends_of_the_range(which):
    N, HV = sizes(which)
    x = torch.tensor([float("-inf"), -1e30, -200.0, 200.0, 1e30, float("inf"), float("nan"), 0.0], device="cuda").repeat(N * HV // 8 + 1)[:N * HV].view(N, HV)
    zero = torch.zeros(HV, device="cuda")
    h0 = torch.ones(N, HV, 128, 128, device="cuda")
    ht = call(x, zero, zero, torch.full((N, HV), -float("inf"), device="cuda"), None, h0, False, 128)
    want = torch.tensor([1.0, 1.0, 1.0, 0.0, 0.0, 0.0, np.nan, 0.5], device="cuda").repeat(N * HV // 8 + 1)[:N * HV].view(N, HV)
    got = ht.amax((-1, -2))
    assert torch.equal(got.isnan(), want.isnan()) and torch.allclose(got, want, rtol=2.0 ** -20, atol=2.0 ** -120, equal_nan=True)
