"""The gradient of the decays, token by token and head by head, where most of the sums it is made of cancel.

With f and v_new of a chunk with start state h and gradient dh of the state behind it (csrc/delta.cuh), dg_t is a sum over what crosses from the tokens in front of t
to those from t on:
    dg_t = sum over i >= t > j of (E_ij k_i k_j + F_ij q_i k_j)  +  sum over i >= t of (scale Gam_i q_i (dO_i h^T) - beta_i Gam_i k_i (f_i h^T))
           + sum over j < t of w_j k_j (v_new_j dh^T)  +  Gam_last <h, dh>,           E_ij = -beta_i D_ij f_i v_new_j,  F_ij = scale D_ij dO_i v_new_j
The kernel takes it as a sum of all rows' products with their own gradients, in which a pair (i, j) on one side of t stands twice with opposite signs.  Both have
the same rounded E_ij or F_ij, so they cancel up to float32.

Bound.  Of what crosses, a term of E has three roundings to bf16 (f, v_new, E), one of F two, the others two of an operand each: 3 * 2^-8, and 2^-12 for the decays
(arguments up to 150 in float32).  Everything, crossing or not, passes float32 sums: at most 128 products in a tensor core, whose steps are off by at most 2^-23,
and some 50 steps of 2^-24 behind it: 2^-15 of the sum of the absolute products."""
import pytest
import torch

from oracle.kda_oracle import recurrent_kda, rel_l2_err
from test_gated_delta_gpu import GRAD, leave_no_memory, make, reference, run      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def dg_bound(d):
    x = {n: t.cuda().double() for n, t in d.items()}
    B, T, H, K = x["q"].shape
    scale, S, starts = K ** -0.5, x["h0"], []
    step = lambda S, a, b: recurrent_kda(x["q"][:, a:b], x["k"][:, a:b], x["v"][:, a:b], x["g"][:, a:b].unsqueeze(-1).expand(B, b - a, H, K), x["beta"][:, a:b],      # noqa: E731
                                         initial_state=S, output_final_state=True)
    for a in range(0, T, 64):
        starts.append(S)
        S = step(S, a, min(T, a + 64))[1]
    dh, out = x["dht"], torch.zeros_like(x["g"])
    for a in reversed(range(0, T, 64)):
        b = min(T, a + 64)
        q, k, v, do, g, beta = (x[n][:, a:b].transpose(1, 2) for n in ("q", "k", "v", "do", "g", "beta"))
        h, n = starts[a // 64], b - a
        G = g.cumsum(-1)
        low = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        D = torch.where(low, (G.unsqueeze(-1) - G.unsqueeze(-2)).masked_fill(~low, 0).exp(), 0.0)
        T2 = lambda t: t.transpose(-1, -2)      # noqa: E731
        kk, qk = k @ T2(k), q @ T2(k)
        bt, gam, w = beta.unsqueeze(-1), G.exp().unsqueeze(-1), (G[..., -1:] - G).exp().unsqueeze(-1)
        Tm = torch.linalg.inv(torch.eye(n, device="cuda", dtype=torch.float64) + (bt * D * kk).tril(-1))
        vn = Tm @ (bt * (v - gam * (k @ h)))
        f = T2(Tm) @ (T2(scale * D * qk) @ do + w * (k @ dh))
        E, F = (bt * D * (f.abs() @ T2(vn.abs()))).tril(-1), scale * D * (do.abs() @ T2(vn.abs()))
        M = E * kk.abs() + F * qk.abs()
        z = (w * k.abs() * (vn.abs() @ T2(dh.abs()))).sum(-1)
        y = (gam * (bt * k.abs() * (f.abs() @ T2(h.abs())) + scale * q.abs() * (do.abs() @ T2(h.abs())))).sum(-1)
        last = gam[..., -1, 0] * (h * dh).abs().sum((-1, -2))
        behind = lambda t: t.flip(-1).cumsum(-1).flip(-1)      # noqa: E731
        pairs = (M.flip(-2).cumsum(-2).flip(-2) * low.tril(-1)).sum(-1)      # over i >= t > j
        crossing = pairs + behind(y) + (z.cumsum(-1) - z) + last.unsqueeze(-1)
        products = E * (k.abs() @ T2(k.abs())) + F * (q.abs() @ T2(k.abs()))
        everything = behind(products.sum(-1) + products.sum(-2) + y + z) + (z.sum(-1) + last).unsqueeze(-1)
        out[:, a:b] = ((3 * 2.0 ** -8 + 2.0 ** -12) * crossing + 2.0 ** -15 * everything).transpose(1, 2)
        leaf = h.detach().requires_grad_()
        o, end = step(leaf, a, b)
        (dh,) = torch.autograd.grad((o, end), leaf, (x["do"][:, a:b], dh))
    return out


def check(d, **kw):
    got, ref, bound = run(d, **kw)["dg"].double(), reference(d)["dg"], dg_bound(d)
    off = (got - ref).abs()
    print("share of the bound", float((off / bound).max()), "largest dg in bounds", float((ref.abs() / bound).max()))
    assert (off <= bound).all()
    return got, ref, bound


def heads(t):
    return t.transpose(1, 2).flatten(2).unbind(1)


@pytest.mark.parametrize("slices", [1, 2, 4])
@pytest.mark.parametrize("mild", [0.01, 1.0, 30.0])
def test_every_heads_decay(mild, slices):
    """Slow, ordinary and quick decays (30: 200 tokens of which each all but forgets the one before): every head's gradient within the tolerance of the other gradients,
    which a lost or wrong term in any of them fails."""
    got, ref, bound = check(make(1, 200, 4, 4, 128, 128, seed=21, mild=mild), slices=slices)
    for h, (a, b, c) in enumerate(zip(heads(got), heads(ref), heads(bound))):
        assert rel_l2_err(a, b) <= GRAD, h
        # where few tokens count, the bound on each token tells as well (where many do, the absolute products that it counts are far above their sum)
        assert mild < 30 or (b.abs() > c).any(), h


def test_decays_that_leave_nothing():
    """Behind decays of exp(-150) on average dg is a number below float32's noise in the sums it is taken from."""
    check(make(1, 200, 4, 4, 128, 128, seed=21, mild=3000.0))


@pytest.mark.parametrize("K,V", [(64, 64), (8, 128), (20, 37), (1, 1)])
def test_head_sizes(K, V):
    """(1, 1: every key is the same up to its sign and overwrites the state, and the terms cancel; the other sizes have their norm checked beside the other gradients)"""
    got, ref, bound = check(make(1, 100, 2, 2, K, V, seed=K * 7 + V))
    assert rel_l2_err(got, ref) <= GRAD if K > 1 else (ref.abs() > bound).any()


def test_no_decay():
    got, ref, bound = check(make(1, 150, 2, 2, 128, 128, seed=21, mild=0.0))
    assert rel_l2_err(got, ref) <= GRAD


def test_a_gradient_of_zeros_is_found():
    """What these checks are worth: quick decays, where test_gated_delta_gpu.py has its own bound alone."""
    d = make(1, 200, 4, 4, 128, 128, seed=21, mild=30.0)
    ref, bound = reference(d)["dg"], dg_bound(d)
    for h in range(4):
        nothing = ref.clone()
        nothing[:, :, h] = 0
        assert rel_l2_err(nothing[:, :, h], ref[:, :, h]) > GRAD and ((nothing - ref).abs() > bound)[:, :, h].any()
