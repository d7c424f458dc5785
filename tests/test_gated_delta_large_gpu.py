"""Offsets beyond 32 bits: rows, pools and packed sequences whose last elements lie behind 2^31 elements or bytes give what the same numbers give on their own."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def leave_no_memory():
    gc.collect()
    torch.cuda.empty_cache()
    yield
    gc.collect()
    torch.cuda.empty_cache()


def fill(*shape):
    return torch.empty(*shape, dtype=BF, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(sum(shape)))


@pytest.mark.parametrize("cols", [128, 77])
def test_norms_of_many_rows(cols):
    from kda_b200 import gated_rms_norm, residual_rms_norm
    rows, last = 2 ** 31 // cols + 1001, 1000
    w = fill(cols)
    x, z, d = (fill(rows, cols).requires_grad_(i < 2) for i in range(3))
    tail = [t[-last:].detach().clone().requires_grad_(t.requires_grad) for t in (x, z, d)]
    for f in (lambda a, b: gated_rms_norm(a, b, w), lambda a, b: residual_rms_norm(a, b, w, post_weight=w)[0]):
        y, y1 = f(x, z), f(*tail[:2])
        assert torch.equal(y[-last:], y1) or (y[-last:].float() - y1.float()).norm() <= 2.0 ** -8 * y1.float().norm()
        g, g1 = torch.autograd.grad(y, [x, z], d), torch.autograd.grad(y1, tail[:2], tail[2])
        for a, b in zip(g, g1):      # (other kernels for other sizes: their sums round in another order, in front of one rounding to bf16)
            assert (a[-last:].float() - b.float()).norm() <= 2.0 ** -8 * b.float().norm()
        del y, y1, g, g1


def test_a_packed_call_of_many_tokens():
    from kda_b200 import chunk_gated_delta
    H, D, last = 32, 128, 100
    T = 2 ** 31 // (H * D) + 200
    q, k, v, do = (fill(1, T, H, D) for _ in range(4))
    g = -torch.rand(1, T, H, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    beta = torch.rand(1, T, H, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    cu = torch.tensor([0, 70, *range(4096, T - last - 4096, 4096), T - last, T], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v, g, beta)]
    o, ht = chunk_gated_delta(*leaves, use_qk_l2norm_in_kernel=True, output_final_state=True, cu_seqlens=cu)
    grads = torch.autograd.grad(o, leaves, do)
    part = [t.detach()[:, -last:].clone().requires_grad_() for t in leaves]
    o1, ht1 = chunk_gated_delta(*part, use_qk_l2norm_in_kernel=True, output_final_state=True)
    g1 = torch.autograd.grad(o1, part, do[:, -last:])
    rel = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())      # noqa: E731
    assert rel(o[:, -last:], o1) <= 2.0 ** -8 and rel(ht[-1:], ht1) <= 2.0 ** -13
    for a, b in zip(grads, g1):
        assert rel(a[:, -last:], b) <= 4 * 2.0 ** -8


@pytest.mark.parametrize("N,T", [(2, 1), (150, 1), (40, 2)])      # the per-warp kernel, whole states, half states
def test_decode_from_a_large_pool(N, T):
    from kda_b200 import fused_recurrent_gated_delta_fwd
    H, D = 32, 128
    S = 2 ** 31 // (H * D * D) + 2 * N * T
    pool = torch.zeros(S, H, D, D, device="cuda")
    slots = (S - 1 - torch.arange(N * T, device="cuda").view(N, T)).int()
    near = torch.zeros(N * T, H, D, D, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(3))
    pool[slots.flatten().long()] = near
    q, k, v = (fill(N, T, H, D) for _ in range(3))
    g, beta = -torch.rand(N, T, H, device="cuda"), torch.rand(N, T, H, device="cuda")
    index = torch.arange(N * T, device="cuda", dtype=torch.int32).view(N, T)
    one = (lambda t: t[:, 0]) if T == 1 else (lambda t: t)
    a, _ = fused_recurrent_gated_delta_fwd(q, k, v, g, beta, initial_state=pool, ssm_state_indices=one(slots), use_qk_l2norm_in_kernel=True)
    b, _ = fused_recurrent_gated_delta_fwd(q, k, v, g, beta, initial_state=near, ssm_state_indices=one(index), use_qk_l2norm_in_kernel=True)
    assert torch.equal(a, b) and torch.equal(pool[slots.flatten().long()], near)
    assert not pool[: S - N * T].any()


def test_backward_twice_through_one_forward():
    from kda_b200 import chunk_gated_delta, gated_rms_norm
    x = [fill(2, 130, 2, 64).requires_grad_() for _ in range(3)]
    g = (-torch.rand(2, 130, 2, device="cuda")).requires_grad_()
    o, ht = chunk_gated_delta(*x, g, torch.rand(2, 130, 2, device="cuda"), use_qk_l2norm_in_kernel=True, output_final_state=True)
    y = gated_rms_norm(o, x[2])
    first = torch.autograd.grad((y, ht), [*x, g], (torch.ones_like(y), torch.ones_like(ht)), retain_graph=True)
    again = torch.autograd.grad((y, ht), [*x, g], (torch.ones_like(y), torch.ones_like(ht)))
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    # an expanded gradient (a sum's) and a missing one
    o, ht = chunk_gated_delta(*x, g, torch.rand(2, 130, 2, device="cuda"), output_final_state=True)
    assert all(torch.isfinite(t).all() for t in torch.autograd.grad(ht.sum(), [x[1], x[2], g]))
