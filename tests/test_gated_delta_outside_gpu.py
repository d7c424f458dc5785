"""Rows that belong to no sequence of a packed call (in front of the first, behind the last, or all of them where there is no sequence): o and the gradients
are zero there, on every path that a call can take, whatever stood in the memory."""
import pytest
import torch

from test_gated_delta_gpu import leave_no_memory, make, run      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
PATHS = [(128, 128, BF), (64, 64, BF), (20, 37, BF), (64, 64, F32), (128, 32, F32)]


def poison():
    """fills what the allocator hands out next with NaN"""
    for n in (1 << 10, 1 << 14, 1 << 18, 1 << 22):
        blocks = [torch.full((n,), float("nan"), device="cuda") for _ in range(16)]
        del blocks


@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("K,V,dtype", PATHS)
def test_no_sequence_at_all(K, V, dtype, grads):
    d = make(1, 70, 2, 4, K, V, seed=1, h0=False, dtype=dtype)
    d["dht"] = d["dht"][:0]
    poison()
    got = run(d, cu=torch.zeros(1, dtype=torch.int32, device="cuda"), grads=grads)
    assert got["ht"].shape == (0, 4, K, V)
    for n in ("o", "dq", "dk", "dv", "dg", "dbeta") if grads else ("o",):
        assert got[n].shape[1] == 70 and not got[n].any(), n


@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("K,V,dtype", PATHS)
def test_in_front_and_behind(K, V, dtype, grads):
    d = make(1, 200, 2, 4, K, V, seed=2, n_states=2, dtype=dtype)
    if not grads:      # neither are these rows read
        for n in ("q", "k", "v", "g", "beta"):
            d[n][:, :10] = d[n][:, 170:] = float("nan")
    poison()
    got = run(d, cu=torch.tensor([10, 60, 170], dtype=torch.int32, device="cuda"), grads=grads)
    one = run({n: (t[:, 10:60] if n not in ("h0", "dht") else t[:1]) for n, t in d.items()}, grads=grads)
    for n in ("o", "dq", "dk", "dv", "dg", "dbeta") if grads else ("o",):
        assert not got[n][:, :10].any() and not got[n][:, 170:].any(), n
        assert (got[n][:, 10:170] != 0).any() and torch.isfinite(got[n].float()).all(), n
        if dtype == BF:
            assert torch.equal(got[n][:, 10:60], one[n]), n


@pytest.mark.parametrize("K,V,dtype,tr", [(64, 64, BF, False), (128, 128, BF, True), (256, 32, BF, False), (32, 96, F32, False), (64, 32, F32, True)])
@pytest.mark.parametrize("cu", [[10, 60, 170], [0, 0, 170], [200, 200], [0], [0, 200], [3, 50, 51, 51, 90, 137]])
def test_token_by_token(K, V, dtype, tr, cu):
    from kda_b200 import fused_recurrent_gated_delta
    d = {n: t.cuda() for n, t in make(1, 200, 2, 4, K, V, seed=3, h0=False, dtype=dtype).items() if t is not None}
    poison()
    o, _ = fused_recurrent_gated_delta(d["q"], d["k"], d["v"], d["g"], d["beta"], cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), transpose_state_layout=tr)
    assert not o[:, :cu[0]].any() and not o[:, cu[-1]:].any() and (o[:, cu[0]:cu[-1]].any() or cu[0] == cu[-1])


def test_a_servers_padded_output():
    """Decode into a caller's buffer, packed: the rows behind the last sequence become zero too, and a call without one zeroes all."""
    from kda_b200 import fused_recurrent_gated_delta_fwd
    d = {n: t.cuda() for n, t in make(1, 12, 2, 2, 128, 128, seed=4, h0=False).items() if t is not None}
    pool = torch.randn(9, 2, 128, 128, device="cuda")
    args = [d[n] for n in ("q", "k", "v", "g", "beta")]
    slots = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    out = torch.full_like(d["v"], float("nan"))
    fused_recurrent_gated_delta_fwd(*args, initial_state=pool, cu_seqlens=torch.tensor([0, 3, 7], dtype=torch.int32, device="cuda"), ssm_state_indices=slots, out=out)
    assert out[:, :7].isfinite().all() and out[:, :7].any() and not out[:, 7:].any()
    before = pool.clone()
    out = torch.full_like(d["v"], float("nan"))
    fused_recurrent_gated_delta_fwd(*args, initial_state=pool, cu_seqlens=torch.zeros(1, dtype=torch.int32, device="cuda"), ssm_state_indices=slots[:0], out=out)
    assert not out.any() and torch.equal(pool, before)


@pytest.mark.parametrize("tr", [False, True])
def test_a_padded_entry_and_padded_rows(tr):
    """A packed decode call of four sequences, two of them padded entries, in a buffer that is much larger than their tokens."""
    from kda_b200 import fused_recurrent_gated_delta_fwd
    d = {n: t.cuda() for n, t in make(1, 1000, 2, 2, 64, 64, seed=6, h0=False).items() if t is not None}
    cu, slots = torch.tensor([5, 8, 10, 13, 14], dtype=torch.int32, device="cuda"), torch.tensor([[0, 1, 2], [-1, 3, 3], [4, 5, 6], [9, 9, 9]], dtype=torch.int32, device="cuda")
    pool = torch.randn(8, 2, 64, 64, device="cuda")
    out = torch.full_like(d["v"], float("nan"))
    fused_recurrent_gated_delta_fwd(*[d[n] for n in ("q", "k", "v", "g", "beta")], initial_state=pool, cu_seqlens=cu, ssm_state_indices=slots, out=out, transpose_state_layout=tr)
    there = torch.zeros(1000, dtype=torch.bool, device="cuda")
    there[5:8] = there[10:13] = True
    assert out[:, there].isfinite().all() and out[:, there].abs().sum((0, 2, 3)).all() and not out[:, ~there].any()


@pytest.mark.parametrize("cu", [[0, 400], [-64, 70], [50, 20, 70], [90, 100]])
def test_float32_offsets_beyond_the_tensors(cu):
    """Training in float32 with offsets that do not fit: they are cut to the tensors, and rows outside come out as zeros."""
    from kda_b200 import chunk_gated_delta
    d = make(1, 70, 2, 2, 64, 64, seed=5, h0=False, dtype=F32)
    x = {n: d[n].cuda().requires_grad_() for n in ("q", "k", "v", "g", "beta")}
    o, _ = chunk_gated_delta(*x.values(), cu_seqlens=torch.tensor(cu, device="cuda"))
    grads = torch.autograd.grad(o, list(x.values()), torch.ones_like(o))
    inside = torch.zeros(70, dtype=torch.bool)
    inside[max(0, cu[0]):max(0, *cu)] = True
    for t in (o, *grads):
        assert torch.isfinite(t).all() and not t[:, ~inside.cuda()].any()
