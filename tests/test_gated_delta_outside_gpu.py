"""Rows that belong to no sequence of a packed call (in front of the first, behind the last, or all of them where there is no sequence): o and the gradients
are zero there, on every path that a call can take, whatever stood in the memory."""
import pytest
import torch

from test_gated_delta_gpu import leave_no_memory, make, run      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
PATHS = [(128, 128, BF), (64, 64, BF), (20, 37, BF)]


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
