"""Grouped value heads whose gradients of q and k nearly cancel.  Each head's dq, dk is rounded to bf16 before the group's sum (csrc/delta_api.cu), so the error is
one of the terms, not of the sum: a head's own gradient is good to 4 * 2^-8 (test_gated_delta_gpu.py: that with its rounding), and the sum, taken in float32, rounds once more."""
import pytest
import torch

from test_gated_delta_gpu import GRAD, leave_no_memory, make, reference, run      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grp", [2, 4])
@pytest.mark.parametrize("norm", [False, True])
def test_heads_of_a_group_that_cancel(grp, norm):
    H = 2
    d = make(2, 150, H, H * grp, 128, 128, seed=grp, normed=not norm)
    for n in ("v", "g", "beta", "do"):      # a group's heads see the same sequence, every other one with the gradients' sign turned
        first = d[n].view(2, 150, H, grp, *d[n].shape[3:])[:, :, :, :1]
        d[n] = first.expand(2, 150, H, grp, *d[n].shape[3:]).reshape(d[n].shape).clone()
    for n in ("h0", "dht"):
        d[n] = d[n].view(2, H, grp, 128, 128)[:, :, :1].expand(2, H, grp, 128, 128).reshape(2, H * grp, 128, 128).clone()
    turn = torch.tensor([1.0, -1.0]).repeat(H * grp // 2)
    near = 1 + turn.clamp(max=0).abs() * 2.0 ** -6      # (1 + 2^-6 is a bf16 number)
    d["do"] = (d["do"].float() * (turn * near)[:, None]).bfloat16()
    d["dht"] = d["dht"] * (turn * near)[:, None, None]
    kw = dict(use_qk_l2norm_in_kernel=True) if norm else {}
    got, ref = run(d, **kw), reference(d, use_qk_l2norm=norm)
    spread = {n: (t.repeat_interleave(grp, 2) if n in ("q", "k") else t) for n, t in d.items()}
    terms = reference(spread, use_qk_l2norm=norm)      # a q and a k of its own for every value head
    for n in ("dq", "dk"):
        t = terms[n].reshape(*terms[n].shape[:2], H, grp, 128)
        assert torch.allclose(t.sum(3), ref[n], rtol=1e-9, atol=1e-12)
        size = sum(float(x.norm()) for x in t.unbind(3))
        off = float((got[n].double() - ref[n]).norm())
        print(n, off / size, float(ref[n].norm()) / size)
        assert float(ref[n].norm()) < size / 16      # they do cancel
        assert off <= GRAD * size + 2.0 ** -8 * float(ref[n].norm())
