"""The norms' kernel for many rows when a wait gives up: the warps of a row meet in barriers, so one that left alone would keep the others there.  The kernel comes to its end, its
status word says that results are missing, and the rows of the other CTAs are right.  One warp's verdict is handed in
(csrc/debug/kda_norm_ring_test.cu); its CTA's other waits then run out by themselves, after a second or two."""
import ctypes as C

import pytest
import torch

from test_gated_delta_gpu import leave_no_memory      # noqa: F401  (the fixture)
from test_norms_gpu import BF, gated_ref
from test_status_gpu import _debug_lib

pytestmark = pytest.mark.gpu
NONE = -1


def call(x, z, dy, cta, warp, turn):
    """(outputs, status) of the debug build's kernel"""
    from kda_b200 import _lib
    lib = _debug_lib()
    lib.kda_b200_debug_ring_lost.argtypes = [C.POINTER(_lib.NormArgs), C.c_int, C.c_int, C.c_int, C.c_void_p, C.POINTER(C.c_uint32), C.c_void_p]
    rows, cols = x.shape
    out = [torch.zeros_like(x) for _ in range(2 if dy is not None else 1)]
    partial = torch.zeros(256, cols, device="cuda") if dy is not None else None
    a = _lib.NormArgs(x=x.data_ptr(), gate=z.data_ptr(), rows=rows, cols=cols, io_dtype=_lib.KDA_BF16, gate_dtype=_lib.KDA_BF16, weight_dtype=_lib.KDA_BF16, eps=1e-6)
    if dy is None:
        a.y = out[0].data_ptr()
    else:
        a.dy, a.dx, a.dgate = dy.data_ptr(), out[0].data_ptr(), out[1].data_ptr()
    status = C.c_uint32(0)
    torch.cuda.synchronize()
    assert lib.kda_b200_debug_ring_lost(C.byref(a), cta, warp, turn, partial.data_ptr() if partial is not None else None, C.byref(status), torch.cuda.current_stream().cuda_stream) == 0
    return out, status.value


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("cols", [128, 1000, 2048, 8192])      # a row's threads: part of a warp, 2 warps, 4, 16
@pytest.mark.parametrize("warp,turn", [(0, 0), (1, 2)])
def test_one_warps_wait_gives_up(cols, backward, warp, turn):
    rows = (1 << 25) // cols
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x, z, dy = (torch.randn(rows, cols, generator=gen, device="cuda").to(BF) for _ in range(3))
    dy = dy if backward else None
    good, status = call(x, z, dy, 0, NONE, 0)
    assert status == 0
    lost, status = call(x, z, dy, 5, warp, turn)
    assert status == 1
    wrong = torch.stack([(a != b).any(1) for a, b in zip(good, lost)]).any(0)
    assert int(wrong.sum()) <= (rows + 147) // 148 + 512      # no more than one CTA's share, in whole stages
    again, status = call(x, z, dy, 0, NONE, 0)
    assert status == 0 and all(torch.equal(a, b) for a, b in zip(good, again))
    if not backward:
        ref = gated_ref(x[:64].double(), z[:64].double(), None, 1e-6, "sigmoid")
        assert float((good[0][:64].double() - ref).norm()) <= 2.0 ** -7 * float(ref.norm())
