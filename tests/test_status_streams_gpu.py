"""Reading a status word waits for the work in front of it on every stream: torch's side streams do not wait for the default one, nor it for them."""
import pytest
import torch

from test_gated_delta_gpu import leave_no_memory, make      # noqa: F401  (the fixture)
from test_status_gpu import _debug_lib

pytestmark = pytest.mark.gpu
LONG = 400_000_000      # clock cycles, about 0.2 s


@pytest.mark.parametrize("what", ["norm", "recurrent", "chunk"])
def test_the_word_is_read_behind_work_on_a_side_stream(what):
    from kda_b200 import _lib
    read = dict(norm=_lib.norm_status, recurrent=_lib.recurrent_status, chunk=lambda: _lib.chunk_status(ws.data_ptr()))[what]
    ws = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    read()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(LONG)
    assert read() == 0 and s.query()


def test_a_wait_that_gave_up_on_a_side_stream_is_seen():
    from kda_b200 import _lib
    ws = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert _debug_lib().kda_b200_debug_wait_giveup(ws.data_ptr(), 0x8, s.cuda_stream) == 0
    assert _lib.chunk_status(ws.data_ptr()) == 0x8


def test_checked_mode_reports_a_call_on_a_side_stream():
    from kda_b200 import _lib, chunk_gated_delta
    d = {n: t.cuda() for n, t in make(1, 10, 1, 1, 64, 64, seed=65).items()}
    cu = torch.tensor([0, 400], dtype=torch.int32, device="cuda")
    torch.zeros(1 << 20, device="cuda")      # (what the call's workspace is made of)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.zeros(1 << 20, device="cuda")
        torch.cuda._sleep(LONG)
        with pytest.raises(_lib.KdaError, match="cu_seqlens"):
            chunk_gated_delta(*[d[n] for n in ("q", "k", "v", "g", "beta")], cu_seqlens=cu)
    torch.cuda.synchronize()
