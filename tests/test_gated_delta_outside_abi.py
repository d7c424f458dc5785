"""CPU tests of calls of the gated delta rule without any sequence: what they write has to be there."""
import ctypes as C

import pytest

from test_abi import lib      # noqa: F401  (the fixture)
from test_gated_delta_abi import delta_args


@pytest.mark.parametrize("missing", ["o"])
def test_forward_without_sequences(lib, missing):      # noqa: F811
    assert lib.kda_delta_chunk_fwd(C.byref(delta_args(N=0, **{missing: 0})), None) == -1
    assert lib.kda_delta_chunk_fwd(C.byref(delta_args(N=0, tokens=0, **{missing: 0})), None) == 0


@pytest.mark.parametrize("missing", ["dq", "dk", "dv", "dg", "dbeta"])
def test_backward_without_sequences(lib, missing):      # noqa: F811
    assert lib.kda_delta_chunk_bwd(C.byref(delta_args(N=0, **{missing: 0})), None) == -1
    assert lib.kda_delta_chunk_bwd(C.byref(delta_args(N=0, tokens=0, **{missing: 0})), None) == 0


def test_decode_without_sequences(lib):      # noqa: F811
    from kda_b200 import _lib
    call = lambda **kw: lib.kda_delta_recurrent_fwd(C.byref(_lib.RecurrentArgs(**{**dict(N=0, T=4, tokens=4, H=2, K=64, V=64, io_dtype=_lib.KDA_BF16, cu_seqlens=512), **kw})), 0, 0, None)      # noqa: E731
    assert call(o=0) == -1 and call(tokens=0) == 0 and call(o=512, io_dtype=7) == -3
