"""CPU tests of the entry points of the gated delta rule with one decay per head and of the norms: structs, workspace sizes, and arguments that are refused on the
host before anything is launched."""
import ctypes as C

import pytest
import torch

from test_abi import _header_fields, lib      # noqa: F401  (the fixture)


def test_bindings_have_the_headers_fields(lib):      # noqa: F811
    from kda_b200 import _lib
    for struct, cls in (("kda_delta_args", _lib.DeltaArgs), ("kda_norm_args", _lib.NormArgs)):
        assert list(cls._fields_) == _header_fields(struct), struct


def delta_args(**kw):
    from kda_b200 import _lib
    names = ("q", "k", "v", "g", "beta", "o", "d_o", "dq", "dk", "dv", "dg", "dbeta", "workspace", "bwd_workspace")
    a = dict(tokens=128, N=2, H=4, HQ=2, K=64, V=64, io_dtype=_lib.KDA_BF16, g_dtype=_lib.KDA_FP32, beta_dtype=_lib.KDA_FP32, workspace_bytes=1 << 30,
             bwd_workspace_bytes=1 << 30, **{n: 512 for n in names})
    a.update(kw)
    return _lib.DeltaArgs(**a)


BAD_DELTA = [(dict(K=12), -2), (dict(K=0), -2), (dict(K=136), -2), (dict(V=256), -2), (dict(H=0), -2), (dict(HQ=3), -2), (dict(HQ=8), -2), (dict(N=-1), -2), (dict(tokens=-1), -2),
             (dict(N=3), -2), (dict(scan_slices=3), -2), (dict(tokens=1 << 31, N=1), -2), (dict(H=1 << 30, HQ=0), -2), (dict(io_dtype=0), -3), (dict(g_dtype=7), -3),
             (dict(beta_dtype=-1), -3), (dict(q=0), -1), (dict(beta=0), -1), (dict(workspace=0), -1), (dict(q=520), -4), (dict(h0=516), -4), (dict(workspace=640), -4),
             (dict(g=514), -4), (dict(beta=513), -4), (dict(cu_seqlens=514), -4),
             (dict(workspace_bytes=64), -5)]


@pytest.mark.parametrize("bad,code", BAD_DELTA)
def test_chunk_refusals(lib, bad, code):      # noqa: F811
    from kda_b200 import _lib
    if "io_dtype" in bad:
        bad = dict(io_dtype=_lib.KDA_FP32)
    a = delta_args(**bad)
    assert lib.kda_delta_chunk_fwd(C.byref(a), None) == code
    assert lib.kda_delta_chunk_bwd(C.byref(a), None) == code


@pytest.mark.parametrize("bad,code", [(dict(dq=0), -1), (dict(d_o=0), -1), (dict(dbeta=0), -1), (dict(bwd_workspace=0), -1), (dict(bwd_workspace=640), -4), (dict(dv=520), -4),
                                      (dict(d_ht=516), -4), (dict(bwd_workspace_bytes=64), -5)])
def test_chunk_backward_refusals(lib, bad, code):      # noqa: F811
    assert lib.kda_delta_chunk_bwd(C.byref(delta_args(**bad)), None) == code


def test_null_and_nothing_to_do(lib):      # noqa: F811
    for f in (lib.kda_delta_chunk_fwd, lib.kda_delta_chunk_bwd, lib.kda_gated_norm_fwd, lib.kda_gated_norm_bwd, lib.kda_residual_norm_fwd, lib.kda_residual_norm_bwd):
        assert f(None, None) == -1
    assert lib.kda_delta_recurrent_fwd(None, 0, 0, None) == -1
    assert lib.kda_norm_status(None) == -1
    assert lib.kda_delta_chunk_fwd(C.byref(delta_args(tokens=0, N=0)), None) == 0


def test_recurrent_refusals(lib):      # noqa: F811
    from kda_b200 import _lib
    def call(slots=4, columns=1, **kw):
        a = dict(N=2, T=1, tokens=2, H=2, K=64, V=64, io_dtype=_lib.KDA_BF16, g_raw_dtype=_lib.KDA_FP32, beta_raw_dtype=_lib.KDA_BF16, q=512, k=512, v=512, g=512, beta=512, o=512,
                 h0=512, ht=512)
        a.update(kw)
        return lib.kda_delta_recurrent_fwd(C.byref(_lib.RecurrentArgs(**a)), slots, columns, None)
    assert call(g_raw_dtype=9) == call(beta_raw_dtype=9) == -3
    assert call(K=48) == call(V=40) == call(HQ=3) == call(tokens=5) == -2
    assert call(slots=0, state_indices=512) == call(columns=0, state_indices=512) == call(slots=-1, state_indices=512) == -2      # nothing can be followed
    assert call(state_indices=512, ht=1024) == -2
    assert call(num_accepted_tokens=512) == call(v=0) == -1
    assert call(q=520) == call(h0=516, ht=516) == call(g=514) == call(beta=513) == call(state_indices=514) == call(A_log=513) == -4
    assert call(N=0, tokens=0) == 0


def norm_args(**kw):
    from kda_b200 import _lib
    names = ("x", "gate", "residual", "weight", "y", "r", "dy", "dr", "dx", "dgate", "dresidual", "dweight", "workspace")
    a = dict(rows=4, cols=128, io_dtype=_lib.KDA_BF16, gate_dtype=_lib.KDA_BF16, residual_dtype=_lib.KDA_FP32, weight_dtype=_lib.KDA_BF16, post_dtype=_lib.KDA_BF16,
             scale_dtype=_lib.KDA_BF16, workspace_bytes=1 << 30, **{n: 512 for n in names})
    a.update(kw)
    return _lib.NormArgs(**a)


@pytest.mark.parametrize("bad,code", [(dict(cols=0), -2), (dict(rows=-1), -2), (dict(rows=1 << 41), -2), (dict(io_dtype=5), -3), (dict(weight_dtype=5), -3), (dict(x=0), -1)])
def test_norm_refusals(lib, bad, code):      # noqa: F811
    a = norm_args(**bad)
    for f in (lib.kda_gated_norm_fwd, lib.kda_gated_norm_bwd, lib.kda_residual_norm_fwd, lib.kda_residual_norm_bwd):
        assert f(C.byref(a), None) == code


def test_norm_refusals_of_one_call(lib):      # noqa: F811
    limit = lib.kda_gated_norm_fwd(C.byref(norm_args(cols=8193)), None)
    assert limit < 0 and b"maximum" in lib.kda_b200_strerror(limit)
    gf, gb, rf, rb = ((lambda f: lambda **kw: f(C.byref(norm_args(**kw)), None))(getattr(lib, n)) for n in
                      ("kda_gated_norm_fwd", "kda_gated_norm_bwd", "kda_residual_norm_fwd", "kda_residual_norm_bwd"))
    assert gf(activation=2) == -2 and gf(gate_dtype=9) == -3 and rf(residual_dtype=9) == -3
    assert gf(gate=0) == gf(y=0) == gb(dgate=0) == gb(dy=0) == gb(workspace=0) == -1
    assert rf(weight=0) == rf(residual=0) == rf(r=0) == rb(dx=0) == rb(dy=0, dr=0) == rb(workspace=0) == -1
    assert gf(x=513) == rf(residual=514) == gf(weight=513) == rb(dr=514) == gb(dgate=513) == -4
    assert gb(workspace_bytes=16) == rb(workspace_bytes=16) == -5 and gb(workspace=520) == -4


def test_workspace_sizes(lib):      # noqa: F811
    f = lib.kda_delta_chunk_workspace_bytes
    assert 0 < f(4096, 1, 2, 128, 128, 0) < f(4096, 1, 2, 128, 128, 1) < f(8192, 1, 2, 128, 128, 1) < f(8192, 1, 4, 128, 128, 1)
    assert f(-1, 1, 2, 128, 128, 0) == f(64, -1, 2, 128, 128, 0) == f(64, 1, 0, 128, 128, 0) == 0
    b = lib.kda_delta_chunk_bwd_workspace_bytes
    assert 0 < b(4096, 1, 4, 4, 128, 128) < b(4096, 1, 4, 2, 128, 128)      # grouped heads: gradients per value head
    n = lib.kda_norm_bwd_workspace_bytes
    assert 0 < n(10, 128, 1) < n(10, 128, 2) and n(10, 0, 1) == n(10, 9000, 1) == n(10, 128, 3) == n(-1, 128, 1) == 0


def test_large_workspace_is_counted_in_64_bits(lib):      # noqa: F811
    per_token = lib.kda_delta_chunk_workspace_bytes(1 << 20, 1, 64, 128, 128, 1) / 2 ** 20
    assert lib.kda_delta_chunk_workspace_bytes(1 << 30, 1, 64, 128, 128, 1) > 2 ** 30 * per_token * 0.99


def test_python_entries_refuse_cpu_tensors(lib):      # noqa: F811
    import kda_b200 as K
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    g = torch.zeros(1, 4, 2)
    x, w = torch.zeros(4, 64), torch.ones(64)
    for call in (lambda: K.chunk_gated_delta(q, q, q, g, g), lambda: K.fused_recurrent_gated_delta(q, q, q, g, g), lambda: K.gated_rms_norm(x, x, w),
                 lambda: K.residual_rms_norm(x, x, w)):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    with pytest.raises(ValueError):
        K.gated_rms_norm(x, x, w, activation="tanh")
    for name in ("chunk_gated_delta", "fused_recurrent_gated_delta", "fused_recurrent_gated_delta_fwd", "gated_rms_norm", "residual_rms_norm"):
        assert name in K.__all__ and getattr(K, name).__doc__
