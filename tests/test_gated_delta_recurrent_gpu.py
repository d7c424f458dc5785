"""The decode call of the gated delta rule with one decay per head against float64, token by token.

Tolerances, of the norm.  The state is float32: a token's decay is off by at most 2^-21 of itself (its argument, up to 16, times 2^-24, and an exponential of two
steps), a sum of up to 256 products in a tree by 2^-20 of its terms, whose magnitudes add up to 16 times a random sum's at most: up to 64 tokens
that forget as they go 2^-14.  o in bf16 rounds once more: 2^-8 + 2^-14."""
import gc

import numpy as np
import pytest
import torch

from _abi import bulk_decode_batch
from oracle.kda_oracle import rel_l2_err

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
STATE = 2.0 ** -14


@pytest.fixture(scope="module", autouse=True)
def leave_no_memory():
    yield
    gc.collect()
    torch.cuda.empty_cache()


def tol(dtype):
    return STATE + (2.0 ** -8 if dtype == BF else 0.0)


def make(B, T, H, HV, K, V, seed, dtype=BF, gate_dtype=F32, raw=False):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)      # noqa: E731
    q, k = (x / x.norm(dim=-1, keepdim=True) for x in (randn(B, T, H, K), randn(B, T, H, K) + 0.3))
    g = randn(B, T, HV) if raw else -torch.nn.functional.softplus(randn(B, T, HV) - 1)
    beta = randn(B, T, HV) if raw else torch.sigmoid(randn(B, T, HV))
    return dict(q=q.to(dtype).cuda(), k=k.to(dtype).cuda(), v=randn(B, T, HV, V).to(dtype).cuda(), g=g.to(gate_dtype).cuda(), beta=beta.to(gate_dtype).cuda())


def reference(x, S, scale=None, l2=False, A_log=None, dt_bias=None, lower_bound=None, sigmoid=False):
    """x's sequences [B, T, ..] from states S [B, HV, K, V]: (o, states behind every token [B, T, HV, K, V]), all in float64."""
    q, k, v, g, beta = (x[n].double() for n in ("q", "k", "v", "g", "beta"))
    grp = v.shape[2] // q.shape[2]
    if l2:
        q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    q, k = q.repeat_interleave(grp, 2), k.repeat_interleave(grp, 2)
    if A_log is not None:
        y = g + (dt_bias.double() if dt_bias is not None else 0.0)
        a = A_log.double().exp()
        g = lower_bound * torch.sigmoid(a * y) if lower_bound is not None else -a * torch.where(y > 30, y, torch.log1p(y.clamp(max=30).exp()))
    if sigmoid:
        beta = torch.sigmoid(beta)
    S, o, states = S.double(), [], []
    for t in range(q.shape[1]):
        S = S * g[:, t].exp()[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - torch.einsum("bhk,bhkv->bhv", k[:, t], S))
        S = S + k[:, t, :, :, None] * u[:, :, None]
        o.append((scale or q.shape[-1] ** -0.5) * torch.einsum("bhk,bhkv->bhv", q[:, t], S))
        states.append(S)
    return torch.stack(o, 1), torch.stack(states, 1)


def states(n, HV, K, V, seed=5):
    return 0.3 * torch.randn(n, HV, K, V, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("K,V", [(32, 32), (64, 64), (128, 128), (128, 96), (256, 64), (64, 256)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_scans(K, V, dtype):
    from kda_b200 import fused_recurrent_gated_delta
    x, h0 = make(2, 37, 2, 4, K, V, K + V, dtype), states(2, 4, K, V)
    o, ht = fused_recurrent_gated_delta(**x, initial_state=h0, output_final_state=True, use_qk_l2norm_in_kernel=True, scale=0.7)
    ref, S = reference(x, h0, scale=0.7, l2=True)
    assert rel_l2_err(o, ref) <= tol(dtype) and rel_l2_err(ht, S[:, -1]) <= STATE and o.dtype == dtype
    o0, none = fused_recurrent_gated_delta(**x)
    assert none is None and rel_l2_err(o0, reference(x, torch.zeros_like(h0))[0]) <= tol(dtype)


@pytest.mark.parametrize("lens", [[1], [5, 0, 1, 33], [0, 0]])
def test_packed(lens):
    from kda_b200 import fused_recurrent_gated_delta
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int64).cuda()
    x, h0 = make(1, max(sum(lens), 1), 2, 2, 64, 64, 3), states(len(lens), 2, 64, 64)
    o, ht = fused_recurrent_gated_delta(**x, initial_state=h0, output_final_state=True, cu_seqlens=cu)
    for i, n in enumerate(lens):
        a = int(cu[i])
        if n == 0:
            assert torch.equal(ht[i], h0[i])
            continue
        ref, S = reference({k: t[:, a:a + n] for k, t in x.items()}, h0[i:i + 1])
        assert rel_l2_err(o[:, a:a + n], ref) <= tol(BF) and rel_l2_err(ht[i:i + 1], S[:, -1]) <= STATE


@pytest.mark.parametrize("gate_dtype", [F32, BF])
@pytest.mark.parametrize("lower_bound", [None, -5.0])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("tr", [False, True])
def test_gate_in_kernel(gate_dtype, lower_bound, bias, tr):
    from kda_b200 import fused_recurrent_gated_delta
    HV = 4
    x, h0 = make(3, 5, 2, HV, 128, 128, 8, gate_dtype=gate_dtype, raw=True), states(3, HV, 128, 128)
    A, b = torch.linspace(-1, 1.5, HV).cuda(), torch.linspace(-2, 1, HV).cuda() if bias else None
    o, ht = fused_recurrent_gated_delta(**x, A_log=A, dt_bias=b, initial_state=h0.transpose(-1, -2).contiguous() if tr else h0, output_final_state=True, use_gate_in_kernel=True,
                                        use_beta_sigmoid_in_kernel=True, lower_bound=lower_bound, transpose_state_layout=tr)
    ref, S = reference(x, h0, A_log=A, dt_bias=b, lower_bound=lower_bound, sigmoid=True)
    assert rel_l2_err(o, ref) <= tol(BF) and rel_l2_err(ht.transpose(-1, -2) if tr else ht, S[:, -1]) <= STATE


def run_pool(x, pool, slots, **kw):
    from kda_b200 import fused_recurrent_gated_delta_fwd
    o, st = fused_recurrent_gated_delta_fwd(**x, initial_state=pool, ssm_state_indices=slots, **kw)
    assert st is pool
    return o


def few_and_many():
    return ["few", "many"]


def batch(which):
    """(sequences, heads): a small batch, and one that takes the kernel with whole states in shared memory"""
    return (5, 6) if which == "few" else bulk_decode_batch()


@pytest.mark.parametrize("which", few_and_many())
@pytest.mark.parametrize("tr", [False, True])
def test_one_token_from_a_pool(which, tr):
    N, HV = batch(which)
    x = make(N, 1, HV // 2, HV, 128, 128, 9, gate_dtype=BF)
    pool = 0.3 * torch.randn(N + 3, HV, 128, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    before = pool.clone()
    slots = torch.randperm(N + 3, generator=torch.Generator().manual_seed(2))[:N].int().cuda()
    o = run_pool(x, pool, slots, use_qk_l2norm_in_kernel=True, transpose_state_layout=tr)
    S0 = before[slots.long()]
    eo, es = 0.0, 0.0
    for a in range(0, N, 8):      # (the reference holds eight states at a time)
        part = {k: t[a:a + 8] for k, t in x.items()}
        ref, S = reference(part, S0[a:a + 8].transpose(-1, -2) if tr else S0[a:a + 8], l2=True)
        got = pool[slots[a:a + 8].long()]
        eo, es = max(eo, rel_l2_err(o[a:a + 8], ref)), max(es, rel_l2_err(got.transpose(-1, -2) if tr else got, S[:, -1]))
    assert eo <= tol(BF) and es <= STATE
    rest = torch.ones(N + 3, dtype=torch.bool)
    rest[slots.long().cpu()] = False
    assert torch.equal(pool[rest.cuda()], before[rest.cuda()])


@pytest.mark.parametrize("N,HV", [(2, 3), (40, 8)])      # below and above half a state per SM
@pytest.mark.parametrize("tr", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_draft_tokens(N, HV, tr, dtype):
    """Every token's state goes to its own slot; the next step starts behind the accepted tokens."""
    T = 4
    pool = states(N * T + 2, HV, 128, 128)
    if tr:
        pool = pool.transpose(-1, -2).contiguous()
    before = pool.clone()
    slots = torch.randperm(N * T + 2, generator=torch.Generator().manual_seed(4))[:N * T].view(N, T).int().cuda()
    accepted = (torch.arange(N) % T + 1).int().cuda()
    x = make(N, T, HV, HV, 128, 128, 12, dtype)
    o = run_pool(x, pool, slots, num_accepted_tokens=accepted, transpose_state_layout=tr)
    view = (lambda t: t.transpose(-1, -2)) if tr else (lambda t: t)
    ref, S = reference(x, view(before[slots[torch.arange(N).cuda(), accepted.long() - 1].long()]))
    assert rel_l2_err(o, ref) <= tol(dtype)
    assert rel_l2_err(view(pool[slots.long().flatten()].view(N, T, HV, 128, 128)), S) <= STATE


@pytest.mark.parametrize("N,HV,T", [(5, 6, 1), (0, 0, 1), (3, 3, 3), (40, 8, 3)])
@pytest.mark.parametrize("tr", [False, True])
def test_padded_entries(N, HV, T, tr):
    """Slots outside the pool: nothing but zeros in o, no state touched; a later token's slot outside it only loses that state."""
    if N == 0:
        N, HV = bulk_decode_batch()
    S_ = N * T
    pool = 0.3 * torch.randn(S_, HV, 128, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    whole, part = pool.clone(), pool.clone()
    slots = torch.randperm(S_, generator=torch.Generator().manual_seed(6)).view(N, T).int()
    x = make(N, T, HV, HV, 128, 128, 13)
    good = slots.cuda()
    o = run_pool(x, whole, good if T > 1 else good[:, 0], transpose_state_layout=tr)
    bad = slots.clone()
    bad[1], bad[N - 1], bad[2, 0] = -1, S_, 2 ** 31 - 1
    if T > 1:
        bad[0, 1] = -7
    bad = bad.cuda()
    o2 = run_pool(x, part, bad if T > 1 else bad[:, 0], transpose_state_layout=tr)
    out = torch.zeros(N, dtype=torch.bool)
    out[[1, 2, N - 1]] = True
    assert torch.count_nonzero(o2[out.cuda()]) == 0 and torch.equal(o2[~out.cuda()], o[~out.cuda()])
    kept = (bad >= 0) & (bad < S_) & ~out.cuda()[:, None]
    assert torch.equal(part[good[kept].long()], whole[good[kept].long()])
    assert torch.equal(part[good[~kept].long()], pool[good[~kept].long()])


@pytest.mark.parametrize("N,HV", [(3, 3), (40, 8)])
def test_accepted_counts_outside_the_table(N, HV):
    pool = states(N * 2, HV, 128, 128)
    before = pool.clone()
    slots = torch.arange(N * 2).view(N, 2).int().cuda()
    accepted = torch.ones(N, dtype=torch.int32)
    accepted[0], accepted[1] = 0, 3
    x = make(N, 2, HV, HV, 128, 128, 14)
    o = run_pool(x, pool, slots, num_accepted_tokens=accepted.cuda())
    assert torch.count_nonzero(o[:2]) == 0 and torch.equal(pool[:4], before[:4])
    ref, S = reference({k: t[2:] for k, t in x.items()}, before[slots[2:, 0].long()])
    assert rel_l2_err(o[2:], ref) <= tol(BF) and rel_l2_err(pool[slots[2:].long().flatten()].view(S.shape), S) <= STATE


@pytest.mark.parametrize("N,HV", [(2, 3), (40, 8)])
def test_fewer_columns_than_tokens(N, HV):
    """Through the C entry: a table of one column for two tokens keeps the first token's state only."""
    import ctypes as C
    from kda_b200 import _lib
    lib = _lib.load()
    x = make(N, 2, HV, HV, 128, 128, 21)
    wide, slim = states(2 * N, HV, 128, 128), states(2 * N, HV, 128, 128)
    before = wide.clone()
    table = torch.arange(2 * N, dtype=torch.int32).view(N, 2).cuda()
    ref = run_pool(x, wide, table, scale=0.1)
    first, o = table[:, 0].contiguous(), torch.empty_like(ref)
    a = _lib.RecurrentArgs(q=x["q"].data_ptr(), k=x["k"].data_ptr(), v=x["v"].data_ptr(), g=x["g"].data_ptr(), beta=x["beta"].data_ptr(), h0=slim.data_ptr(), ht=slim.data_ptr(),
                           o=o.data_ptr(), state_indices=first.data_ptr(), state_indices_stride=1, tokens=2 * N, N=N, T=2, H=HV, K=128, V=128, HQ=HV, io_dtype=_lib.KDA_BF16,
                           g_raw_dtype=_lib.KDA_FP32, beta_raw_dtype=_lib.KDA_FP32, scale=0.1)
    assert lib.kda_delta_recurrent_fwd(C.byref(a), 2 * N, 1, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    assert torch.equal(o, ref) and torch.equal(slim[first.long()], wide[first.long()])
    assert torch.equal(slim[table[:, 1].long()], before[table[:, 1].long()])


@pytest.mark.parametrize("which", few_and_many())
def test_the_same_bits_alone_and_in_a_batch(which):
    """A sequence's result does not depend on its neighbours, NaN among them."""
    N, HV = batch(which)
    x = make(N, 1, HV, HV, 128, 128, 15)
    pool = 0.3 * torch.randn(N, HV, 128, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    a, b = pool.clone(), pool.clone()
    slots = torch.arange(N, dtype=torch.int32, device="cuda")
    o = run_pool(x, a, slots)
    y = {k: t.clone() for k, t in x.items()}
    for t in y.values():
        t[1] = float("nan")
    o2 = run_pool(y, b, slots)
    keep = [i for i in range(N) if i != 1]
    assert torch.equal(o2[keep], o[keep]) and torch.equal(b[keep], a[keep]) and torch.isnan(o2[1]).all()
    x1 = {k: t[2:3] for k, t in x.items()}
    if which == "few":
        alone = pool.clone()
        assert torch.equal(run_pool(x1, alone, slots[2:3])[0], o[2]) and torch.equal(alone[2], a[2])


def test_decay_of_minus_infinity_forgets():
    x, h0 = make(2, 3, 2, 2, 64, 64, 16), states(2, 2, 64, 64)
    x["g"][:, 1] = -float("inf")
    from kda_b200 import fused_recurrent_gated_delta
    o, ht = fused_recurrent_gated_delta(**x, initial_state=h0, output_final_state=True)
    ref, S = reference({k: t[:, 1:] for k, t in x.items()}, torch.zeros_like(h0))
    assert rel_l2_err(o[:, 1:], ref) <= tol(BF) and rel_l2_err(ht, S[:, -1]) <= STATE


def test_prefill_hands_over_to_decode():
    """The chunked form's final states carry on token by token."""
    from kda_b200 import chunk_gated_delta
    x = make(3, 70, 2, 4, 128, 128, 17)
    head, tail = ({k: t[:, s].contiguous() for k, t in x.items()} for s in (slice(0, 66), slice(66, 70)))
    o1, pool = chunk_gated_delta(**head, output_final_state=True, use_qk_l2norm_in_kernel=True)
    out = [o1]
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    for t in range(4):
        out.append(run_pool({k: v[:, t:t + 1].contiguous() for k, v in tail.items()}, pool, slots, use_qk_l2norm_in_kernel=True))
    ref, S = reference(x, torch.zeros(3, 4, 128, 128).cuda(), l2=True)
    assert rel_l2_err(torch.cat(out, 1), ref) <= tol(BF) and rel_l2_err(pool, S[:, -1]) <= 2.0 ** -13


def test_strides_out_and_other_streams():
    from kda_b200 import fused_recurrent_gated_delta_fwd
    x = make(4, 1, 4, 4, 128, 128, 18)
    pool = states(4, 4, 128, 128)
    a, b = pool.clone(), pool.clone()
    slots = torch.arange(4, dtype=torch.int64, device="cuda")
    o = run_pool(x, a, slots)
    qkv = torch.cat([x["q"], x["k"], x["v"]], -1)      # slices of one projection; odd element offsets for the gate
    gb = torch.cat([x["g"][..., :1], x["g"], x["beta"]], -1)
    side = torch.cuda.Stream()
    out = torch.empty_like(o)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r, _ = fused_recurrent_gated_delta_fwd(qkv[..., :128], qkv[..., 128:256], qkv[..., 256:], gb[..., 1:5], gb[..., 5:], initial_state=b, ssm_state_indices=slots, out=out)
    side.synchronize()
    assert r.data_ptr() == out.data_ptr() and torch.equal(out, o) and torch.equal(a, b)


@pytest.mark.captures_graph
@pytest.mark.parametrize("which", few_and_many())
def test_replays_from_a_graph(which):
    N, HV = batch(which)
    x = make(N, 1, HV, HV, 128, 128, 19)
    pool = 0.3 * torch.randn(N, HV, 128, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    start = pool.clone()
    slots = torch.arange(N, dtype=torch.int32, device="cuda")
    o1 = run_pool(x, pool, slots)
    o2 = run_pool(x, pool, slots)
    end = pool.clone()
    pool.copy_(start)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        o = run_pool(x, pool, slots)
    pool.copy_(start)
    g.replay()
    assert torch.equal(o, o1)
    g.replay()
    assert torch.equal(o, o2) and torch.equal(pool, end)
    slots.fill_(-1)      # the whole batch padded
    g.replay()
    assert torch.count_nonzero(o) == 0 and torch.equal(pool, end)


def test_refusals():
    from kda_b200 import fused_recurrent_gated_delta, fused_recurrent_gated_delta_fwd
    x, h0 = make(2, 1, 2, 4, 64, 64, 20), states(2, 4, 64, 64)
    bad = lambda **kw: {**x, **kw}      # noqa: E731
    with pytest.raises(AssertionError):
        fused_recurrent_gated_delta(**bad(g=x["g"][..., None].expand(2, 1, 4, 64)))
    with pytest.raises(AssertionError):
        fused_recurrent_gated_delta(**bad(g=x["g"][..., :3]))
    with pytest.raises(AssertionError):
        fused_recurrent_gated_delta(**bad(v=x["v"][:, :, :3]))
    with pytest.raises(NotImplementedError):
        fused_recurrent_gated_delta(**bad(q=x["q"][..., :48], k=x["k"][..., :48]))
    with pytest.raises(ValueError):
        fused_recurrent_gated_delta(**x, initial_state=h0[:1])
    with pytest.raises(ValueError):
        fused_recurrent_gated_delta(**x, initial_state=h0.cpu())
    with pytest.raises((AssertionError, ValueError)):
        fused_recurrent_gated_delta(**x, initial_state=h0.bfloat16())
    with pytest.raises(AssertionError):
        fused_recurrent_gated_delta(**x, use_gate_in_kernel=True)
    with pytest.raises(ValueError):
        fused_recurrent_gated_delta(**x, A_log=torch.zeros(4).cuda(), dt_bias=torch.zeros(4 * 64).cuda(), use_gate_in_kernel=True)
    slots = torch.zeros(2, dtype=torch.int32).cuda()
    with pytest.raises(ValueError):
        fused_recurrent_gated_delta_fwd(**x, initial_state=h0, ssm_state_indices=slots[:1])
    with pytest.raises(ValueError):
        fused_recurrent_gated_delta_fwd(**x, initial_state=h0, num_accepted_tokens=slots)
    with pytest.raises(ValueError):
        fused_recurrent_gated_delta_fwd(**x, initial_state=h0, ssm_state_indices=slots, inplace_final_state=False)
    with pytest.raises(ValueError):
        fused_recurrent_gated_delta_fwd(**x, initial_state=h0.transpose(-1, -2), ssm_state_indices=slots)
    with pytest.raises(Exception):
        fused_recurrent_gated_delta_fwd(**x, initial_state=h0[:0], ssm_state_indices=slots)
    with pytest.raises(AssertionError):
        fused_recurrent_gated_delta_fwd(**x)
