"""The chunked gated delta rule with one decay per head against float64: token by token, gradients by float64 autograd (the oracle with that decay in every key
channel), and against differences.

Tolerances.  A rounding to bf16 is off by at most 2^-8 of the value.  o and dv round once behind sums whose operands are inputs or bf16 pairs (2^-16 each):
2^-8 + 2^-12.  Final states and dh0 are float32: per chunk five pair roundings (state, r, w v_new, Tm, and the products of two low parts, which are left out), at most
5 * 2^-16 of the terms, which decay from chunk to chunk: 2^-13.  dq, dk, dg, dbeta: every term is a product with one bf16 operand that is not an input
or, behind E, two, and E's own product has one; with the result's rounding four times 2^-8."""
import gc

import numpy as np
import pytest
import torch

from oracle.kda_oracle import recurrent_kda, recurrent_kda_grads, rel_l2_err

pytestmark = pytest.mark.gpu
ONCE, STATE, GRAD = 2.0 ** -8 + 2.0 ** -12, 2.0 ** -13, 4 * 2.0 ** -8
TOL = dict(o=ONCE, ht=STATE, dq=GRAD, dk=GRAD, dv=ONCE, dg=GRAD, dbeta=GRAD, dh0=STATE)


@pytest.fixture(scope="module", autouse=True)
def leave_no_memory():
    yield
    gc.collect()
    torch.cuda.empty_cache()


def make(B, T, H, HV, K, V, seed, n_states=None, h0=True, normed=True, mild=None, dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)      # noqa: E731
    q, k = randn(B, T, H, K), randn(B, T, H, K) + 0.3      # keys with something in common, as behind an activation
    if normed:
        q, k = (x / x.norm(dim=-1, keepdim=True) for x in (q, k))
    A = torch.exp(torch.linspace(0, np.log(16.0), HV))
    g = -A * torch.nn.functional.softplus(randn(B, T, HV) - 3) * (1.0 if mild is None else mild)
    N = n_states or B
    return dict(q=q.to(dtype), k=k.to(dtype), v=randn(B, T, HV, V).to(dtype), g=g, beta=torch.sigmoid(randn(B, T, HV)), h0=0.3 * randn(N, HV, K, V) if h0 else None,
                do=randn(B, T, HV, V).to(dtype), dht=0.5 * randn(N, HV, K, V))


def reference(d, grads=True, **kw):
    grp = d["v"].shape[2] // d["q"].shape[2]
    K = d["q"].shape[-1]
    cuda = {n: (t.cuda() if t is not None else None) for n, t in d.items()}
    spread = lambda t: t.repeat_interleave(grp, 2)      # noqa: E731
    gk = cuda["g"].unsqueeze(-1).expand(*cuda["g"].shape, K)
    h0 = cuda["h0"]
    if not grads:
        o, ht = recurrent_kda(spread(cuda["q"]), spread(cuda["k"]), cuda["v"], gk, cuda["beta"], initial_state=h0, output_final_state=True, **kw)
        return dict(o=o, ht=ht)
    r = recurrent_kda_grads(spread(cuda["q"]), spread(cuda["k"]), cuda["v"], gk, cuda["beta"], cuda["do"], cuda["dht"], initial_state=h0, **kw)
    r["dg"] = r["dg"].sum(-1)
    for n in ("dq", "dk"):
        r[n] = r[n].reshape(*r[n].shape[:2], -1, grp, K).sum(3)
    return r


def run(d, cu=None, slices=0, grads=True, **kw):
    from kda_b200 import chunk_gated_delta, delta
    delta.SCAN_SLICES = slices
    try:
        x = {n: (d[n].cuda().requires_grad_(grads) if d[n] is not None else None) for n in ("q", "k", "v", "g", "beta", "h0")}
        o, ht = chunk_gated_delta(x["q"], x["k"], x["v"], x["g"], x["beta"], initial_state=x["h0"], output_final_state=True, cu_seqlens=cu, **kw)
        if not grads:
            return dict(o=o, ht=ht)
        names = [n for n in x if x[n] is not None]
        g = torch.autograd.grad((o, ht), [x[n] for n in names], (d["do"].cuda(), d["dht"].cuda()))
        return dict(o=o.detach(), ht=ht.detach(), **{("dh0" if n == "h0" else "d" + n): t for n, t in zip(names, g)})
    finally:
        delta.SCAN_SLICES = 0


def check(got, ref):
    # exp of a sum of g below -88 is no normal float32 number (2^-126) and counts as zero: dh0 behind 200 quick decays, exp(-1000) and less
    errors = {n: rel_l2_err(t, ref[n]) if ref[n].abs().max() >= 2.0 ** -126 else float(t.abs().max() >= 2.0 ** -126) for n, t in got.items()}
    for n, t in got.items():
        assert t.shape == ref[n].shape and torch.isfinite(t.float()).all(), n
    print({n: f"{e:.2e}" for n, e in errors.items()})
    bad = {n: e for n, e in errors.items() if not e <= TOL[n]}
    assert not bad, bad


def dg_bound(d):
    """How far dg may be off, token by token, where its terms cancel (one head size of one column: every key is the same up to its sign and overwrites the
    state; quick decays).  The kernel forms, per chunk with start state h and gradient dh of its end state,
        dG_i = sum_j F_ij q_i k_j + scale Gam_i q_i (dO_i h^T)  +  sum_j E_ij k_i k_j - beta_i Gam_i k_i (f_i h^T)  -  sum_j (E_ji k_j + F_ji q_j) k_i - w_i k_i (v_new_i dh^T)
        dG_last += Gam_last <h, dh> + sum_i w_i k_i (v_new_i dh^T),     dg_t = sum of dG_i, i >= t,
    with E_ij = -beta_i D_ij f_i v_new_j and F_ij = scale D_ij dO_i v_new_j.  E is rounded once and so are f and v_new in it: 3 * 2^-8 of the products' absolute
    values; every other term has two rounded operands.  So dg_t is off by at most 3 * 2^-8 (and float32's share, 2^-16) of the sum of the terms' absolute
    values, and by its own rounding."""
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
        kk, qk = k @ k.transpose(-1, -2), q @ k.transpose(-1, -2)
        Tm = torch.linalg.inv(torch.eye(n, device="cuda", dtype=torch.float64) + (beta.unsqueeze(-1) * D * kk).tril(-1))
        gam, w, bt = G.exp().unsqueeze(-1), (G[..., -1:] - G).exp().unsqueeze(-1), beta.unsqueeze(-1)
        vn = Tm @ (bt * (v - gam * (k @ h)))
        f = Tm.transpose(-1, -2) @ ((scale * D * qk).transpose(-1, -2) @ do + w * (k @ dh))
        E = (bt * D * (f.abs() @ vn.abs().transpose(-1, -2))).tril(-1) * kk.abs()
        F = scale * D * (do.abs() @ vn.abs().transpose(-1, -2)) * qk.abs()
        z = (w * k.abs() * (vn.abs() @ dh.abs().transpose(-1, -2))).sum(-1)
        terms = (E + F).sum(-1) + (E + F).sum(-2) + z + (gam * (bt * k.abs() * (f.abs() @ h.abs().transpose(-1, -2)) + scale * q.abs() * (do.abs() @ h.abs().transpose(-1, -2)))).sum(-1)
        last = gam[..., -1, 0] * (h * dh).abs().sum((-1, -2)) + z.sum(-1)
        out[:, a:b] = (terms.flip(-1).cumsum(-1).flip(-1) + last.unsqueeze(-1)).transpose(1, 2)
        leaf = h.detach().requires_grad_()
        o, end = step(leaf, a, b)
        (dh,) = torch.autograd.grad((o, end), leaf, (x["do"][:, a:b], dh))
    return (3 * 2.0 ** -8 + 2.0 ** -16) * out


def check_dg(got, ref, d):
    off = (got["dg"].double() - ref["dg"]).abs()
    assert (off <= dg_bound(d) + 2.0 ** -8 * ref["dg"].abs()).all()


@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 130, 320])
def test_forward_lengths(T):
    d = make(2, T, 2, 2, 128, 128, seed=T)
    check(run(d, grads=False), reference(d, grads=False))


@pytest.mark.parametrize("slices", [1, 2, 4])
def test_every_layout(slices):
    d = make(1, 200, 2, 2, 128, 128, seed=11)
    check(run(d, slices=slices), reference(d))


@pytest.mark.parametrize("T", [1, 63, 64, 65, 130, 257])
def test_gradients_lengths(T):
    d = make(2, T, 2, 2, 128, 128, seed=100 + T)
    check(run(d), reference(d))


@pytest.mark.parametrize("K,V", [(64, 64), (128, 64), (64, 128), (96, 96), (32, 8), (8, 128), (40, 72), (20, 37), (1, 1)])
@pytest.mark.parametrize("slices", [0, 1, 2])
def test_head_sizes(K, V, slices):
    d = make(1, 100, 2, 2, K, V, seed=K * 7 + V)
    got, ref = run(d, slices=slices), reference(d)
    check_dg(got, ref, d)
    if K == 1:
        got.pop("dg")
    check(got, ref)


@pytest.mark.parametrize("grp", [2, 4])
def test_grouped_value_heads_and_norm(grp):
    d = make(2, 150, 2, 2 * grp, 128, 128, seed=5 + grp, normed=False)
    check(run(d, use_qk_l2norm_in_kernel=True), reference(d, use_qk_l2norm=True))


def test_norm_scale_no_state():
    d = make(1, 150, 2, 2, 128, 64, seed=32, h0=False, normed=False)
    check(run(d, scale=0.2, use_qk_l2norm_in_kernel=True), reference(d, scale=0.2, use_qk_l2norm=True))


@pytest.mark.parametrize("mild", [0.0, 0.01, 30.0, 3000.0])
def test_slow_and_quick_decays(mild):
    """Quick ones: every token forgets the one before, and dg is a small difference of its terms."""
    d = make(1, 200, 4, 4, 128, 128, seed=21, mild=mild)
    got, ref = run(d), reference(d)
    check_dg(got, ref, d)
    if mild > 1:
        got.pop("dg")
    check(got, ref)


def test_forgetting_gate():
    """g = -inf resets a head's state: what lies before has no influence, and nothing is NaN."""
    d = make(1, 150, 1, 2, 128, 128, seed=22)
    d["g"][:, 70] = -float("inf")
    got = run(d, grads=False)
    tail = {n: (t[:, 70:] if t is not None and n not in ("h0", "dht") else t) for n, t in d.items()}
    tail["g"] = tail["g"].clone()
    tail["g"][:, 0] = 0
    tail["h0"] = torch.zeros_like(d["h0"])
    ref = reference(tail, grads=False)
    assert rel_l2_err(got["o"][:, 70:], ref["o"]) <= ONCE and rel_l2_err(got["ht"], ref["ht"]) <= STATE


def test_half_types_of_gate_and_beta():
    d = make(1, 130, 2, 2, 128, 128, seed=23)
    d["g"], d["beta"] = d["g"].bfloat16(), d["beta"].bfloat16()
    got = run(d)
    assert got["dg"].dtype == got["dbeta"].dtype == torch.bfloat16
    check(got, reference(d))


def test_masked_tokens_beta_zero():
    """beta = 0 writes nothing; its gradient is that of the formula, not of a division by it."""
    d = make(1, 130, 2, 2, 128, 128, seed=24)
    d["beta"][:, 20:40] = 0
    check(run(d), reference(d))


@pytest.mark.parametrize("lens", [[130, 1, 64, 77], [0, 5, 0, 200, 0], [1] * 9, [65, 63]])
def test_packed(lens):
    """A packed batch: against float64, and bit for bit what each sequence gives alone."""
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32)
    d = make(1, sum(lens), 2, 4, 128, 128, seed=33 + len(lens), n_states=len(lens))
    got = run(d, cu=cu.cuda())
    check(got, reference(d, cu_seqlens=cu))
    for n, m in enumerate(lens):
        if m == 0:
            assert torch.equal(got["ht"][n].cpu(), d["h0"][n]) and torch.equal(got["dh0"][n].cpu(), d["dht"][n])
            continue
        a, b = int(cu[n]), int(cu[n + 1])
        one = {x: (t[:, a:b] if x not in ("h0", "dht") else t[n:n + 1]) for x, t in d.items()}
        alone = run(one)
        for x, t in alone.items():
            assert torch.equal(t, got[x][n:n + 1] if x in ("ht", "dh0") else got[x][:, a:b]), (n, x)


def test_neighbours_do_not_leak():
    """A sequence full of NaN and infinities beside another one in the same chunk's rows leaves that one's results as they are."""
    lens = [70, 33, 90]
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32).cuda()
    d = make(1, sum(lens), 2, 2, 128, 128, seed=40, n_states=3)
    clean = run(d, cu=cu)
    for n, bad in (("q", float("nan")), ("k", float("inf")), ("v", float("nan")), ("do", -float("inf")), ("g", float("nan")), ("beta", float("nan"))):
        d[n][:, 70:103] = bad
    got = run(d, cu=cu)
    for x in got:
        if x in ("ht", "dh0"):
            assert torch.equal(got[x][0], clean[x][0]) and torch.equal(got[x][2], clean[x][2]), x
        else:
            assert torch.equal(got[x][:, :70], clean[x][:, :70]) and torch.equal(got[x][:, 103:], clean[x][:, 103:]), x


def test_rows_of_no_sequence():
    """Rows in front of the first and behind the last sequence come out as zeros, gradients too."""
    d = make(1, 200, 1, 2, 64, 64, seed=41, n_states=2)
    cu = torch.tensor([10, 60, 170], dtype=torch.int32).cuda()
    got = run(d, cu=cu)
    for x in ("o", "dq", "dk", "dv", "dg", "dbeta"):
        assert not got[x][:, :10].any() and not got[x][:, 170:].any(), x
    one = {x: (t[:, 10:60] if x not in ("h0", "dht") else t[:1]) for x, t in d.items()}
    alone = run(one)
    for x in ("o", "dq", "dk", "dv", "dg", "dbeta"):
        assert torch.equal(alone[x], got[x][:, 10:60]), x


def test_gradients_against_differences():
    """<gradient, direction> is the slope of the loss along it, from two float64 evaluations of the recurrence."""
    d = make(1, 90, 1, 2, 64, 64, seed=50)
    got = run(d)
    gen = torch.Generator().manual_seed(3)

    def loss(x):
        r = reference(x, grads=False)
        return float((r["o"] * d["do"].cuda().double()).sum() + (r["ht"] * d["dht"].cuda().double()).sum())

    base = {n: (t.double() if t is not None else None) for n, t in d.items()}
    for n in ("q", "k", "v", "g", "beta", "h0"):
        g = got["dh0" if n == "h0" else "d" + n].double().cpu()
        u = torch.randn(g.shape, generator=gen, dtype=torch.float64)
        u = u / u.norm() + g / g.norm()      # a direction in which the slope is not lost in the gradient's rounding
        slope = (loss({**base, n: base[n] + 1e-5 * u}) - loss({**base, n: base[n] - 1e-5 * u})) / 2e-5
        assert abs(slope - float((g * u).sum())) <= 2 * GRAD * float(g.norm() * u.norm()), n


def test_intermediate_precision_of_long_states():
    """512 chunks: the state's error does not grow with the sequence."""
    d = make(1, 32768, 1, 2, 128, 128, seed=60)
    got, ref = run(d, grads=False), reference(d, grads=False)
    assert rel_l2_err(got["ht"], ref["ht"]) <= 2e-5 and rel_l2_err(got["o"], ref["o"]) <= ONCE


def test_transposed_states_and_strides():
    from kda_b200 import chunk_gated_delta
    d = make(2, 100, 2, 2, 64, 128, seed=61)
    x = {n: t.cuda() for n, t in d.items()}
    o, ht = chunk_gated_delta(x["q"], x["k"], x["v"], x["g"], x["beta"], initial_state=x["h0"], output_final_state=True)
    o2, ht2 = chunk_gated_delta(x["q"], x["k"], x["v"], x["g"], x["beta"], initial_state=x["h0"].transpose(-1, -2).contiguous(), output_final_state=True,
                                transpose_state_layout=True)
    assert torch.equal(o, o2) and torch.equal(ht, ht2.transpose(-1, -2))
    odd = {n: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t) for n, t in x.items()}      # no 16-byte alignment
    o3, ht3 = chunk_gated_delta(odd["q"], odd["k"], odd["v"], odd["g"], odd["beta"], initial_state=odd["h0"], output_final_state=True)
    assert torch.equal(o, o3) and torch.equal(ht, ht3)
    wide = torch.cat([x["q"], x["k"]], -1)      # slices of one projection
    o4, _ = chunk_gated_delta(wide[..., :64], wide[..., 64:], x["v"].transpose(1, 2).contiguous().transpose(1, 2), x["g"], x["beta"], initial_state=x["h0"])
    assert torch.equal(o, o4)


def test_float32():
    """float32 runs token by token: with gradients the exact kernels (1e-4 is that path's bound), without the recurrent one."""
    d = make(1, 70, 1, 2, 64, 64, seed=62, dtype=torch.float32)
    got, ref = run(d), reference(d)
    for n in got:
        assert rel_l2_err(got[n], ref[n]) <= 1e-5, n
    got = run(d, grads=False)
    assert rel_l2_err(got["o"], ref["o"]) <= 1e-5 and rel_l2_err(got["ht"], ref["ht"]) <= 1e-5


def test_no_gradient_wanted_for_some():
    from kda_b200 import chunk_gated_delta
    d = {n: t.cuda() for n, t in make(1, 70, 1, 2, 64, 64, seed=63).items()}
    full = run({n: t.cpu() for n, t in d.items()})
    d["v"].requires_grad_()
    o, ht = chunk_gated_delta(d["q"], d["k"], d["v"], d["g"], d["beta"], initial_state=d["h0"], output_final_state=True)
    (dv,) = torch.autograd.grad(ht, d["v"], d["dht"], retain_graph=True)      # o's gradient is missing
    (dv2,) = torch.autograd.grad(o, d["v"], d["do"])
    assert rel_l2_err(dv.double() + dv2.double(), full["dv"].double()) <= 3 * 2.0 ** -8
    with pytest.raises(NotImplementedError):
        o, _ = chunk_gated_delta(d["q"], d["k"], d["v"], d["g"], d["beta"])
        torch.autograd.grad(o, d["v"], d["do"], create_graph=True)


def test_refusals():
    from kda_b200 import chunk_gated_delta
    d = {n: t.cuda() for n, t in make(1, 10, 2, 2, 64, 64, seed=64).items()}
    args = [d[n] for n in ("q", "k", "v", "g", "beta")]
    with pytest.raises(RuntimeError):
        chunk_gated_delta(*[t.cpu() for t in args])
    with pytest.raises(AssertionError):
        chunk_gated_delta(*args[:3], args[3].unsqueeze(-1).expand(1, 10, 2, 64), args[4])
    with pytest.raises(ValueError):
        chunk_gated_delta(*args[:4], args[4].cpu())
    with pytest.raises(ValueError):
        chunk_gated_delta(*args, initial_state=d["h0"][:, :1])
    with pytest.raises(ValueError):
        chunk_gated_delta(*[torch.cat([t, t]) for t in args], cu_seqlens=torch.tensor([0, 10], device="cuda"))
    with pytest.raises(NotImplementedError):
        chunk_gated_delta(*[t.half() if i < 3 else t for i, t in enumerate(args)])
    with pytest.raises(NotImplementedError):
        big = torch.zeros(1, 10, 2, 192, device="cuda", dtype=torch.bfloat16)
        chunk_gated_delta(big, big, big, args[3], args[4])


def test_bad_cu_seqlens_is_reported():
    from kda_b200 import _lib, chunk_gated_delta
    d = {n: t.cuda() for n, t in make(1, 10, 1, 1, 64, 64, seed=65).items()}
    with pytest.raises(_lib.KdaError):
        chunk_gated_delta(*[d[n] for n in ("q", "k", "v", "g", "beta")], cu_seqlens=torch.tensor([0, 400], device="cuda"))


def test_nothing_to_do():
    from kda_b200 import chunk_gated_delta
    d = {n: t.cuda() for n, t in make(2, 0, 2, 2, 64, 64, seed=66).items()}
    o, ht = chunk_gated_delta(*[d[n] for n in ("q", "k", "v", "g", "beta")], initial_state=d["h0"], output_final_state=True)
    assert o.shape == (2, 0, 2, 64) and torch.equal(ht, d["h0"])


@pytest.mark.captures_graph
def test_replays_from_a_graph():
    from kda_b200 import chunk_gated_delta
    d = {n: t.cuda() for n, t in make(1, 200, 2, 2, 128, 128, seed=67, n_states=2).items()}
    cu = torch.tensor([0, 90, 200], dtype=torch.int32, device="cuda")
    call = lambda: chunk_gated_delta(*[d[n] for n in ("q", "k", "v", "g", "beta")], initial_state=d["h0"], output_final_state=True, cu_seqlens=cu)      # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1, h1 = call()
    with torch.cuda.graph(g2):
        o2, h2 = call()
    d["v"].copy_(torch.randn_like(d["v"]))
    g1.replay()
    g2.replay()
    o, h = call()
    assert torch.equal(o, o1) and torch.equal(h, h1) and torch.equal(o, o2) and torch.equal(h, h2)


def test_same_bits_again_and_on_another_stream():
    d = make(2, 300, 2, 4, 128, 128, seed=68)
    a, b = run(d), run(d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = run(d)
    torch.cuda.synchronize()
    for n in a:
        assert torch.equal(a[n], b[n]) and torch.equal(a[n], c[n]), n
