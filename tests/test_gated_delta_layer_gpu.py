"""The operators together, as a layer uses them: the residual norm, projections, the gated delta rule, its gated norm, the output projection and the next residual
norm; a training step against float64, prompts that are answered token by token, two layers at once, and a captured step.

Tolerances, of a result's norm.  Every hand-over between operators is a bf16 tensor: half a step, 2^-8 at most.  The layer's forward has six of them in a row
(y, a projection, o, the gated norm, the output projection, y), none of which grows an error by more than the norms and bounded gates let it, twofold at most: 12 * 2^-8.  The
gradients run through as many again, of which those of the rule carry 4 * 2^-8: 32 * 2^-8."""
import gc

import pytest
import torch

from oracle.kda_oracle import recurrent_kda, rel_l2_err

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
FORWARD, BACKWARD = 12 * 2.0 ** -8, 32 * 2.0 ** -8
H, HV, D, E = 2, 4, 64, 192      # heads of q and k, value heads, their size, the model's width


@pytest.fixture(scope="module", autouse=True)
def leave_no_memory():
    yield
    gc.collect()
    torch.cuda.empty_cache()


def weights(seed):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)      # noqa: E731
    return {"qkv": (randn(E, (2 * H + HV) * D) / E ** 0.5).to(BF).cuda(), "gate": (randn(E, HV * D) / E ** 0.5).to(BF).cuda(), "ab": (randn(E, 2 * HV) / E ** 0.5).to(BF).cuda(),
            "out": (randn(HV * D, E) / (HV * D) ** 0.5).to(BF).cuda(), "n1": (1 + 0.1 * randn(E)).cuda(), "n2": (1 + 0.1 * randn(D)).to(BF).cuda(), "n3": (1 + 0.1 * randn(E)).cuda(),
            "post": (1 + 0.1 * randn(E)).cuda(), "s": (0.5 + 0.1 * randn(E)).cuda(), "A": torch.linspace(-1, 1, HV).cuda()}


def inputs(B, T, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(B, T, E, generator=gen).to(BF).cuda(), torch.randn(B, T, E, generator=gen).cuda()


def parts(y, w):
    B, T = y.shape[:2]
    qkv, ab = y @ w["qkv"].to(y.dtype), (y @ w["ab"].to(y.dtype)).to(F32 if y.dtype == BF else y.dtype)
    q, k, v = qkv.split([H * D, H * D, HV * D], -1)
    g = -w["A"].to(ab.dtype).exp() * torch.nn.functional.softplus(ab[..., :HV])
    return q.reshape(B, T, H, D), k.reshape(B, T, H, D), v.reshape(B, T, HV, D), g, torch.sigmoid(ab[..., HV:]), (y @ w["gate"].to(y.dtype)).reshape(B, T, HV, D)


def layer(x, res, w, rule):
    from kda_b200 import gated_rms_norm, residual_rms_norm
    y, r = residual_rms_norm(x, res, w["n1"])
    q, k, v, g, beta, z = parts(y, w)
    o, state = rule(q, k, v, g, beta)
    o = gated_rms_norm(o, z, w["n2"], activation="silu")
    return (*residual_rms_norm(o.flatten(-2) @ w["out"], r, w["n3"], scale=w["s"], post_weight=w["post"]), state)


def chunked(q, k, v, g, beta):
    from kda_b200 import chunk_gated_delta
    return chunk_gated_delta(q, k, v, g, beta, output_final_state=True, use_qk_l2norm_in_kernel=True)


def layer64(x, res, w, keep=None):
    w = {n: t.double() for n, t in w.items()}
    rms = lambda t: torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6)      # noqa: E731
    r = res.double() + x.double()
    y = r / rms(r) * w["n1"]
    q, k, v, g, beta, z = parts(y, w)
    q, k = (t.repeat_interleave(HV // H, 2) for t in (q, k))
    o, state = recurrent_kda(q, k, v, g[..., None].expand(*g.shape, D), beta, output_final_state=True, use_qk_l2norm=True)
    if keep is not None:
        keep += [o, y, beta]
    o = o / rms(o) * w["n2"] * torch.nn.functional.silu(z)
    b = o.flatten(-2) @ w["out"]
    r = r + w["s"] * (b / rms(b) * w["post"])
    return r / rms(r) * w["n3"], r, state


@pytest.mark.parametrize("B,T", [(2, 100), (1, 1), (3, 64)])
def test_a_training_step(B, T):
    w = {n: t.requires_grad_() for n, t in weights(1).items()}
    x, res = (t.requires_grad_() for t in inputs(B, T, 2))
    leaves = [x, res, *w.values()]
    dy, dr = inputs(B, T, 3)
    y, r, state = layer(x, res, w, chunked)
    grads = torch.autograd.grad((y, r), leaves, (dy, dr))
    keep = []
    y64, r64, s64 = layer64(x, res, w, keep)
    for got, ref in ((y, y64), (r, r64), (state, s64)):
        assert rel_l2_err(got, ref) <= FORWARD
    ref64 = torch.autograd.grad((y64, r64), leaves + keep[:1], (dy.double(), dr.double()))
    # One token from no state: o = scale beta (q k) v, and the norm behind it drops every factor of a head's o.  So beta's gradient is zero but for eps, a sum of terms
    # dO o / beta that cancel; each of them carries the rounding of dO, and through ab's projection (1 - beta) y of it.
    o, y0, beta = (t.detach() for t in keep)
    terms = (y0[..., :, None] * ((ref64[-1] * o).abs().sum(-1) * (1 - beta))[..., None, :]).norm() if T == 1 else 0.0
    for leaf, got, ref in zip(leaves, grads, ref64):
        size = ref.norm() + (terms if leaf is w["ab"] else 0.0)
        assert got.dtype == leaf.dtype and (got.double() - ref).norm() <= BACKWARD * size


def test_a_prompt_and_its_answer():
    """A prompt in one call and four tokens in one call each give what the whole gives."""
    from kda_b200 import fused_recurrent_gated_delta_fwd
    w, (x, res) = weights(4), inputs(3, 74, 5)
    y, r, pool = layer(x[:, :70].contiguous(), res[:, :70].contiguous(), w, chunked)
    ys, rs = [y], [r]
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    one = lambda q, k, v, g, beta: fused_recurrent_gated_delta_fwd(q, k, v, g, beta, initial_state=pool, ssm_state_indices=slots, use_qk_l2norm_in_kernel=True)      # noqa: E731
    for t in range(70, 74):
        y, r, _ = layer(x[:, t:t + 1].contiguous(), res[:, t:t + 1].contiguous(), w, one)
        ys.append(y)
        rs.append(r)
    y64, r64, s64 = layer64(x, res, w)
    assert rel_l2_err(torch.cat(ys, 1), y64) <= FORWARD and rel_l2_err(torch.cat(rs, 1), r64) <= FORWARD and rel_l2_err(pool, s64) <= FORWARD


def test_packed_and_padded_batches_agree():
    from kda_b200 import chunk_gated_delta
    lens = [70, 1, 33]
    w, (x, res) = weights(6), inputs(1, sum(lens), 7)
    cu = torch.tensor([0, 70, 71, 104], dtype=torch.int32, device="cuda")
    packed = lambda q, k, v, g, beta: chunk_gated_delta(q, k, v, g, beta, output_final_state=True, use_qk_l2norm_in_kernel=True, cu_seqlens=cu)      # noqa: E731
    y, r, state = layer(x, res, w, packed)
    for i, n in enumerate(lens):
        a = int(cu[i])
        y1, r1, s1 = layer(x[:, a:a + n].contiguous(), res[:, a:a + n].contiguous(), w, chunked)
        assert rel_l2_err(y[:, a:a + n], y1) <= FORWARD and rel_l2_err(state[i:i + 1], s1) <= FORWARD


def step(x, res, w, dy, dr):
    y, r, state = layer(x, res, w, chunked)
    grads = torch.autograd.grad((y, r), [x, res, *w.values()], (dy, dr))
    return [y.detach(), r.detach(), state.detach(), *grads]      # (a capture finds no older graph of the same leaves alive: torch's own rule)


def test_two_steps_at_once():
    """Two streams, a step each, interleaved by the host: every call has workspaces of its own."""
    w = {n: t.requires_grad_() for n, t in weights(8).items()}
    data = [(*(t.requires_grad_() for t in inputs(2, 300, s)), *inputs(2, 300, s + 50)) for s in (9, 10)]
    alone = [step(a, b, w, dy, dr) for a, b, dy, dr in data]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(3):
        for i, (a, b, dy, dr) in enumerate(data):
            with torch.cuda.stream(streams[i]):
                got[i] = step(a, b, w, dy, dr)
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.captures_graph
def test_captured_steps_share_the_pool():
    """Two captured steps with one memory pool, replayed in turns on new inputs."""
    w = {n: t.requires_grad_() for n, t in weights(11).items()}
    x, res = (t.requires_grad_() for t in inputs(2, 100, 12))
    dy, dr = inputs(2, 100, 13)
    new = inputs(2, 100, 14)
    first = [t.clone() for t in step(x, res, w, dy, dr)]
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append([t.clone() for t in step(x, res, w, dy, dr)])
        pool = g.pool()
        graphs.append(g)
    for g, out in zip(graphs, outs):
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, first))
    with torch.no_grad():
        x.copy_(new[0])
        res.copy_(new[1])
    second = [t.clone() for t in step(x, res, w, dy, dr)]
    for g, out in reversed(list(zip(graphs, outs))):
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, second))
