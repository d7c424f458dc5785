"""What a layer does around and with the gated delta rule, as cases that can be measured: the operator with one decay per head and token (prompts,
training steps, decode steps of a server), the norm and gate behind it, and the norms and the scaled sum at the residual stream.

A case is a dict; `op` says which operator it is:
  "chunk"      whole sequences: o and final states, or (`train`) o and every gradient
  "recurrent"  decode steps: states in a pool updated in place, one or a few tokens per sequence
  "gated"      y = RMSNorm(x) * weight * act(gate) over the columns of a head, or (`train`) with its gradients
  "residual"   r = residual + scale * RMSNorm(x) * post_weight; y = RMSNorm(r) * weight, or (`train`) with its gradients
and the rest its sizes and options:
  seqs, tokens, packed, shortest   sequences and tokens per sequence; packed: uneven lengths from `shortest` to `tokens` in one row, with cu_seqlens
  heads, value_heads, dim          heads of q and k, of v, and columns of a head
  layer                            chunk: q and k are normalised by the operator; recurrent: so they are, and the gate and beta arrive as the layer's raw values
  draft                            recurrent: tokens per sequence, each with a state slot of its own
  rows, cols, act, post, stream    norms: rows and columns; the gate's activation; whether the block's output has a norm of its own; the residual stream's type
"""
from __future__ import annotations

import math

import torch

own = False

CHUNK = 64
EPS = 1e-6
_BF, _F = torch.bfloat16, torch.float32


def listed():
    return [
        # a short prompt on an idle server: the time to the first token
        dict(name="prefill_1x333", op="chunk", train=False, packed=False, seqs=1, tokens=333, shortest=333, heads=32, value_heads=32, dim=128, layer=False),
        # prompts of a server's queue, read in together; value heads share keys
        dict(name="prefill_packed_12", op="chunk", train=False, packed=True, seqs=12, tokens=8192, shortest=100, heads=16, value_heads=32, dim=128, layer=True),
        # one long document
        dict(name="prefill_1x32768", op="chunk", train=False, packed=False, seqs=1, tokens=32768, shortest=32768, heads=32, value_heads=32, dim=128, layer=True),
        # a fine-tuning step of a small model, sequences of an odd length
        dict(name="train_2x1000_d64", op="chunk", train=True, packed=False, seqs=2, tokens=1000, shortest=1000, heads=8, value_heads=8, dim=64, layer=False),
        # a pre-training step
        dict(name="train_8x4096", op="chunk", train=True, packed=False, seqs=8, tokens=4096, shortest=4096, heads=32, value_heads=32, dim=128, layer=True),
        # one conversation: every generated token is such a call per layer
        dict(name="decode_1", op="recurrent", seqs=1, draft=1, heads=32, value_heads=32, dim=128, layer=True),
        # some dozens of requests with speculative tokens
        dict(name="decode_24_draft_4", op="recurrent", seqs=24, draft=4, heads=16, value_heads=32, dim=128, layer=True),
        # a server under load
        dict(name="decode_1000", op="recurrent", seqs=1000, draft=1, heads=32, value_heads=32, dim=128, layer=False),
        # behind decode_24's operator
        dict(name="gated_96_tokens", op="gated", train=False, rows=96 * 32, cols=128, act="silu"),
        # behind the pre-training step's operator
        dict(name="gated_train_8x4096", op="gated", train=True, rows=8 * 4096 * 32, cols=128, act="sigmoid"),
        # between two blocks of a decode step
        dict(name="residual_48", op="residual", train=False, rows=48, cols=4096, post=False, stream="bf16"),
        # between two blocks of the pre-training step, both norms, the stream in 32 bits
        dict(name="residual_train_8x4096", op="residual", train=True, rows=8 * 4096, cols=4096, post=True, stream="fp32"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "chunk", "recurrent", "recurrent", "gated", "residual"])
    if op == "chunk":
        train = rng.random() < 0.5
        dim = rng.choice([64, 96, 128, 128])
        value_heads = rng.choice([2, 4, 8, 16, 32])
        heads = max(1, value_heads // rng.choice([1, 1, 2, 4]))
        packed = rng.random() < 0.4
        tokens = _spread(rng, 20, 4000 if train else 24000)
        seqs = min(_spread(rng, 2 if packed else 1, 16), max(1, (8 * 4096 if train else 49152) // tokens))
        return dict(op=op, train=train, packed=packed, seqs=seqs, tokens=tokens, shortest=rng.randint(1, tokens) if packed else tokens, heads=heads,
                    value_heads=value_heads, dim=dim, layer=rng.random() < 0.5)
    if op == "recurrent":
        value_heads, draft = rng.choice([8, 16, 32]), rng.choice([1, 1, 2, 3, 5])
        return dict(op=op, seqs=_spread(rng, 1, 1900 // (1 + draft)), draft=draft, heads=value_heads // rng.choice([1, 2]), value_heads=value_heads, dim=128,
                    layer=rng.random() < 0.5)
    if op == "gated":
        cols = rng.choice([64, 96, 128, 256, 200, 77])
        return dict(op=op, train=rng.random() < 0.6, rows=_spread(rng, 5, (1 << 27) // cols), cols=cols, act=rng.choice(["silu", "sigmoid"]))
    cols = rng.choice([1024, 2048, 4096, 5120, 2500, 1001])
    return dict(op=op, train=rng.random() < 0.6, rows=_spread(rng, 3, (1 << 27) // cols), cols=cols, post=rng.random() < 0.5, stream=rng.choice(["bf16", "fp32"]))


def _lengths(c):
    """The packed sequences' lengths: between `shortest` and `tokens`, spread over the logarithm, the longest somewhere in the middle."""
    n, lo, hi = c["seqs"], c["shortest"], c["tokens"]
    if n == 1:
        return [hi]
    return [int(round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * ((5 * i + 3) % n) / (n - 1)))) for i in range(n)]


def prepare(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if c["op"] in ("chunk", "recurrent"):
        lens = _lengths(c) if c["op"] == "chunk" and c["packed"] else None
        B, T = (1, sum(lens)) if lens else (c["seqs"], c["tokens"] if c["op"] == "chunk" else c["draft"])
        H, HV, D = c["heads"], c["value_heads"], c["dim"]
        N = len(lens) if lens else B
        # queries and keys behind a short convolution and SiLU, heads that forget slowly and quickly
        q, k = (torch.nn.functional.silu(randn(B, T, H, D)) for _ in range(2))
        if not c["layer"]:
            q, k = (x / x.square().sum(-1, keepdim=True).add(EPS).sqrt() for x in (q, k))
        q, k, v = q.to(_BF), k.to(_BF), randn(B, T, HV, D).to(_BF)
        A_log = torch.log(torch.linspace(1.0, 16.0, HV, device=dev))
        dt_bias = torch.log(torch.expm1(torch.exp(torch.linspace(math.log(0.1), math.log(0.001), HV, device=dev))))
        raw, logits = randn(B, T, HV), randn(B, T, HV)
        s = dict(case=c, q=q, k=k, v=v, scale=D ** -0.5)
        if c["op"] == "recurrent":
            if c["layer"]:
                s.update(g=raw.to(_BF), beta=logits.to(_BF), A_log=A_log, dt_bias=dt_bias)
            else:
                s.update(g=-A_log.exp() * torch.nn.functional.softplus(raw + dt_bias), beta=torch.sigmoid(logits), A_log=None, dt_bias=None)
            slots = N * T + N // 4 + 1
            order = torch.randperm(slots, generator=gen, device=dev)[:N * T]
            s["slots"] = order.view(N, T).to(torch.int32)
            # how many of the last call's tokens were accepted: the state to start from
            s["accepted"] = torch.randint(1, T + 1, (N,), generator=gen, device=dev).to(torch.int32)
            s["pool"] = 0.3 * randn(slots, HV, D, D)
            return s
        g, beta = -A_log.exp() * torch.nn.functional.softplus(raw + dt_bias), torch.sigmoid(logits)
        s["cu"] = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev) if lens else None
        s["lens"] = lens
        if lens:      # where a padded batch has its tokens (the plain form works on one)
            at = torch.full((N, max(lens)), -1, dtype=torch.long)
            t0 = 0
            for i, n in enumerate(lens):
                at[i, :n] = torch.arange(t0, t0 + n)
                t0 += n
            s["at"] = at.to(dev)
        if c["train"]:
            s.update(g=g.to(_BF), beta=beta.to(_BF), h0=None, do=randn(B, T, HV, D).to(_BF))
            for n in ("q", "k", "v", "g", "beta"):
                s[n] = s[n].requires_grad_()
        else:
            s.update(g=g, beta=beta, h0=0.3 * randn(N, HV, D, D))
        return s
    rows, cols = c["rows"], c["cols"]
    train = c["train"]
    if c["op"] == "gated":
        s = dict(case=c, x=(2 * randn(rows, cols)).to(_BF), gate=randn(rows, cols).to(_BF), weight=(1 + 0.1 * randn(cols)).to(_BF))
        names = ("x", "gate", "weight")
        s["dy"] = randn(rows, cols).to(_BF) if train else None
    else:
        stream = _BF if c["stream"] == "bf16" else _F
        s = dict(case=c, x=(2 * randn(rows, cols)).to(_BF), residual=(3 * randn(rows, cols)).to(stream), weight=(1 + 0.1 * randn(cols)).to(_BF),
                 post=(1 + 0.1 * randn(cols)).to(_BF) if c["post"] else None, scale=(0.2 + 0.05 * randn(cols)).to(_BF))
        names = ("x", "residual", "weight", "post", "scale")
        s["dy"], s["dr"] = (randn(rows, cols).to(_BF), randn(rows, cols).to(stream)) if train else (None, None)
    s["names"] = [n for n in names if s[n] is not None]
    if train:
        for n in s["names"]:
            s[n] = s[n].requires_grad_()
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------------------------------

def _unit(x):
    return x / (x.square().sum(-1, keepdim=True) + EPS).sqrt()


def _plain_chunks(q, k, v, g, beta, h0, scale):
    """The rule on whole sequences [B, T, H, ...] in 32 bits, 64 tokens at a time: within a chunk the updates are one triangular system."""
    B, T, H, D = q.shape
    pad = -T % CHUNK
    n = (T + pad) // CHUNK

    def cut(x):
        x = torch.nn.functional.pad(x, (0, 0) * (x.dim() - 2) + (0, pad))
        return x.view(B, n, CHUNK, *x.shape[2:]).transpose(2, 3)      # [B, n, H, 64, ...]

    q, k, v, g, beta = (cut(x) for x in (q, k, v, g, beta))
    G = g.double().cumsum(-1)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = torch.exp((G.unsqueeze(-1) - G.unsqueeze(-2)).masked_fill(~low, -math.inf).float())      # of token j's write at token i
    A = (beta.unsqueeze(-1) * decay * (k @ k.transpose(-1, -2))).tril(-1)
    inv = torch.eye(CHUNK, device=q.device).expand_as(A)
    i = torch.arange(CHUNK, device=q.device)
    for b in (1, 2, 4, 8, 16, 32):      # inverse of I + A: blocks of b are inverted, now pairs of them
        off = ((i // (2 * b)).unsqueeze(1) == i // (2 * b)) & ((i // b).unsqueeze(1) != i // b)
        inv = inv - inv @ (A * off) @ inv
    P = decay * (q @ k.transpose(-1, -2)) * scale
    gam = G.exp().float().unsqueeze(-1)
    kg, qg = beta.unsqueeze(-1) * gam * k, scale * gam * q
    kl = torch.exp(G[..., -1:] - G).float().unsqueeze(-1) * k
    vb = beta.unsqueeze(-1) * v
    last = gam[..., -1:, :]
    h, o = h0, []
    for c in range(n):
        w = inv[:, c] @ (vb[:, c] - kg[:, c] @ h)
        o.append(qg[:, c] @ h + P[:, c] @ w)
        h = last[:, c] * h + kl[:, c].transpose(-1, -2) @ w
    return torch.stack(o, 1).transpose(2, 3).reshape(B, n * CHUNK, H, D)[:, :T], h


def _plain_chunk(s):
    c = s["case"]
    q, k, v, g, beta = (s[n].float() for n in ("q", "k", "v", "g", "beta"))
    if c["layer"]:
        q, k = _unit(q), _unit(k)
    grp = c["value_heads"] // c["heads"]
    q, k = q.repeat_interleave(grp, 2), k.repeat_interleave(grp, 2)
    if s["lens"]:      # a padded batch; its empty places neither write nor decay
        there = s["at"] >= 0
        q, k, v, g, beta = (x[0][s["at"].clamp(min=0)] * there.view(*there.shape, *[1] * (x.dim() - 2)) for x in (q, k, v, g, beta))
    h0 = s["h0"] if s["h0"] is not None else torch.zeros(q.shape[0], c["value_heads"], c["dim"], c["dim"], device=q.device)
    o, h = _plain_chunks(q, k, v, g, beta, h0, s["scale"])
    if s["lens"]:
        o = o[there].unsqueeze(0)
    return o.to(_BF), h


def _plain_recurrent(s):
    c = s["case"]
    q, k, v, g, beta = (s[n].float() for n in ("q", "k", "v", "g", "beta"))
    if c["layer"]:
        q, k = _unit(q), _unit(k)
        g, beta = -s["A_log"].exp() * torch.nn.functional.softplus(g + s["dt_bias"]), torch.sigmoid(beta)
    grp = c["value_heads"] // c["heads"]
    q, k = q.repeat_interleave(grp, 2), k.repeat_interleave(grp, 2)
    slots = s["slots"].long()
    h = s["pool"][slots.gather(1, s["accepted"].long().unsqueeze(1) - 1)[:, 0]]
    o = []
    for t in range(c["draft"]):
        h = h * g[:, t].exp()[..., None, None]
        w = beta[:, t].unsqueeze(-1) * (v[:, t] - (k[:, t].unsqueeze(-1) * h).sum(-2))
        h = h + k[:, t].unsqueeze(-1) * w.unsqueeze(-2)
        o.append(s["scale"] * (q[:, t].unsqueeze(-1) * h).sum(-2))
        s["pool"][slots[:, t]] = h
    return torch.stack(o, 1).to(_BF), s["pool"]


def _rms(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _plain_gated(s):
    z = s["gate"].float()
    return (_rms(s["x"].float()) * s["weight"].float() * torch.sigmoid(z) * (z if s["case"]["act"] == "silu" else 1.0)).to(_BF)


def _plain_residual(s):
    x = s["x"].float()
    if s["post"] is not None:
        x = _rms(x) * s["post"].float()
    r = s["residual"].float() + s["scale"].float() * x
    return (_rms(r) * s["weight"].float()).to(_BF), r.to(s["residual"].dtype)


# ---- one pass -------------------------------------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        import kda_b200 as K
    if c["op"] == "recurrent":
        if not own:
            return _plain_recurrent(s)
        o, pool = K.fused_recurrent_gated_delta_fwd(
            s["q"], s["k"], s["v"], s["g"], s["beta"], A_log=s["A_log"], dt_bias=s["dt_bias"], initial_state=s["pool"], scale=s["scale"],
            ssm_state_indices=s["slots"], num_accepted_tokens=s["accepted"], use_qk_l2norm_in_kernel=c["layer"], use_gate_in_kernel=c["layer"],
            use_beta_sigmoid_in_kernel=c["layer"])
        return o, pool
    if c["op"] == "chunk":
        if own:
            o, h = K.chunk_gated_delta(s["q"], s["k"], s["v"], s["g"], s["beta"], scale=s["scale"], initial_state=s["h0"], output_final_state=not c["train"],
                                       use_qk_l2norm_in_kernel=c["layer"], cu_seqlens=s["cu"])
        else:
            o, h = _plain_chunk(s)
        if not c["train"]:
            return o, h
        return (o.detach(),) + torch.autograd.grad(o, [s[n] for n in ("q", "k", "v", "g", "beta")], s["do"])
    if c["op"] == "gated":
        y = K.gated_rms_norm(s["x"], s["gate"], s["weight"], eps=EPS, activation=c["act"]) if own else _plain_gated(s)
        if not c["train"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, [s[n] for n in s["names"]], s["dy"])
    y, r = K.residual_rms_norm(s["x"], s["residual"], s["weight"], scale=s["scale"], post_weight=s["post"], eps=EPS) if own else _plain_residual(s)
    if not c["train"]:
        return y, r
    return (y.detach(), r.detach()) + torch.autograd.grad((y, r), [s[n] for n in s["names"]], (s["dy"], s["dr"]))


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------------

def work(c):
    if c["op"] in ("chunk", "recurrent"):
        lens = _lengths(c) if c["op"] == "chunk" and c["packed"] else [c["tokens"] if c["op"] == "chunk" else c["draft"]] * c["seqs"]
        tokens, H, HV, D = sum(lens), c["heads"], c["value_heads"], c["dim"]
        if c["op"] == "recurrent":
            moved = 4 * D * D * HV * c["seqs"] * (1 + c["draft"])      # the states: one read per sequence, one write per token
            small = 2 * tokens * D * (2 * H + 2 * HV) + tokens * HV * (4 if c["layer"] else 8)
            return dict(bytes=moved + small, flops=tokens * HV * 7 * D * D)
        per = 2 * D * (2 * H + 2 * HV) + (4 if c["train"] else 8) * HV      # q, k, v, g, beta in, o out
        products = 2 * D * (2 * CHUNK + 3 * D) + 4 * CHUNK * D               # with keys; with the state; with the chunk's own values
        if c["train"]:
            return dict(bytes=tokens * (per + 2 * D * (4 * H + 4 * HV) - 2 * D * HV + 8 * HV + 2 * D * HV), flops=tokens * HV * 3 * products)
        return dict(bytes=tokens * per + 8 * D * D * HV * len(lens), flops=tokens * HV * products)
    n = c["rows"] * c["cols"]
    if c["op"] == "gated":      # x, gate in, y out; with gradients dy in, dx, dgate out and x, gate once more
        return dict(bytes=n * 2 * (8 if c["train"] else 3), flops=n * (30 if c["train"] else 8))
    w = 2 if c["stream"] == "bf16" else 4
    # x, residual in, y, r out; with gradients dy, dr in, dx, dresidual out and (their norms' inputs) r and, with a norm or a scale of its own, x once more
    return dict(bytes=n * (2 + w + 2 + w) + (n * (2 + w + 2 + w + w + 2) if c["train"] else 0), flops=n * (30 if c["train"] else 10))


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------------------

def _steps(c, s):
    """Inputs as [tokens, sequences, value heads, ...] in 64 bits with nothing in the places behind a sequence's end, and how to get back."""
    q, k, v, g, beta = (s[n].detach().double() for n in ("q", "k", "v", "g", "beta"))
    grp = c["value_heads"] // c["heads"]
    rq = rk = None
    if c["layer"]:
        rq, rk = ((x * x).sum(-1, keepdim=True).add(EPS).rsqrt() for x in (q, k))
        q, k = q * rq, k * rk
    raw = (q, k, rq, rk)
    q, k = q.repeat_interleave(grp, 2), k.repeat_interleave(grp, 2)
    lens = s.get("lens")

    def lay(x):
        if not lens:
            return x.transpose(0, 1).contiguous()
        out = torch.zeros(max(lens), len(lens), *x.shape[2:], dtype=torch.float64, device=x.device)
        t0 = 0
        for i, n in enumerate(lens):
            out[:n, i] = x[0, t0:t0 + n]
            t0 += n
        return out

    def back(x):
        return torch.cat([x[:n, i] for i, n in enumerate(lens)]).unsqueeze(0) if lens else x.transpose(0, 1)

    return [lay(x) for x in (q, k, v, g, beta)], back, raw


def _exact_rule(c, s):
    (q, k, v, g, beta), back, (qn, kn, rq, rk) = _steps(c, s)
    T, N, H, D = q.shape
    scale, a = s["scale"], g.exp()[..., None, None]
    S = s["h0"].double() if s["h0"] is not None else torch.zeros(N, H, D, D, dtype=torch.float64, device=q.device)

    def step(S, t):
        P = S * a[t]
        u = v[t] - torch.einsum("nhkv,nhk->nhv", P, k[t])
        return P, u, torch.addcmul(P, k[t].unsqueeze(-1), (beta[t].unsqueeze(-1) * u).unsqueeze(-2))

    o, every, marks = torch.empty_like(v), 64, []
    for t in range(T):
        if c["train"] and t % every == 0:
            marks.append(S)
        S = step(S, t)[2]
        o[t] = scale * torch.einsum("nhkv,nhk->nhv", S, q[t])
    if not c["train"]:
        return back(o), S
    do = (lambda x: x.transpose(0, 1) if not s["lens"] else None)(s["do"].double())
    if s["lens"]:
        do = torch.zeros_like(v)
        t0 = 0
        for i, n in enumerate(s["lens"]):
            do[:n, i] = s["do"][0, t0:t0 + n].double()
            t0 += n
    dq, dk, dv, dg, db = (torch.empty_like(x) for x in (q, k, v, g, beta))
    dS = torch.zeros_like(S)
    for m in range(len(marks) - 1, -1, -1):
        t0, t1 = m * every, min(T, (m + 1) * every)
        kept, S = [], marks[m]
        for t in range(t0, t1):
            P, u, S = step(S, t)
            kept.append((P, u, S))
        for t in range(t1 - 1, t0 - 1, -1):
            P, u, S = kept[t - t0]
            dS = torch.addcmul(dS, (scale * q[t]).unsqueeze(-1), do[t].unsqueeze(-2))
            dq[t] = scale * torch.einsum("nhkv,nhv->nhk", S, do[t])
            dw = torch.einsum("nhkv,nhk->nhv", dS, k[t])
            du = beta[t].unsqueeze(-1) * dw
            db[t] = (dw * u).sum(-1)
            dv[t] = du
            dk[t] = torch.einsum("nhkv,nhv->nhk", dS, beta[t].unsqueeze(-1) * u) - torch.einsum("nhkv,nhv->nhk", P, du)
            dS = torch.addcmul(dS, k[t].unsqueeze(-1), du.unsqueeze(-2), value=-1)
            dg[t] = (dS * P).sum((-1, -2))
            dS = dS * a[t]
    dq, dk, dv, dg, db = (back(x) for x in (dq, dk, dv, dg, db))
    hq = c["heads"]
    dq, dk = (x.reshape(*x.shape[:2], hq, -1, D).sum(3) for x in (dq, dk))
    if c["layer"]:      # through the rows' normalisation
        dq, dk = rq * (dq - qn * (qn * dq).sum(-1, keepdim=True)), rk * (dk - kn * (kn * dk).sum(-1, keepdim=True))
    return back(o), dq, dk, dv, dg, db


def _exact_decode(c, s):
    if c["layer"]:
        z = s["g"].double() + s["dt_bias"].double()
        s = dict(s, g=-s["A_log"].double().exp() * torch.logaddexp(z, torch.zeros_like(z)), beta=1 / (1 + (-s["beta"].double()).exp()))
    (q, k, v, g, beta), back, _ = _steps(c, s)
    pool, o = s["pool"].double(), torch.empty_like(v)
    S = torch.stack([pool[s["slots"][n, s["accepted"][n] - 1]] for n in range(c["seqs"])])
    for t in range(c["draft"]):
        S = S * g[t].exp()[..., None, None]
        S = S + torch.einsum("nhk,nhv->nhkv", k[t], beta[t].unsqueeze(-1) * (v[t] - torch.einsum("nhkv,nhk->nhv", S, k[t])))
        o[t] = s["scale"] * torch.einsum("nhkv,nhk->nhv", S, q[t])
        pool.index_copy_(0, s["slots"][:, t].long(), S)
    return back(o), pool


def _exact_norms(c, s):
    t = {n: s[n].detach().double() for n in s["names"]}
    D, x = c["cols"], t["x"]

    def through(d, y, rstd):      # gradient of y = x rstd(x) with respect to x
        return rstd * (d - y * (d * y).sum(-1, keepdim=True) / D)

    rstd = (x.pow(2).sum(-1, keepdim=True) / D + EPS).pow(-0.5)
    n = x * rstd
    if c["op"] == "gated":
        sg = 1 / (1 + (-t["gate"]).exp())
        act, dact = (t["gate"] * sg, sg * (1 + t["gate"] * (1 - sg))) if c["act"] == "silu" else (sg, sg * (1 - sg))
        y = n * t["weight"] * act
        if not c["train"]:
            return y
        d = s["dy"].double()
        return y, through(d * t["weight"] * act, n, rstd), d * n * t["weight"] * dact, (d * n * act).sum(0)
    b = n * t["post"] if c["post"] else x
    r = t["residual"] + t["scale"] * b
    rr = (r.pow(2).sum(-1, keepdim=True) / D + EPS).pow(-0.5)
    y = r * rr * t["weight"]
    if not c["train"]:
        return y, r
    d = s["dy"].double()
    dr = s["dr"].double() + through(d * t["weight"], r * rr, rr)
    db = dr * t["scale"]
    found = [through(db * t["post"], n, rstd) if c["post"] else db, dr, (d * r * rr).sum(0)]
    if c["post"]:
        found.append((db * n).sum(0))
    return (y, r, *found, (dr * b).sum(0))


def exact(c, seed):
    with torch.no_grad():
        s = prepare(c, seed)
        return _exact_rule(c, s) if c["op"] == "chunk" else _exact_decode(c, s) if c["op"] == "recurrent" else _exact_norms(c, s)
