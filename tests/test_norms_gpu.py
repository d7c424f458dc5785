"""The norms around a block against float64 and its autograd.

Tolerances, relative in the 2-norm.  Inputs count as they are; inside, everything is float32: a sum over n columns in a tree of at most 8 sequential additions and
log2 levels, products and a reciprocal square root of 2 ulp -- below 2^-19 of the terms for up to 8192 columns.  A bf16 result adds its rounding, 2^-8.  A gradient
through a norm subtracts a mean (dn - n mean(dn n)): its terms are at most twice dn, 2^-17.  Sums over rows (float32, at most 2^17 rows here in at most
148 * 512 partial sums of 2^10 sequential additions): 2^-24 * 2^11 of the terms' absolute sum, which for random signs is up to sqrt(rows) of the result: the
tests compare them with the absolute sum."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32
SHAPES = [(1, 1), (3, 7), (5, 8), (100, 77), (33, 96), (1000, 128), (17, 256), (9, 257), (4, 1000), (5, 1001), (3, 4096), (2, 4100), (3, 8191), (2, 8192)]
RING = [(300000, 8), (300001, 7), (30001, 77), (25000, 96), (16385, 128), (16384, 128), (9001, 256), (8200, 257), (2101, 1000), (2100, 1001), (860, 2500), (520, 4096), (513, 4100),
        (261, 8191), (257, 8192)]

RING_FORWARD = [(1200001, 7), (110000, 77), (65537, 128), (8400, 1000), (8387, 1001), (3361, 2500), (2101, 4096), (2049, 4100), (1027, 8191), (1026, 8192)]

@pytest.fixture(scope="module", autouse=True)
def leave_no_memory():
    yield
    gc.collect()
    torch.cuda.empty_cache()


def tol(dtype):
    return 2.0 ** -17 + (2.0 ** -8 if dtype == BF else 0.0)


def close(x, ref, what, scale=None):
    """scale: what the error is relative to, where that is not the result itself"""
    assert x.shape == ref.shape and torch.isfinite(x.float()).all(), what
    err, size = (x.double() - ref).norm(), ref.norm() if scale is None else scale.norm()
    extra = 2.0 ** -8 * ref.norm() if x.dtype == BF and scale is not None else 0.0
    assert float(err) <= (tol(x.dtype) if scale is None else 2.0 ** -13) * float(size) + extra, (what, float(err / size))


def inputs(rows, cols, seed, *types):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(*((rows, cols) if big else (cols,)), generator=gen, device="cuda").add_(0.0 if big else 1.0).to(t).requires_grad_() for big, t in types]


def gated_ref(x, z, w, eps, act):
    s = torch.sigmoid(z)
    return x * (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * (w if w is not None else 1.0) * (z * s if act == "silu" else s)


def residual_ref(x, r, w, s, p, eps):
    rms = lambda t: t * (t.pow(2).mean(-1, keepdim=True) + eps).rsqrt()      # noqa: E731
    r = r + s * (rms(x) * p if p is not None else x)
    return rms(r) * w, r


def check_gated(rows, cols, types, act, seed, weight=True, eps=1e-6):
    from kda_b200 import gated_rms_norm
    x, z, w = inputs(rows, cols, seed, (True, types[0]), (True, types[1]), (False, types[2]))
    w = w if weight else None
    leaves = [t for t in (x, z, w) if t is not None]
    dy = torch.randn(rows, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 1)).to(types[0])
    y = gated_rms_norm(x, z, w, eps=eps, activation=act)
    got = torch.autograd.grad(y, leaves, dy)
    L = [t.detach().double().requires_grad_() for t in leaves]
    ref = gated_ref(L[0], L[1], L[2] if weight else None, eps, act)
    grads = torch.autograd.grad(ref, L, dy.double())
    assert y.dtype == types[0] and all(g.dtype == t.dtype for g, t in zip(got, leaves))
    close(y, ref, "y")
    close(got[0], grads[0], "dx", scale=None if cols > 1 else dy.double())      # one column: x / |x| does not move
    close(got[1], grads[1], "dgate")
    if weight:
        terms = (dy.double() * gated_ref(L[0], L[1], None, eps, act)).abs().sum(0)
        close(got[2], grads[2], "dweight", scale=terms)
    with torch.no_grad():
        assert torch.equal(gated_rms_norm(x, z, w, eps=eps, activation=act), y)


def check_residual(rows, cols, types, post, scale, seed, eps=1e-6):
    from kda_b200 import residual_rms_norm
    x, r, w, s, p = inputs(rows, cols, seed, (True, types[0]), (True, types[1]), (False, types[2]), (False, types[2]), (False, types[0]))
    p, s = p if post else None, s if scale is None else scale
    leaves = [t for t in (x, r, w, s, p) if isinstance(t, torch.Tensor)]
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    dy, dr = (torch.randn(rows, cols, device="cuda", generator=gen).to(t) for t in types[:2])
    y, out = residual_rms_norm(x, r, w, scale=s, post_weight=p, eps=eps)
    got = dict(zip([id(t) for t in leaves], torch.autograd.grad((y, out), leaves, (dy, dr))))
    L = {id(t): t.detach().double().requires_grad_() for t in leaves}
    at = lambda t: L.get(id(t), t)      # noqa: E731
    ref, rout = residual_ref(at(x), at(r), at(w), at(s), at(p), eps)
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad((ref, rout), [L[id(t)] for t in leaves], (dy.double(), dr.double()))))
    assert y.dtype == types[0] and out.dtype == types[1]
    close(y, ref, "y")
    close(out, rout, "r")
    with torch.no_grad():
        rms = lambda t: (t.pow(2).mean(-1, keepdim=True) + eps).rsqrt()      # noqa: E731
        n1 = at(x) * rms(at(x)) if post else at(x)
        b = n1 * at(p) if post else n1
        t = grads[id(r)]
        # where gradients cancel (a norm takes out what lies along its row) errors are relative to what went in
        into = dr.double().abs() + (dy.double() * at(w) * rms(rout)).abs()
    close(got[id(r)], grads[id(r)], "dresidual", scale=into)
    close(got[id(x)], grads[id(x)], "dx", scale=(into * at(s)).abs() * (at(p) * rms(at(x)) if post else 1.0))
    close(got[id(w)], grads[id(w)], "dweight", scale=(dy.double() * rout * rms(rout)).abs().sum(0))
    if scale is None:
        close(got[id(s)], grads[id(s)], "dscale", scale=(into * b.abs()).sum(0))
    if post:
        close(got[id(p)], grads[id(p)], "dpost_weight", scale=(into * (at(s) * n1).abs()).sum(0))
    assert t.shape == r.shape


@pytest.mark.parametrize("rows,cols", SHAPES + RING + RING_FORWARD)
def test_gated(rows, cols):
    check_gated(rows, cols, (BF, BF, BF), "silu" if rows % 2 else "sigmoid", seed=rows + cols)


@pytest.mark.parametrize("rows,cols", [(50, 128), (9, 1001), (16400, 128), (2100, 1001)])
@pytest.mark.parametrize("types", [(F, F, F), (BF, F, F), (F, BF, BF)])
def test_gated_types(rows, cols, types):
    check_gated(rows, cols, types, "silu", seed=3)
    check_gated(rows, cols, types, "sigmoid", seed=4, weight=False, eps=1e-3)


@pytest.mark.parametrize("rows,cols", SHAPES + RING + RING_FORWARD)
def test_residual(rows, cols):
    check_residual(rows, cols, (BF, F if rows % 2 else BF, BF), post=cols % 2 == 0, scale=None if rows % 3 else 0.7, seed=rows + cols)


@pytest.mark.parametrize("rows,cols", [(50, 128), (9, 1001), (3, 4096), (16400, 128), (520, 4096)])
@pytest.mark.parametrize("types", [(F, F, F), (BF, F, F), (F, BF, BF)])
@pytest.mark.parametrize("post", [False, True])
def test_residual_types(rows, cols, types, post):
    check_residual(rows, cols, types, post, None, seed=5)


@pytest.mark.parametrize("rows", [40, 20000])
def test_one_gradient_is_missing(rows):
    from kda_b200 import residual_rms_norm
    x, r, w = inputs(rows, 128, 7, (True, BF), (True, F), (False, BF))
    g = torch.randn(rows, 128, device="cuda")
    y, out = residual_rms_norm(x, r, w)
    a = torch.autograd.grad(y, (x, r, w), g.to(BF), retain_graph=True)
    b = torch.autograd.grad(out, (x, r), g, retain_graph=True)
    both = torch.autograd.grad((y, out), (x, r, w), (g.to(BF), g))
    close(both[1], a[1].double() + b[1].double(), "dresidual", scale=a[1].double().abs() + b[1].double().abs())
    assert torch.equal(a[2], both[2]) and torch.equal(b[1], g)


def test_strided_inputs_and_odd_addresses():
    from kda_b200 import gated_rms_norm
    x, z, w = (t.detach() for t in inputs(64, 256, 8, (True, BF), (True, BF), (False, BF)))
    y = gated_rms_norm(x, z, w)
    wide = torch.cat([x, z], -1)
    assert torch.equal(gated_rms_norm(wide[:, :256], wide[:, 256:], w), y)
    shift = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)      # noqa: E731
    odd = gated_rms_norm(shift(x), shift(z), shift(w))
    close(odd, y.double(), "odd")
    big, gate = (torch.randn(20000, 128, device="cuda").to(BF) for _ in range(2))
    close(gated_rms_norm(shift(big), shift(gate)), gated_rms_norm(big, gate).double(), "odd, many rows")
    assert torch.equal(gated_rms_norm(x.view(4, 16, 256), z.view(4, 16, 256), w).view(64, 256), y)


@pytest.mark.parametrize("rows", [5, 20000])
def test_bad_rows_stay_alone(rows):
    """A row of NaN or infinities, and a row of zeros, leave the others as they are."""
    from kda_b200 import residual_rms_norm
    x, r, w = (t.detach() for t in inputs(rows, 128, 9, (True, BF), (True, BF), (False, BF)))
    y, out = residual_rms_norm(x, r, w, post_weight=w)
    x[1], x[2], r[3] = float("nan"), float("inf"), 0
    x[3] = 0
    y2, out2 = residual_rms_norm(x, r, w, post_weight=w)
    keep = [i for i in range(rows) if i not in (1, 2, 3)]
    assert torch.equal(y[keep], y2[keep]) and torch.equal(out[keep], out2[keep])
    assert not y2[3].any() and y2[1].isnan().all()


def test_same_bits_again():
    from kda_b200 import residual_rms_norm
    leaves = inputs(20000, 256, 10, (True, BF), (True, F), (False, BF), (False, BF), (False, BF))
    gy, gr = torch.randn(20000, 256, device="cuda").to(BF), torch.randn(20000, 256, device="cuda")
    x, r, w, s, p = leaves
    runs = [torch.autograd.grad(residual_rms_norm(x, r, w, s, p), leaves, (gy, gr)) for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@pytest.mark.captures_graph
@pytest.mark.parametrize("rows", [48, 20000])
def test_replays_from_a_graph(rows):
    from kda_b200 import gated_rms_norm
    x, z, w = (t.detach() for t in inputs(rows, 128, 11, (True, BF), (True, BF), (False, BF)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        gated_rms_norm(x, z, w)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = gated_rms_norm(x, z, w)
    x.copy_(torch.randn_like(x))
    g.replay()
    assert torch.equal(y, gated_rms_norm(x, z, w))


def test_empty_and_refusals():
    from kda_b200 import gated_rms_norm, residual_rms_norm
    x = torch.zeros(0, 128, device="cuda", dtype=BF, requires_grad=True)
    w = torch.ones(128, device="cuda", requires_grad=True)
    y = gated_rms_norm(x, x.detach(), w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 128) and dx.shape == x.shape and not dw.any()
    x = torch.zeros(4, 128, device="cuda", dtype=BF)
    w = torch.ones(128, device="cuda", dtype=BF)
    with pytest.raises(RuntimeError):
        gated_rms_norm(x.cpu(), x.cpu())
    with pytest.raises(ValueError):
        gated_rms_norm(x, x[:2])
    with pytest.raises(ValueError):
        gated_rms_norm(x, x, w[:64])
    with pytest.raises(ValueError):
        gated_rms_norm(x, x, activation="tanh")
    with pytest.raises(ValueError):
        residual_rms_norm(x, x.cpu(), w)
    with pytest.raises(ValueError):
        residual_rms_norm(x, x, w, scale=torch.ones(4, device="cuda"))
    with pytest.raises(NotImplementedError):
        gated_rms_norm(x.half(), x.half())
    with pytest.raises(NotImplementedError):
        residual_rms_norm(torch.zeros(2, 8200, device="cuda"), torch.zeros(2, 8200, device="cuda"), torch.zeros(8200, device="cuda"))
    with pytest.raises(NotImplementedError):
        a = x.clone().requires_grad_()
        torch.autograd.grad(gated_rms_norm(a, x), a, x, create_graph=True)
