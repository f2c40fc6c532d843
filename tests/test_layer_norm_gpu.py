"""Layer norm and its gradients against their definition in 64 bits.

Bounds.  u = 2**-24.  The mean of D values is off by at most (log2 D + 8) u of the mean magnitude (sums of threads of up to 32 values, then a tree), and is
corrected; with d = x - mean exact to u |x|, y carries some (16 + log2 D) u of |n| and of max|x| / sigma, times |w|, and the type's half step.
The same holds for the two sums of dx.  A sum over rows has at most `rows` terms in fp32: rows u of the sum of magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def draw(S, D, dtype, seed=0, mean=0.5, std=1.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    return [(n(S, D) * std + mean).to(dtype), n(S, D).to(dtype), (1 + 0.3 * n(D)), 0.3 * n(D), n(S, D).to(dtype), n(S, D).to(dtype)]


def defined(h, w, b, eps, dy, dh):
    """Y, dH, dw, db and their bounds, in 64 bits."""
    D = h.shape[-1]
    h, w, b, dy = (None if t is None else t.double() for t in (h, w, b, dy))
    mu = h.mean(-1, keepdim=True)
    rstd = 1 / ((h - mu).square().mean(-1, keepdim=True) + eps).sqrt()
    n = (h - mu) * rstd
    ww = torch.ones_like(h[0]) if w is None else w
    k = (16 + math.log2(D)) * U
    slack = k * (n.abs() + h.abs().amax(-1, keepdim=True) * rstd)   # of n
    y = n * ww + (0 if b is None else b)
    by = slack * ww.abs() + 2 * U * y.abs()
    g = dy * ww
    c1, c2 = g.mean(-1, keepdim=True), (g * n).mean(-1, keepdim=True)
    dx = rstd * (g - c1 - n * c2)
    size = rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    bx = 2 * k * size + rstd * (slack * c2.abs() + n.abs() * (g.abs() * slack).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.double()
        bx = bx + 2 * U * dx.abs()
    rows = h.shape[0]
    dw, db = (dy * n).sum(0), dy.sum(0)
    bw = rows * U * (dy * n).abs().sum(0) + (dy.abs() * slack).sum(0)
    bb = rows * U * dy.abs().sum(0)
    return (y, dx, dw, db), (by, bx, bw, bb)


def check(got, want, bound, what):
    t = half(got.dtype)
    bound = bound + t * (want.abs() + bound) + torch.finfo(got.dtype).tiny * t
    off = (got.double() - want).abs()
    assert got.shape == want.shape and bool((off <= bound).all()), f"{what}: {float((off / bound).max()):.2f} of the bound"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("own", [True, False])   # weights in the rows' type, or float32
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("S,D", [(1, 1), (1, 8), (3, 7), (9, 256), (70, 200), (5, 257), (33, 1000), (4, 1001), (300, 1024), (40, 2056), (11, 4096), (6, 8192), (5, 8200), (3, 9001),
                                 (2, 16385), (3, 40000)])
def test_forward_and_gradients(S, D, residual, own, dtype):
    import paralleltnnlayers_b200 as P
    x, r, w, b, dy, dh = draw(S, D, dtype, seed=S + D)
    if own:
        w, b = w.to(dtype), b.to(dtype)
    leaves = [t.requires_grad_() for t in ((x, r, w, b) if residual else (x, w, b))]
    out = P.LayerNormFunction.apply(x, w, b, 1e-5, r if residual else None)
    y, h = out if residual else (out, x)
    if residual:
        assert torch.equal(h.detach(), (x.detach().float() + r.detach().float()).to(dtype))
    (wy, wx, ww, wb), (by, bx, bw, bb) = defined(h.detach(), w.detach(), b.detach(), 1e-5, dy, dh if residual else None)
    check(y.detach(), wy, by, "y")
    grads = torch.autograd.grad(out, leaves, (dy, dh) if residual else dy)
    check(grads[0], wx, bx, "dx")
    if residual:
        assert torch.equal(grads[0], grads[1])
    check(grads[-2], ww, bw, "dw")
    check(grads[-1], wb, bb, "db")
    plain = P.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5, r.detach() if residual else None)
    assert torch.equal(plain[0] if residual else plain, y.detach())


@pytest.mark.parametrize("S,D", [(2000, 64), (2500, 300), (700, 1536), (1200, 4096), (400, 9000)])
def test_many_rows(S, D):
    """Rows of several turns of every CTA."""
    import paralleltnnlayers_b200 as P
    x, _, w, b, dy, _ = draw(S, D, torch.float32, seed=D)
    y, mean, rstd = P.layer_norm_save(x, w, b, 1e-5)
    d = P.layer_norm_backward(dy, x, w, b, mean, rstd)
    want, bound = defined(x, w, b, 1e-5, dy, None)
    for got, v, e, what in zip((y, *d), want, bound, ("y", "dx", "dw", "db")):
        check(got, v, e, what)
    again = P.layer_norm_backward(dy, x, w, b, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(d, again))


@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("residual", [False, True])
def test_without_weight_or_bias(weight, bias, residual):
    import paralleltnnlayers_b200 as P
    x, r, w, b, dy, dh = draw(37, 344, torch.float32)
    w, b, r = w if weight else None, b if bias else None, r if residual else None
    leaves = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
    out = P.LayerNormFunction.apply(x, w, b, 1e-6, r)
    y, h = out if residual else (out, x)
    want, bound = defined(h.detach(), None if w is None else w.detach(), None if b is None else b.detach(), 1e-6, dy, dh if residual else None)
    check(y.detach(), want[0], bound[0], "y")
    grads = list(torch.autograd.grad(out, leaves, (dy, dh) if residual else dy))
    check(grads[0], want[1], bound[1], "dx")
    if weight:
        check(grads[1], want[2], bound[2], "dw")
    if bias:
        check(grads[1 + weight], want[3], bound[3], "db")
    # one gradient alone, of each leaf, and through one of two results
    for leaf, g in zip(leaves, grads):
        out = P.LayerNormFunction.apply(x, w, b, 1e-6, r)
        assert torch.equal(torch.autograd.grad(out, leaf, (dy, dh) if residual else dy)[0], g)
    if residual:
        for k, d in ((0, dy), (1, dh)):
            out = P.LayerNormFunction.apply(x, w, b, 1e-6, r)
            got, = torch.autograd.grad(out[k], r, d)
            if k:
                assert torch.equal(got, dh)
            else:
                check(got, *[v[1] for v in defined(h.detach(), None if w is None else w.detach(), None, 1e-6, dy, None)], "dr")


def test_against_differences():
    import paralleltnnlayers_b200 as P
    x, r, w, b, dy, dh = draw(3, 24, torch.float32, seed=5)
    f = lambda x, w, b, r: sum((p.double() * q.double()).sum() for p, q in zip(P.layer_norm(x, w, b, 1e-5, r), (dy, dh)))  # noqa: E731
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    grads = torch.autograd.grad(P.LayerNormFunction.apply(x, w, b, 1e-5, r), leaves, (dy, dh))
    # step 2**-6: the third derivative gives some 2**-12, the rounding of 144 values of size 4 in fp32 2**-22 * 4 * 12 / 2**-5
    gen = torch.Generator(device="cuda").manual_seed(1)
    for k, g in enumerate(grads):
        v = torch.randn(g.shape, generator=gen, device="cuda")
        at = lambda e: f(*[t.detach() + e * v if i == k else t.detach() for i, t in enumerate((x, w, b, r))])  # noqa: E731,B023
        slope = (at(2.0 ** -6) - at(-2.0 ** -6)) / 2.0 ** -5
        assert abs(float(slope) - float((g.double() * v.double()).sum())) < 2e-2 * float(g.double().norm() * v.double().norm()) / 3


@pytest.mark.parametrize("dtype", TYPES)
def test_a_far_mean(dtype):
    """Deviations are what is squared: a mean far above them costs nothing but the rounding of the values themselves."""
    import paralleltnnlayers_b200 as P
    x = (1000 + torch.randn(20, 777, device="cuda")).to(dtype)
    y = P.layer_norm(x)
    (want, _, _, _), (bound, _, _, _) = defined(x, None, None, 1e-5, x, None)
    check(y, want, bound, "y")
    assert float((y.double() - want).abs().max()) < 2e-3 + 4 * half(dtype)


def test_rows_that_are_constant_or_not_finite():
    import paralleltnnlayers_b200 as P
    for D in (40, 1000, 20000):
        x = torch.randn(5, D, device="cuda")
        want = P.layer_norm(x)
        z = x.clone()
        z[1] = 3.5
        z[2, 7], z[3, 9] = float("inf"), float("nan")
        y = P.layer_norm(z)
        assert not y[1].any() and y[2].isnan().all() and y[3].isnan().all()
        assert torch.equal(y[0], want[0]) and torch.equal(y[4], want[4])
        w = torch.randn(D, device="cuda", requires_grad=True)
        z[2:4] = 3.5
        z.requires_grad_()
        dz, dw = torch.autograd.grad(P.LayerNormFunction.apply(z, w), (z, w), torch.ones_like(z))
        assert dz.isfinite().all() and dw.isfinite().all()


def test_no_rows_views_and_shapes():
    import paralleltnnlayers_b200 as P
    w = torch.randn(24, device="cuda", requires_grad=True)
    x = torch.zeros(0, 24, device="cuda", requires_grad=True)
    y = P.LayerNormFunction.apply(x, w, w * 2)
    assert y.shape == (0, 24)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros(0, 24, device="cuda"))
    assert dx.shape == (0, 24) and not dw.any()
    x = torch.randn(4, 48, 6, device="cuda").transpose(1, 2)
    assert torch.equal(P.layer_norm(x, eps=1e-3), P.layer_norm(x.contiguous(), eps=1e-3))
    assert P.layer_norm(torch.randn(48, device="cuda")).shape == (48,)
    odd = torch.randn(4 * 48 + 1, device="cuda")[1:].view(4, 48)   # (rows off their boundary)
    (want, _, _, _), (bound, _, _, _) = defined(odd, None, None, 1e-5, odd, None)
    check(P.layer_norm(odd), want, bound, "y")


def test_streams_and_graphs():
    import paralleltnnlayers_b200 as P
    x, r, w, b, dy, dh = draw(900, 520, torch.bfloat16)
    w, b = w.bfloat16(), b.bfloat16()
    y, h, mean, rstd = P.layer_norm_save(x, w, b, 1e-5, r)
    want = P.layer_norm_backward(dy, h, w, b, mean, rstd, dh)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = P.layer_norm_backward(dy, h, w, b, mean, rstd, dh)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
            o = P.layer_norm_save(x, w, b, 1e-5, r)
            d = P.layer_norm_backward(dy, o[1], w, b, o[2], o[3], dh)
        graphs.append((g, o, d))
    for k in (0, 1, 0):
        graphs[k][0].replay()
        assert torch.equal(graphs[k][1][0], y) and all(torch.equal(p, q) for p, q in zip(graphs[k][2], want))
