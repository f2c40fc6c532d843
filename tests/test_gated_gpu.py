"""The gated feed-forward block against its definition in 64 bits.

Bounds, for each entry.  e = finfo(type).eps / 2 is a rounding to the type, u = 2**-23 an addition of the tensor core (which may cut its sum off).  G and U
are sums of I products: eG = (I + 2) u |X| |Wg|.  act has slopes below 1.13 and curvatures below 1; its exponential is off by (|G| + 8) u of itself.  The
backward rounds dG and dU once, e, and sums 2 F (dX) or `rows` (dW) products of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
BF16, F16 = torch.bfloat16, torch.float16
ACTS = ["silu", "gelu", "gelu_tanh"]


def _p():
    import paralleltnnlayers_b200 as P
    return P


def inputs(rows, I, F, dtype, seed=0, std=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s, std=1.0: (torch.randn(*s, generator=gen, device="cuda") * std).to(dtype)  # noqa: E731
    return {"x": n(rows, I, std=std), "Wg": n(I, F, std=I ** -0.5), "Wu": n(I, F, std=I ** -0.5), "dh": n(rows, F)}


def act64(act, G):
    if act == "silu":
        return torch.nn.functional.silu(G)
    return torch.nn.functional.gelu(G, approximate="tanh" if act == "gelu_tanh" else "none")


def definition(t, act):
    x, Wg, Wu, dh = (t[k].double() for k in ("x", "Wg", "Wu", "dh"))
    rows, I = x.shape
    F = Wg.shape[1]
    e, tiny = torch.finfo(t["x"].dtype).eps / 2, torch.finfo(t["x"].dtype).smallest_normal * torch.finfo(t["x"].dtype).eps
    G, V = (x @ Wg).requires_grad_(), x @ Wu
    eG, eU = ((I + 2) * U * x.abs() @ w.abs() for w in (Wg, Wu))
    a = act64(act, G)
    slope = torch.autograd.grad(a.sum(), G)[0]
    G, a = G.detach(), a.detach()
    rel = (G.abs() + 8) * U
    H = a * V
    bH = 1.13 * eG * (V.abs() + eU) + (a.abs() + rel * a.abs()) * eU + (rel + e) * H.abs() + tiny
    dG, dU = dh * V * slope, dh * a
    # (act(G) is G times a share whose error is relative; its slope is a sum of terms of at most |G| + 2)
    bG = dh.abs() * (1.13 * eU + (V.abs() + eU) * (eG + rel * (G.abs() + 2) * slope.abs().clamp(max=1.13))) + e * dG.abs() + tiny
    bU = dh.abs() * (1.13 * eG + rel * a.abs()) + e * dU.abs() + tiny
    dx = dG @ Wg.t() + dU @ Wu.t()
    bx = bG @ Wg.abs().t() + bU @ Wu.abs().t() + (2 * F + 2) * U * (dG.abs() @ Wg.abs().t() + dU.abs() @ Wu.abs().t()) + e * dx.abs() + tiny
    g = {"H": (H, bH), "dx": (dx, bx)}
    for k, d, b in (("dWg", dG, bG), ("dWu", dU, bU)):
        w = x.t() @ d
        g[k] = (w, x.abs().t() @ b + (rows + 2) * U * x.abs().t() @ d.abs() + e * w.abs() + tiny)
    return g, (G, eG), (V, eU)


def near(got, want, what):
    ref, bound = want
    assert got.shape == ref.shape and bool(torch.isfinite(got).all()), what
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), f"{what}: worst {float((err / bound).max()):.3f} of the bound"


CASES = [(1, 64, 128), (1, 1, 1), (3, 8, 8), (5, 63, 127), (16, 200, 264), (40, 512, 1000), (64, 520, 129), (65, 65, 257), (129, 136, 384), (300, 264, 130),
         (257, 1030, 515), (4300, 72, 300), (700, 2048, 136)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_forward_and_gradients(case, dtype, act):
    P = _p()
    rows, I, F = case
    t = inputs(rows, I, F, dtype, seed=rows + F)
    want, G, V = definition(t, act)
    near(P.dense_gated(t["x"], t["Wg"], t["Wu"], act), want["H"], "forward")
    H, g, u = P.dense_gated_save(t["x"], t["Wg"], t["Wu"], act)
    near(H, want["H"], "forward that keeps G and U")
    near(g, G, "G")
    near(u, V, "U")
    leaves = [t[k].clone().requires_grad_() for k in ("x", "Wg", "Wu")]
    h = P.DenseGatedFunction.apply(*leaves, act)
    assert torch.equal(h.detach(), H)
    for k, d in zip(("dx", "dWg", "dWu"), torch.autograd.grad(h, leaves, t["dh"])):
        near(d, want[k], k)
    P.device_status()


def test_activations_far_out():
    """Gates of some hundreds: the exponential overflows on one side and vanishes on the other."""
    P = _p()
    for act in ACTS:
        t = inputs(50, 64, 128, BF16, std=100.0)
        want, _, _ = definition(t, act)
        leaves = [t[k].clone().requires_grad_() for k in ("x", "Wg", "Wu")]
        h = P.DenseGatedFunction.apply(*leaves, act)
        near(h.detach(), want["H"], act)
        for k, d in zip(("dx", "dWg", "dWu"), torch.autograd.grad(h, leaves, t["dh"])):
            near(d, want[k], k)


def test_gradients_against_differences():
    P = _p()
    t = inputs(60, 40, 48, F16, seed=9)
    leaves = [t[k].clone().requires_grad_() for k in ("x", "Wg", "Wu")]
    grads = torch.autograd.grad(P.DenseGatedFunction.apply(*leaves, "silu"), leaves, t["dh"])
    gen = torch.Generator(device="cuda").manual_seed(10)
    for k, g in zip(("x", "Wg", "Wu"), grads):
        d, h = torch.randn(t[k].shape, generator=gen, device="cuda").double(), 1e-5
        f = lambda s: ((lambda v: act64("silu", v["x"] @ v["Wg"]) * (v["x"] @ v["Wu"]))({n: t[n].double() + (s * h * d if n == k else 0) for n in t}) * t["dh"].double()).sum()  # noqa: E731,B023
        # gradients in float16: every entry within two roundings and its sums of the exact one, the difference within h**2
        assert abs(float((g.double() * d).sum() - (f(1) - f(-1)) / (2 * h))) <= 4e-3 * float((g.double() * d).abs().sum())


def test_some_gradients_only():
    P = _p()
    t = inputs(70, 72, 136, BF16)
    leaves = [t[k].clone().requires_grad_() for k in ("x", "Wg", "Wu")]
    full = torch.autograd.grad(P.DenseGatedFunction.apply(*leaves, "gelu"), leaves, t["dh"])
    for need in ((True, False, False), (False, True, True), (False, False, True)):
        some = [t[k].clone().requires_grad_(n) for k, n in zip(("x", "Wg", "Wu"), need)]
        got = torch.autograd.grad(P.DenseGatedFunction.apply(*some, "gelu"), [s for s in some if s.requires_grad], t["dh"])
        assert all(torch.equal(a, b) for a, b in zip(got, [f for f, n in zip(full, need) if n]))
    H, G, V = P.dense_gated_save(t["x"], t["Wg"], t["Wu"], "gelu")
    assert all(torch.equal(a, b) for a, b in zip(P.dense_gated_backward(t["dh"], t["x"], t["Wg"], t["Wu"], G, V, "gelu"), full))
    with torch.no_grad():
        assert not P.DenseGatedFunction.apply(*leaves, "gelu").requires_grad


def test_shapes_strides_and_alignment():
    P = _p()
    t = inputs(48, 72, 40, BF16)
    want = definition(t, "silu")[0]["H"]
    near(P.dense_gated(t["x"].view(4, 12, 72), t["Wg"], t["Wu"]).view(48, 40), want, "three dimensions")
    near(P.dense_gated(t["x"][0], t["Wg"], t["Wu"]).view(1, 40), tuple(a[:1] for a in want), "one dimension")
    off = torch.zeros(48 * 72 + 8, dtype=BF16, device="cuda")[3:3 + 48 * 72].view(48, 72)
    off.copy_(t["x"])
    near(P.dense_gated(off, t["Wg"].t().contiguous().t(), t["Wu"]), want, "off sixteen bytes, another order")
    assert P.dense_gated(t["x"][:0], t["Wg"], t["Wu"]).shape == (0, 40)
    leaves = [t["x"][:0].clone().requires_grad_(), t["Wg"].clone().requires_grad_(), t["Wu"].clone().requires_grad_()]
    d = torch.autograd.grad(P.DenseGatedFunction.apply(*leaves), leaves, torch.zeros(0, 40, dtype=BF16, device="cuda"))
    assert d[0].shape == (0, 72) and not bool(d[1].any()) and not bool(d[2].any())


@pytest.mark.parametrize("rows", [20, 200])
def test_what_is_not_finite_stays_with_its_row_and_column(rows):
    P = _p()
    t = inputs(rows, 200, 264, BF16)
    want = definition(t, "silu")[0]
    for v in (float("nan"), float("inf")):
        x, Wg = t["x"].clone(), t["Wg"].clone()
        x[7, 3], Wg[5, 9] = v, v
        h = P.dense_gated(x, Wg, t["Wu"])
        keep = torch.ones(rows, 264, dtype=torch.bool, device="cuda")
        keep[7], keep[:, 9] = False, False
        near(h[keep], tuple(a[keep] for a in want["H"]), "forward")
        assert not bool(torch.isfinite(h[7]).any())
    dh = t["dh"].clone()
    dh[4, 6] = float("inf")
    leaves = [t[k].clone().requires_grad_() for k in ("x", "Wg", "Wu")]
    d = torch.autograd.grad(P.DenseGatedFunction.apply(*leaves), leaves, dh)
    near(torch.cat((d[0][:4], d[0][5:])), tuple(torch.cat((a[:4], a[5:])) for a in want["dx"]), "dX")
    for k in (1, 2):
        cols = torch.arange(264, device="cuda") != 6
        near(d[k][:, cols], tuple(a[:, cols] for a in want[("dx", "dWg", "dWu")[k]]), "dW")


def test_same_bits_streams_and_graphs():
    P = _p()
    for rows in (24, 600):
        t, u = inputs(rows, 264, 520, BF16), inputs(rows, 264, 520, BF16, seed=3)
        first = P.dense_gated(t["x"], t["Wg"], t["Wu"])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = P.dense_gated(u["x"], u["Wg"], u["Wu"])
            again = P.dense_gated(t["x"], t["Wg"], t["Wu"])
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(first, again)
        held = {k: v.clone() for k, v in t.items()}
        leaves = [held[k].requires_grad_() for k in ("x", "Wg", "Wu")]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            h = P.DenseGatedFunction.apply(*leaves)
            d = torch.autograd.grad(h, leaves, held["dh"])
        for s in (t, u):
            with torch.no_grad():
                for k in held:
                    held[k].copy_(s[k])
            g.replay()
            want = definition(s, "silu")[0]
            near(h.detach(), want["H"], "replayed")
            for k, q in zip(("dx", "dWg", "dWu"), d):
                near(q, want[k], k)
        assert torch.equal(other, h.detach())
    P.device_status()


def test_offsets_past_32_bits():
    """More than 2**31 values of H."""
    P = _p()
    rows, I, F = 270000, 16, 8192
    t = inputs(64, I, F, BF16)
    x = t["x"].repeat(rows // 64 + 1, 1)[:rows].contiguous()
    h = P.dense_gated(x, t["Wg"], t["Wu"])
    want = definition(t, "silu")[0]["H"]
    for at in (0, 64 * 2000, (rows // 64 - 1) * 64):
        near(h[at:at + 64], want, "forward")
    # every repetition is the same rows
    assert torch.equal(h[:rows // 64 * 64].view(-1, 64, F)[::97], h[:64].expand(len(range(0, rows // 64, 97)), 64, F))
