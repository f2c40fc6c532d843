"""The AdamW step over many tensors against the formula in 64 bits.

Bounds.  fp32 arithmetic: a moment is two products and a sum (three roundings of 2**-24 relative to the larger term), the step a quotient, a square root and
three products more, so it is within 16 * 2**-24 of itself where its moments are exact, and the moments' own errors add as much again; a parameter is
rounded once (2**-24 of itself; a 16-bit one eps / 2).  A code is within half a step of q = 127 sqrt(|m| / s) or 254 (v / s)**(1/4) (and fp32's error of
them, below 1e-4 of a step's width).  What a code stands for: c / 127 has two roundings (the constant's and the product's), its square 2 * 2 + 1, times s
6 * 2**-24; of v, squared once more, 2 * 5 + 1 + 1 = 12 * 2**-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
B1, B2, EPS, WD, LR = 0.9, 0.99, 1e-8, 0.02, 3e-3


def _p():
    import paralleltnnlayers_b200 as P
    return P


def definition(w, g, m, v, t, lr=LR):
    w, g, m, v = (a.double() for a in (w, g, m, v))
    m, v = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    step = lr * (m / (1 - B1 ** t)) / ((v / (1 - B2 ** t)).sqrt() + EPS)
    return w - lr * WD * w - step, m, v, step.abs()


def values(n, gen, dtype=torch.float32):
    """Gradients over ten decades, some zero."""
    x = torch.randn(n, generator=gen, device="cuda") * 10 ** (torch.rand(n, generator=gen, device="cuda") * 10 - 8)
    return torch.where(torch.rand(n, generator=gen, device="cuda") < 0.05, 0.0, x).to(dtype)


def near(got, want, bound):
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound.clamp(min=1e-300)).max()):.3f} of the bound"


SIZES = [1, 3, 4, 255, 256, 257, 2047, 2048, 2049, 5000, 70001]


@pytest.mark.parametrize("grad", ["same", "float32"])
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, True), (torch.float16, True), (torch.bfloat16, False)])
def test_step_of_many_sizes(dtype, master, grad):
    P = _p()
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = [torch.randn(n, generator=gen, device="cuda") for n in SIZES]
    p = [a.to(dtype) for a in w] if dtype != torch.float32 else [a.clone() for a in w]
    start = [a.clone() if master else b.float() for a, b in zip(w, p)]
    g = [values(n, gen, dtype if grad == "same" else torch.float32) for n in SIZES]
    m, v = [values(n, gen) for n in SIZES], [values(n, gen).square() for n in SIZES]
    want = [definition(*a, 7) for a in zip(start, g, m, v)]
    P.adamw_step(p, g, m, v, 7, LR, betas=(B1, B2), eps=EPS, weight_decay=WD, master=w if master else None)
    u = 2.0 ** -24
    for k in range(len(SIZES)):
        x, em, ev, step = want[k]
        near(m[k], em, 4 * u * (em.abs() + (1 - B1) * g[k].double().abs()) + 1e-44)
        near(v[k], ev, 4 * u * ev + 1e-44)
        # the step's error: its own 16 roundings, and that of m where its two terms cancel
        slack = LR * 4 * u * (1 - B1) * g[k].double().abs() / (1 - B1 ** 7) / ((ev / (1 - B2 ** 7)).sqrt() + EPS)
        near(w[k] if master else p[k], x, 2 * u * x.abs() + 3 * u * start[k].double().abs() + 24 * u * step + slack
             + (torch.finfo(dtype).eps / 2 * x.abs() + 2.0 ** -25 if dtype != torch.float32 and not master else 0))
        if master:
            assert torch.equal(p[k], w[k].to(dtype))


def _codes(x, signed):
    b = torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)
    s = b.abs().amax(1, keepdim=True)
    q = (b.abs() / torch.where(s > 0, s, 1)) ** (0.5 if signed else 0.25) * (127 if signed else 254)
    return (q * b.sign()).view(-1)[:x.numel()], s.view(-1)


def test_eight_bit_moments():
    P = _p()
    gen = torch.Generator(device="cuda").manual_seed(2)
    p = [torch.randn(n, generator=gen, device="cuda") for n in SIZES]
    blocks = [(n + 255) // 256 for n in SIZES]
    z = lambda ns, t: [torch.zeros(n, dtype=t, device="cuda") for n in ns]  # noqa: E731
    m, v, ms, vs = z(SIZES, torch.int8), z(SIZES, torch.uint8), z(blocks, torch.float32), z(blocks, torch.float32)
    u = 2.0 ** -24
    for t in (1, 2, 3):
        g = [values(n, gen) for n in SIZES]
        held = [P.adamw_moments(a, b, (c, d), torch.float32) for a, b, c, d in zip(m, v, ms, vs)]
        want = [definition(a, b, *c, t) for a, b, c in zip(p, g, held)]
        start = [a.clone() for a in p]
        P.adamw_step(p, g, m, v, t, LR, betas=(B1, B2), eps=EPS, weight_decay=WD, scales=(ms, vs))
        for k in range(len(SIZES)):
            x, em, ev, step = want[k]
            slack = LR * 4 * u * (1 - B1) * g[k].double().abs() / (1 - B1 ** t) / ((ev / (1 - B2 ** t)).sqrt() + EPS)
            near(p[k], x, 2 * u * x.abs() + 3 * u * start[k].double().abs() + 24 * u * step + slack)
            qm, sm = _codes(em, True)
            qv, sv = _codes(ev, False)
            near(ms[k], sm, 8 * u * sm)
            near(vs[k], sv, 8 * u * sv)
            near(m[k].double(), qm, torch.full_like(qm, 0.5 + 1e-3))
            # (at least one where it is above zero)
            near(v[k].double(), torch.where(ev > 0, qv.clamp(min=1), 0.0), torch.full_like(qv, 0.5 + 1e-3))
            a, b = P.adamw_moments(m[k], v[k], (ms[k], vs[k]), torch.float32)
            near(a, (m[k].double() / 127).square() * m[k].double().sign() * ms[k].double().repeat_interleave(256)[:SIZES[k]],
                 4 * u * a.double().abs() + 1e-44)
            near(b, (v[k].double() / 254) ** 4 * vs[k].double().repeat_interleave(256)[:SIZES[k]], 12 * u * b.double().abs() + 1e-44)


def test_what_is_not_finite_stays_with_its_value():
    P = _p()
    g = torch.ones(600, device="cuda")
    g[5], g[300], g[599] = float("nan"), float("inf"), -float("inf")
    bad = ~torch.isfinite(g)
    for small in (False, True):
        p = torch.ones(600, device="cuda")
        m = torch.zeros(600, dtype=torch.int8 if small else torch.float32, device="cuda")
        v = torch.zeros(600, dtype=torch.uint8 if small else torch.float32, device="cuda")
        s = (torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda"))
        for t in (1, 2):
            P.adamw_step([p], [g], [m], [v], t, LR, scales=([s[0]], [s[1]]) if small else None)
        a, b = P.adamw_moments(m, v, s, torch.float32) if small else (m, v)
        assert bool(torch.isnan(p[bad]).all()) and bool(torch.isfinite(p[~bad]).all())
        assert not bool(torch.isfinite(a[bad]).any()) and not bool(torch.isfinite(b[bad]).any())
        assert bool(torch.isfinite(a[~bad]).all()) and bool((b[~bad] > 0).all())
        assert torch.equal(p[~bad], p[~bad][:1].expand_as(p[~bad]))


def test_tiny_and_huge_gradients_keep_their_neighbours():
    """Blocks whose largest value is subnormal, or near the largest float."""
    P = _p()
    for size in (1e-44, 1e-40, 1e-20, 1e18):
        g = torch.full((256,), size, device="cuda")
        p, m, v = torch.ones(256, device="cuda"), torch.zeros(256, dtype=torch.int8, device="cuda"), torch.zeros(256, dtype=torch.uint8, device="cuda")
        s = (torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda"))
        P.adamw_step([p], [g], [m], [v], 1, LR, scales=([s[0]], [s[1]]))
        assert bool(torch.isfinite(p).all()) and bool((p <= 1).all()) and bool((p > 0.9).all())
        assert bool(torch.isfinite(torch.stack(P.adamw_moments(m, v, s, torch.float32))).all())


def test_views_off_sixteen_bytes_and_what_lies_beside_them():
    P = _p()
    gen = torch.Generator(device="cuda").manual_seed(3)
    for off in (1, 2, 3):
        buf = torch.randn(4, 1100, generator=gen, device="cuda")
        before = buf.clone()
        p, g, m, v = (b[off:off + 1001] for b in buf)
        v.abs_()
        want = definition(p, g, m, v, 2)
        P.adamw_step([p], [g], [m], [v], 2, LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
        for a, b in zip((p, m, v), want):
            near(a, b, 1e-6 * b.abs() + 1e-6)
        assert torch.equal(buf[:, :off], before[:, :off]) and torch.equal(buf[:, off + 1001:], before[:, off + 1001:])


def test_more_tensors_than_a_table_holds():
    P = _p()
    n = 1000
    gen = torch.Generator(device="cuda").manual_seed(4)
    sizes = [(k * 37) % 300 for k in range(n)]   # some of no values
    p = [torch.randn(k, generator=gen, device="cuda") for k in sizes]
    g, m, v = ([torch.randn(k, generator=gen, device="cuda") for k in sizes] for _ in range(3))
    v = [a.abs() for a in v]
    want = [definition(*a, 3)[0] for a in zip(p, g, m, v)]
    k0 = P.launch_count()
    P.adamw_step(p, g, m, v, 3, LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    assert P.launch_count() - k0 == 3
    near(torch.cat(p), torch.cat(want), 1e-6 * torch.cat(want).abs() + 1e-7)


def test_captured_step_counts_its_replays_and_reads_the_rate():
    P = _p()
    from paralleltnnlayers_b200.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(5)
    w = [torch.randn(s, generator=gen, device="cuda") for s in (33, (16, 40), 1000)]
    grads = [[torch.randn(a.shape, generator=gen, device="cuda") for a in w] for _ in range(4)]
    rates = [1e-2, 5e-3, 2e-3, 1e-3]
    for bits in (32, 8):
        eager = [torch.nn.Parameter(a.clone()) for a in w]
        opt = AdamW(eager, weight_decay=WD, bits=bits)
        graphed = [torch.nn.Parameter(a.clone()) for a in w]
        lr = torch.tensor(rates[0], device="cuda")
        cap = AdamW(graphed, lr=lr, weight_decay=WD, bits=bits, capturable=True)
        for p in graphed:
            p.grad = torch.zeros_like(p)
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        for k in range(4):
            for group in opt.param_groups:
                group["lr"] = rates[k]
            for p, q, d in zip(eager, graphed, grads[k]):
                p.grad = d
                q.grad.copy_(d)
            lr.fill_(rates[k])
            opt.step()
            if k == 0:
                cap.step()
                torch.cuda.synchronize()
                with torch.cuda.graph(graph, stream=stream):
                    cap.step()
            else:
                graph.replay()
        for p, q in zip(eager, graphed):
            near(q.detach(), p.detach().double(), 1e-6 * p.detach().double().abs() + 2e-7 + (1e-3 if bits == 8 else 0))
        assert int(cap.state[graphed[0]]["step"]) == 4


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimiser_and_its_saved_state(bits, dtype):
    from paralleltnnlayers_b200.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(6)
    make = lambda: [torch.nn.Parameter(torch.full(s, 0.5, device="cuda", dtype=dtype)) for s in ((7, 9), (300,))]  # noqa: E731
    a, b = make(), make()
    one, two = AdamW(a, lr=LR, bits=bits), AdamW(b, lr=LR, bits=bits)
    for k in range(4):
        grads = [torch.randn(p.shape, generator=gen, device="cuda").to(dtype) for p in a]
        if k == 2:   # the second goes on from the first's state
            two = AdamW(b, lr=LR, bits=bits)
            two.load_state_dict(one.state_dict())
            for p, q in zip(a, b):
                assert all(torch.equal(x, two.state[q][n]) and x.dtype == two.state[q][n].dtype for n, x in one.state[p].items() if torch.is_tensor(x))
        for ps, opt in ((a, one), (b, two)):
            for p, g in zip(ps, grads):
                p.grad = g.clone()
            opt.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    a[0].grad = None   # a parameter without a gradient stays
    before = a[0].detach().clone()
    a[1].grad = torch.ones_like(a[1])
    one.step()
    assert torch.equal(a[0].detach(), before) and one.state[a[0]]["step"] == 4 and one.state[a[1]]["step"] == 5


def test_offsets_past_32_bits():
    P = _p()
    n = 2 ** 31 + 300
    p, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    m, v = torch.zeros(n, dtype=torch.int8, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda")
    s = [torch.zeros((n + 255) // 256, device="cuda") for _ in range(2)]
    at = torch.tensor([0, 2 ** 31 - 1, 2 ** 31, n - 300, n - 1], device="cuda")
    g[at] = torch.tensor([1.0, -2.0, 3.0, -4.0, 5.0], dtype=torch.bfloat16, device="cuda")
    P.adamw_step([p], [g], [m], [v], 1, 0.5, weight_decay=0.0, scales=([s[0]], [s[1]]))
    assert torch.equal(p[at], -0.5 * g[at].sign())   # a first step is lr times the gradient's sign
    assert int(torch.count_nonzero(p)) == 4 + (1 if n - 300 != 2 ** 31 else 0) and int(torch.count_nonzero(m)) == len(set(at.tolist()))


def test_a_tensor_twice_is_refused():
    P = _p()
    c = lambda: torch.ones(8, device="cuda")  # noqa: E731
    p, m = c(), c()
    for ps, ms in (([p, p], [c(), c()]), ([c(), c()], [m, m])):
        with pytest.raises(ValueError, match="occurs twice"):
            P.adamw_step(ps, [c(), c()], ms, [c(), c()], 1, LR)


@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-30])
def test_an_eps_of_next_to_nothing(eps):
    """Gradients whose squares are subnormal: the steps are still lr times their signs (v is within 2**-149 of its value: of 1e-40, 1e-5)."""
    P = _p()
    g = torch.tensor([1e-19, -1e-20, 1.0, -3e-3] * 64, device="cuda")
    p, m, v = torch.zeros(256, device="cuda"), torch.zeros(256, device="cuda"), torch.zeros(256, device="cuda")
    P.adamw_step([p], [g], [m], [v], 1, LR, betas=(B1, B2), eps=eps, weight_decay=0.0)
    want = -LR * (g.double() / (g.double().abs() + (eps if eps > 1e-45 else 0)))
    near(p, want, 0.05 * LR * torch.ones_like(want) * (g.double().abs() < 1e-18) + 1e-5 * LR)


def test_a_copied_optimiser_counts_on():
    import copy
    import pickle

    from paralleltnnlayers_b200.optim import AdamW
    p = [torch.nn.Parameter(torch.ones(5, device="cuda")), torch.nn.Parameter(torch.ones(7, device="cuda"))]
    opt = AdamW(p, capturable=True)
    for q in p:
        q.grad = torch.ones_like(q)
    opt.step()
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        ps = other.param_groups[0]["params"]
        for q in ps:
            q.grad = torch.ones_like(q)
        other.step()
        assert [int(other.state[q]["step"]) for q in ps] == [2, 2] and int(opt.state[p[0]]["step"]) == 1


def test_autograd_sees_the_update():
    P = _p()
    p = torch.ones(4, device="cuda", requires_grad=True)
    y = (p * p).sum()
    P.adamw_step([p.detach()], [torch.ones(4, device="cuda")], [torch.zeros(4, device="cuda")], [torch.zeros(4, device="cuda")], 1, LR)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
