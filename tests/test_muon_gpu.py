"""The Muon step and the orthogonalisation against their definition in 64 bits.

Bound, in the Frobenius norm.  A step's products carry operands of 22 bits or more and sums of fp32: what step k adds is at most 2**-21 of |X_k|.  A later step
raises it by the slope of a s + b s^3 + c s^5, at most 4 where singular values are up to 1.21.  So X is off by at most 2**-21 sum_k 4**(steps - k) |X_k|, and by
the half step of its type.  The update is one product and one sum in fp32 more (2**-23 of their sizes).

Where the result has 16 bits (bfloat16 X, 16-bit parameters without a copy), the products of matrices with sides above 64 take operands of 11 bits.  Their
roundings stay in the row or column space of what is multiplied, where later steps do not raise them; they are independent, 2**-12 / 3**0.5 of an operand in
the norm, five operands a step whose products are at most 2.8 times X: 2.8 (5 / 3)**0.5 2**-12 a step, and 8 * 2**-12 of |X| after five."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ABC = (3.4445, -4.7750, 2.0315)


def half(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    return torch.finfo(dtype).tiny * half(dtype)


def matrices(*shape, seed=0, spike=4.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    return n(*shape) + spike * n(*shape[:-1], 1) * n(*shape[:-2], 1, shape[-1])


def defined(X, coefficients=ABC, eps=1e-7, steps=5):
    """X after the steps in 64 bits, and how far off a result may be per matrix, without the rounding to its type."""
    X = X.double()
    X = X / X.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=eps)
    norm = lambda X: X.square().sum((-2, -1)).sqrt()  # noqa: E731
    bound = 4.0 ** steps * norm(X)
    for k in range(steps):
        a, b, c = coefficients[k] if isinstance(coefficients[0], tuple) else coefficients
        A = X @ X.mT if X.shape[-2] <= X.shape[-1] else X.mT @ X
        B = b * A + c * A @ A
        X = a * X + (B @ X if X.shape[-2] <= X.shape[-1] else X @ B)
        bound = bound + 4.0 ** (steps - k - 1) * norm(X)
    return X, bound * 2.0 ** -21


def check(got, want, bound, coarse=False):
    t = half(got.dtype)
    if coarse:
        bound = bound + 2.0 ** -9 * want.square().sum((-2, -1)).sqrt()
    off = (got.double() - want).square().sum((-2, -1)).sqrt()
    bound = bound + t * (want.square().sum((-2, -1)).sqrt() + bound) + least(got.dtype) * math.sqrt(want.shape[-1] * want.shape[-2])
    assert got.shape == want.shape and bool((off <= bound).all()), f"{float((off / bound).max()):.2f} of the bound"


SHAPES = [(1, 1), (1, 7), (9, 1), (5, 3), (16, 16), (16, 17), (17, 130), (33, 20), (64, 64), (64, 1000), (1300, 64), (40, 3, 50), (7, 60, 31), (2, 3, 300, 16), (65, 65), (65, 300),
          (300, 66), (256, 256), (257, 513), (640, 129), (700, 1000), (1001, 701), (3, 70, 90), (4, 200, 72)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalise(shape, dtype):
    import paralleltnnlayers_b200 as P
    X = matrices(*shape, seed=sum(shape)).to(dtype)
    kept = X.clone()
    out = P.orthogonalise(X)
    check(out, *defined(X), coarse=dtype == torch.bfloat16 and min(shape[-2:]) > 64)
    assert torch.equal(X, kept) and torch.equal(out, P.orthogonalise(X))
    P.device_status()


@pytest.mark.parametrize("shape", [(40, 100), (200, 300), (300, 200), (600, 70)], ids=str)
@pytest.mark.parametrize("steps,coefficients", [(0, ABC), (1, ABC), (2, (2.0, -1.5, 0.5)), (8, (1.875, -1.25, 0.375)), (3, ((3.0, -3.2, 1.2), (2.0, -1.5, 0.5), (1.5, -0.5, 0.0)))])
def test_steps_and_coefficients(shape, steps, coefficients):
    import paralleltnnlayers_b200 as P
    X = matrices(*shape, seed=3)
    check(P.orthogonalise(X, coefficients, steps=steps), *defined(X, coefficients, steps=steps))


@pytest.mark.parametrize("shape", [(48, 90), (150, 260), (260, 150), (400, 400), (130, 900)], ids=str)
@pytest.mark.parametrize("rank", [1, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_few_directions(shape, rank, dtype):
    """What rounding adds in the directions that a matrix has not is raised by every step, and has to stay small beside those that it has."""
    import paralleltnnlayers_b200 as P
    gen = torch.Generator(device="cuda").manual_seed(rank)
    U, V = (torch.linalg.qr(torch.randn(n, rank, generator=gen, device="cuda", dtype=torch.float64))[0] for n in shape)
    X = ((U * torch.tensor([1.0, 0.5, 0.25], device="cuda")[:rank]) @ V.mT).to(dtype)
    out = P.orthogonalise(X)
    check(out, *defined(X), coarse=dtype == torch.bfloat16 and min(shape) > 64)
    s = torch.linalg.svdvals(out.double())
    assert 0.6 < float(s[rank - 1]) and float(s[0]) < 1.3


@pytest.mark.parametrize("shape", [(30, 40), (120, 200), (200, 120)], ids=str)
def test_sizes_of_values(shape):
    import paralleltnnlayers_b200 as P
    X = matrices(*shape, seed=1)
    want, bound = defined(X)
    for scale in (1e-30, 1e-12, 1e6, 1e30):
        check(P.orthogonalise(X * scale, eps=1e-37), want, bound + 2.0 ** -22 * want.norm())
    assert not P.orthogonalise(torch.zeros_like(X)).any()
    small = X * 1e-10
    check(P.orthogonalise(small), *defined(small))   # (below eps: divided by that)
    for bad in (float("nan"), float("inf")):
        both = torch.stack([X, X])
        both[0, 3, 4] = bad
        out = P.orthogonalise(both)
        assert out[0].isnan().all()
        check(out[1], want, bound)


def expected(p, g, m, lr, momentum, nesterov, wd, adjust, coefficients=ABC, eps=1e-7, steps=5):
    p, g, m = p.double(), g.double(), m.double()
    m = m + (1 - momentum) * (g - m)
    u = g + momentum * (m - g) if nesterov else m
    X, bound = defined(u, coefficients, eps, steps)
    r, c = p.shape[-2:]
    factor = {"original": max(1.0, r / c) ** 0.5, "match_rms_adamw": 0.2 * max(r, c) ** 0.5, None: 1.0}[adjust]
    # (u itself is rounded to fp32: 2**-22 of |m| and |g|, which the first bound covers as part of |X_0|, twice)
    norm = lambda t: t.square().sum((-2, -1)).sqrt()  # noqa: E731
    big = (norm(g) + norm(m)) / norm(u).clamp(min=eps)
    bound = bound + 4.0 ** steps * 2.0 ** -22 * big
    want = p * (1 - lr * wd) - lr * factor * X
    return want, m, lr * factor * (bound + 2.0 ** -22 * norm(X)) + 2.0 ** -22 * norm(p)


LISTS = [[(3, 16), (64, 16), (64, 16), (40, 200), (8, 8, 32)], [(100, 300), (70, 70), (100, 300), (300, 100)], [(16, 33), (130, 90), (2, 80, 96), (5, 1), (1, 5), (257, 65)]]


@pytest.mark.parametrize("dtype,gtype,copies", [(torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, True), (torch.bfloat16, torch.float32, False),
                                                (torch.float16, torch.float16, False), (torch.float16, torch.float32, True)])
@pytest.mark.parametrize("shapes", LISTS, ids=("small", "large", "both"))
@pytest.mark.parametrize("nesterov,adjust", [(True, "original"), (False, "match_rms_adamw"), (True, None)])
def test_step(shapes, dtype, gtype, copies, nesterov, adjust):
    import paralleltnnlayers_b200 as P
    w = [0.1 * matrices(*s, seed=k, spike=0) for k, s in enumerate(shapes)]
    p = [t.to(dtype) if dtype != torch.float32 else t.clone() for t in w]
    m = [torch.zeros_like(t) for t in w]
    for step in range(2):
        g = [(0.01 * matrices(*s, seed=10 * step + k)).to(gtype) for k, s in enumerate(shapes)]
        want = [expected(a, b, c, 0.02, 0.9, nesterov, 0.1, adjust) for a, b, c in zip(w if copies else p, g, m)]
        before = [t.clone() for t in p]
        P.muon_step(p, g, m, 0.02, 0.9, nesterov, 0.1, adjust=adjust, master=w if copies else None)
        for k, (v, mom, bound) in enumerate(want):
            assert bool(((m[k].double() - mom).abs() <= 2.0 ** -22 * (mom.abs() + g[k].double().abs())).all())
            coarse = 2.0 ** -9 * (v - 0.998 * before[k].double()).square().sum((-2, -1)).sqrt()   # of the update
            check(w[k] if copies else p[k], v, bound + (coarse if dtype != torch.float32 and not copies and min(v.shape[-2:]) > 64 else 0))
            if copies:
                assert torch.equal(p[k], w[k].to(dtype))
    P.device_status()


def test_views_lists_and_rates_on_the_device():
    import paralleltnnlayers_b200 as P
    shapes = [(70, 90), (12, 33), (70, 90)]
    g = [matrices(*s, seed=k) for k, s in enumerate(shapes)]
    def fresh():
        return [0.1 * matrices(*s, seed=7, spike=0) for s in shapes], [torch.zeros(*s, device="cuda") for s in shapes]
    p, m = fresh()
    P.muon_step(p, g, m, 0.02)
    q, n = fresh()
    P.muon_step(q, [t.t().contiguous().t() for t in g], n, torch.tensor(0.02, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(p + m, q + n))
    # off their boundaries, in one buffer
    flat = [torch.zeros(sum(70 * 90 + 1 for _ in shapes), device="cuda") for _ in range(3)]
    views = [[], [], []]
    for lists, buffer in zip(views, flat):
        at = 1
        for s in shapes:
            lists.append(buffer[at: at + s[0] * s[1]].view(s))
            at += s[0] * s[1]
    q, n = fresh()
    for k in range(3):
        for lists, value in zip(views, (q[k], g[k], n[k])):
            lists[k].copy_(value)
    P.muon_step(*views, 0.02)
    assert all(torch.equal(a, b) for a, b in zip(p + m, views[0] + views[2]))
    assert all(float(b[0]) == 0 for b in flat)
    P.muon_step([], [], [], 0.02)
    P.muon_step([torch.zeros(0, 5, device="cuda"), p[1]], [torch.zeros(0, 5, device="cuda"), g[1]], [torch.zeros(0, 5, device="cuda"), m[1]], 0.02)
    assert P.orthogonalise(torch.zeros(3, 0, 4, device="cuda")).shape == (3, 0, 4)


def test_types_and_sizes_in_turn():
    """What a kernel is allowed for the largest matrix stays allowed when other types come with smaller ones."""
    import paralleltnnlayers_b200 as P
    for side in (60, 10, 60, 30, 60):
        for dtype, gtype in ((torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.bfloat16, torch.float32)):
            for n in (side, 7):
                g = matrices(n, 80, seed=n).to(gtype)
                p, m = torch.zeros(n, 80, device="cuda", dtype=dtype), torch.zeros(n, 80, device="cuda")
                P.muon_step([p], [g], [m], 1.0, momentum=0.0, weight_decay=0.0, adjust=None)
                check(-p, *defined(g))


def test_many_matrices():
    """More tensors than a launch's table has, and more matrices of a shape than share launches."""
    import paralleltnnlayers_b200 as P
    X = matrices(300, 9, 14, seed=2)
    p, m = [torch.zeros(9, 14, device="cuda") for _ in range(300)], [torch.zeros(9, 14, device="cuda") for _ in range(300)]
    P.muon_step(p, list(X), m, 1.0, momentum=0.0, weight_decay=0.0, adjust=None)
    check(-torch.stack(p), *defined(X))
    Y = matrices(110, 66, 70, seed=4)
    check(P.orthogonalise(Y), *defined(Y))


def test_many_shapes():
    """More shapes than a launch's table has, and more large matrices than go together."""
    import paralleltnnlayers_b200 as P
    shapes = [(65 + k, 70 + 3 * (k % 7)) if k % 2 else (90, 65 + k) for k in range(60)]
    p, g = [torch.zeros(*s, device="cuda") for s in shapes], [matrices(*s, seed=k) for k, s in enumerate(shapes)]
    P.muon_step(p, g, [torch.zeros_like(t) for t in p], 1.0, momentum=0.0, weight_decay=0.0, adjust=None)
    for a, b in zip(p, g):
        check(-a, *defined(b))
    X = matrices(300, 66, 68, seed=9)
    check(P.orthogonalise(X), *defined(X))
    P.device_status()


def test_long_stacks():
    """Stacks that are taken in several parts, small and large matrices of one call, and one matrix of a long side."""
    import paralleltnnlayers_b200 as P
    X = matrices(9001, 3, 5, seed=5)
    check(P.orthogonalise(X), *defined(X))
    p = [torch.zeros(4100, 2, 2, device="cuda"), torch.zeros(66, 200, device="cuda"), torch.zeros(17, 70001, device="cuda"), torch.zeros(50003, 40, device="cuda")]
    g = [matrices(*t.shape, seed=k) for k, t in enumerate(p)]
    P.muon_step(p, g, [torch.zeros_like(t) for t in p], 1.0, momentum=0.0, weight_decay=0.0, adjust=None)
    for a, b in zip(p, g):
        check(-a, *defined(b))


def test_nothing_to_orthogonalise():
    """A gradient of zeros moves nothing, however small eps is; the weight decays all the same."""
    import paralleltnnlayers_b200 as P
    for shape in ((5, 9), (40, 60), (100, 80)):
        for eps in (1e-7, 1e-30, 1e-200):
            p, z = torch.randn(*shape, device="cuda"), torch.zeros(*shape, device="cuda")
            kept, m = p.clone(), z.clone()
            P.muon_step([p], [z], [m], 0.5, weight_decay=0.5, eps=eps)
            assert torch.equal(p, kept * 0.75) and not m.any()


def test_streams_and_graphs():
    import paralleltnnlayers_b200 as P
    for shapes in ([(16, 40), (100, 120)], [(130, 66), (5, 9)]):
        X = [matrices(*s, seed=1) for s in shapes]
        want = [P.orthogonalise(x) for x in X]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [P.orthogonalise(x) for x in X]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graphs = []
        for x in X:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
                out = P.orthogonalise(x)
            graphs.append((g, out))
        for k in (0, 1, 0):
            graphs[k][0].replay()
            assert torch.equal(graphs[k][1], want[k])


@pytest.mark.parametrize("wide,others", [(1, 0), (1, 1), (3, 7), (8, 66), (37, 0), (37, 1), (38, 3), (150, 20)])
def test_small_sides_together(wide, others):
    """Sides above and below 32 in turn, up to and beyond four CTAs an SM's worth for each of the wide ones; one of them zero, one not a number."""
    import paralleltnnlayers_b200 as P
    shapes = [None] * (wide + others)
    for k in range(wide + others):
        turn = k * wide // (wide + others) != (k + 1) * wide // (wide + others)
        shapes[k] = (33 + k % 32, 64 + 5 * (k % 9)) if turn else (1 + k % 32, 40 - k % 11)
    assert sum(min(s) > 32 for s in shapes) == wide
    for bad in (False, True):
        p, g = [torch.zeros(*s, device="cuda") for s in shapes], [matrices(*s, seed=k) for k, s in enumerate(shapes)]
        if bad:
            g[0].zero_()
            g[-1][0, 0] = float("nan")
        P.muon_step(p, g, [torch.zeros_like(t) for t in p], 1.0, momentum=0.0, weight_decay=0.0, adjust=None)
        for k, (a, b) in enumerate(zip(p, g)):
            if bad and k == len(p) - 1:
                assert bool(a.isnan().all())
            else:
                check(-a, *defined(b))
    P.device_status()
