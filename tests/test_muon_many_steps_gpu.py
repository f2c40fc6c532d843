"""Many Newton-Schulz steps on small matrices: nothing grows without end, whatever directions a matrix lacks.

a s + b s^3 + c s^5 with the usual coefficients takes singular values of up to 1.21 to at most 1.21; with 2 % for what is rounded, X stays below 1.25.
With (1.875, -1.25, 0.375) they go to one.  A rounding (2**-24 of X, of X between two runs of steps and of the product that forms it, and as much of its fp32 sum of up
to 64 terms of one size: 2**-21 in all) is raised by at most one over the smallest singular value until it stays, and that is at least 2**-5 here."""
import pytest
import torch

pytestmark = pytest.mark.gpu
CONVERGENT = (1.875, -1.25, 0.375)


def bounded(X):
    assert bool(X.isfinite().all()) and float(torch.linalg.svdvals(X.double()).max()) < 1.25


@pytest.mark.parametrize("steps", [6, 10, 20, 100])
@pytest.mark.parametrize("side", [8, 16, 33, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_matrices_that_lack_directions(side, steps, dtype):
    import paralleltnnlayers_b200 as P
    gen = torch.Generator(device="cuda").manual_seed(side)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    for rows, cols in ((side, side), (side, 5 * side), (3 * side + 1, side)):
        X = torch.stack([n(rows, 1) @ n(1, cols), n(rows, 3) @ n(3, cols), n(rows, cols), torch.zeros(rows, cols, device="cuda")])
        X[2, 1:3] = 0
        X[2, :, 4] = 0
        X = X.to(dtype)
        out = P.orthogonalise(X, steps=steps)
        bounded(out)
        assert not out[3].any() and not out[2, 1:3].any() and not out[2, :, 4].any()
        assert torch.equal(out, P.orthogonalise(X, steps=steps))
        p, m = torch.zeros_like(X), torch.zeros(X.shape, device="cuda")
        P.muon_step([p], [X], [m], 1.0, momentum=0.0, weight_decay=0.0, adjust=None, steps=steps)
        assert bool((m == X).all())
        bounded(p)


@pytest.mark.parametrize("shape", [(1, 1), (5, 3), (2, 16, 300), (70, 33), (64, 64), (3, 64, 200)], ids=str)
@pytest.mark.parametrize("steps", [12, 30, 100])
def test_steps_that_converge(shape, steps):
    """The polar factor, from runs of eleven steps."""
    import paralleltnnlayers_b200 as P
    gen = torch.Generator(device="cuda").manual_seed(steps)
    rows, cols = shape[-2:]
    n = min(rows, cols)
    U, V = (torch.linalg.qr(torch.randn(*shape[:-2], k, n, generator=gen, device="cuda", dtype=torch.float64))[0] for k in (rows, cols))
    s = 0.5 + 0.5 * torch.rand(*shape[:-2], n, generator=gen, device="cuda", dtype=torch.float64)   # (at least 1 / 16 of the norm)
    X = (U * s.unsqueeze(-2) @ V.mT).float()
    want = X.double()
    want = want / want.square().sum((-2, -1), keepdim=True).sqrt()
    for _ in range(steps):
        A = want @ want.mT
        want = CONVERGENT[0] * want + (CONVERGENT[1] * A + CONVERGENT[2] * A @ A) @ want
    out = P.orthogonalise(X, CONVERGENT, steps=steps)
    off = (out.double() - want).square().sum((-2, -1)).sqrt()
    assert bool((off <= 2.0 ** -21 * 32 * n ** 0.5).all()), float(off.max())


@pytest.mark.parametrize("master", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_step_of_several_runs(dtype, master):
    """The update, with each step's own coefficients, copies and every type: that of the same X."""
    import paralleltnnlayers_b200 as P
    if master and dtype == torch.float32:
        pytest.skip("a float32 parameter has no copy")
    triples = ((3.4445, -4.7750, 2.0315),) * 11 + ((2.0, -1.5, 0.5),) * 2   # runs of five, five and three steps
    gen = torch.Generator(device="cuda").manual_seed(1)
    shapes = [(16, 40), (2, 33, 64), (70, 20), (9, 5), (100, 80)]
    w = [torch.randn(*s, generator=gen, device="cuda") for s in shapes]
    g = [torch.randn(*s, generator=gen, device="cuda").to(dtype) for s in shapes]
    p, m = [t.to(dtype, copy=True) for t in w], [torch.zeros_like(t) for t in w]
    before = [t.clone() for t in (w if master else p)]
    P.muon_step(p, g, m, 0.5, momentum=0.0, weight_decay=0.1, coefficients=triples, steps=13, adjust=None, master=w if master else None)
    for a, b, v, c, copy in zip(p, before, g, m, w):
        assert torch.equal(c, v.float())
        X = P.orthogonalise(v.float(), triples, steps=13)
        want = b.double() * 0.95 - 0.5 * X.double()
        got = copy if master else a
        # (one product and one sum in fp32, 1 - lr wd and lr in fp32 too: four halves of a step; then the type's)
        e = 2.0 ** -22 * (b.double().abs() + X.double().abs())
        assert bool(((got.double() - want).abs() <= e + torch.finfo(got.dtype).eps / 2 * (want.abs() + e) + 2.0 ** -25).all())
        if master:
            assert torch.equal(a, copy.to(dtype))


def test_workspaces():
    """The size for any step is enough for every one; that of a step is what it needs, and X between two runs of steps is in it only where there are two."""
    import ctypes as C

    import paralleltnnlayers_b200 as P

    from paralleltnnlayers_b200 import _lib
    from test_training_operators_refusals import Hyper, Matrix
    lib = _lib.lib
    gen = torch.Generator(device="cuda").manual_seed(2)
    shapes = [(40, 16, 300), (1, 64, 2000), (1, 700, 9)]
    g = [torch.randn(*s, generator=gen, device="cuda") for s in shapes]
    abc = (C.c_double * 3)(3.4445, -4.7750, 2.0315)
    values = sum(t.numel() for t in g)
    for steps in (5, 6, 20):
        h = Hyper(lr=1.0, momentum=0.0, wd=0.0, eps=1e-7, nesterov=0, steps=steps, adjust=0, count=1, coefficients=abc)
        p, m = [torch.zeros_like(t) for t in g], [torch.zeros_like(t) for t in g]
        ms = (Matrix * 3)(*[Matrix(a.data_ptr(), b.data_ptr(), c.data_ptr(), None, *s) for a, b, c, s in zip(p, g, m, shapes)])
        any_step, this = lib.b200cp_muon_step_workspace_bytes(ms, 3, 0, 0), lib.b200cp_muon_workspace_bytes(ms, 3, 0, 0, C.byref(h))
        assert any_step >= this and (any_step - this >= 4 * values) == (steps == 5)
        ws = torch.empty(this + 256, dtype=torch.uint8, device="cuda")
        at = (ws.data_ptr() + 255) // 256 * 256
        stream = torch.cuda.current_stream().cuda_stream
        assert lib.b200cp_muon_step(ms, 3, 0, 0, C.byref(h), at, this - 1, stream) != 0 and not any(t.any() for t in m)
        assert lib.b200cp_muon_step(ms, 3, 0, 0, C.byref(h), at, this, stream) == 0
        for a, b in zip(p, g):
            assert torch.equal(-a, P.orthogonalise(b, steps=steps))
    assert lib.b200cp_muon_workspace_bytes(ms, 3, 0, 0, None) == 0
