"""Derivatives that the operators do not have are refused, not left out."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def operators():
    import paralleltnnlayers_b200 as P
    n = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    h = lambda *s: n(*s).bfloat16()  # noqa: E731
    tokens, which = torch.randint(9, (5,), device="cuda"), torch.randint(2, (5,), device="cuda", dtype=torch.int32)
    return {"embedding": (lambda W: P.EmbeddingFunction.apply(tokens, W, 2.0), [n(9, 16)]),
            "layer_norm": (P.LayerNormFunction.apply, [n(5, 16), n(16), n(16)]),
            "layer_norm_residual": (lambda x, w, b, r: P.LayerNormFunction.apply(x, w, b, 1e-5, r)[0], [n(5, 16), n(16), n(16), n(5, 16)]),
            "adapters": (lambda y, x, A, B: P.DenseAdaptersFunction.apply(y, x, A, B, which), [h(5, 32), h(5, 16), h(2, 16, 4), h(2, 4, 32)]),
            "gated": (P.DenseGatedFunction.apply, [h(5, 16), h(16, 32), h(16, 32)])}


NAMES = ["embedding", "layer_norm", "layer_norm_residual", "adapters", "gated"]


@pytest.mark.parametrize("required", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_tangents(name, required):
    f, args = operators()[name]
    for k in range(len(args)):
        with forward_ad.dual_level():
            given = [forward_ad.make_dual(t, torch.ones_like(t)) if i == k else t for i, t in enumerate(args)]
            if required:
                given = [t if i == k else t.detach().requires_grad_() for i, t in enumerate(given)]
            with pytest.raises(RuntimeError, match="forward-mode|jvp"):
                f(*given)
    f(*args)


def all_operators():
    """Those of all layers: f(*args), and what of args it has gradients of."""
    import paralleltnnlayers_b200 as P
    n = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    out = {name: (f, args) for name, (f, args) in operators().items()}
    out["cp4"] = P.CP4Conv2dFunction.apply, [n(2, 8, 6, 6), n(8, 4), n(8, 4), n(3, 4), n(3, 4)]
    out["cp3"] = P.CP3Conv2dFunction.apply, [n(2, 8, 6, 6), n(8, 4), n(8, 4), n(3, 3, 4)]
    out["rcp"] = P.RCPConv2dFunction.apply, [n(2, 16, 6, 6), n(3, 3, 4), n(4, 4, 4), n(4, 4, 4)]
    out["dense"] = P.CPDenseFunction.apply, [n(3, 16), n(4, 4, 5), n(4, 4, 5)]
    return out


@pytest.mark.parametrize("name", [*NAMES, "cp4", "cp3", "rcp", "dense"])
def test_gradients_of_gradients(name):
    f, args = all_operators()[name]
    leaves = [t.requires_grad_() for t in args]
    y = f(*leaves)
    dy = torch.randn_like(y).requires_grad_()
    plain = torch.autograd.grad(f(*leaves), leaves, dy.detach())
    again = torch.autograd.grad(y, leaves, dy, create_graph=True)
    for k, (p, q) in enumerate(zip(plain, again)):
        torch.testing.assert_close(p, q.detach())
        if name == "adapters" and k == 0:   # (the gradient of what they are added to is dy itself)
            assert q is dy
            continue
        for wrt in (dy, leaves[-1]):
            penalty = q.float().square().sum() + wrt.float().sum()
            if name == "embedding" and wrt is not dy:   # (its gradient does not depend on the table)
                assert bool((torch.autograd.grad(penalty, wrt, retain_graph=True)[0] == 1).all())
                continue
            with pytest.raises(RuntimeError, match="differentiated again"):
                torch.autograd.grad(penalty, wrt, retain_graph=True)
    # a first-order pass beside a graph of others
    w = torch.ones((), device="cuda", requires_grad=True)
    d, = torch.autograd.grad((w ** 3 * y.detach().float()).sum(), w, create_graph=True)
    f(*leaves).backward(torch.ones_like(y))
    d.backward()
    assert all(t.grad is not None for t in (*leaves, w))


def test_what_is_handed_on():
    """The gradient that comes to the sum before a norm passes it as it is: derivatives through it are there."""
    import paralleltnnlayers_b200 as P
    x, r = (torch.randn(3, 8, device="cuda", requires_grad=True) for _ in range(2))
    _, h = P.LayerNormFunction.apply(x, None, None, 1e-5, r)
    d, = torch.autograd.grad((h ** 3).sum(), r, create_graph=True)
    torch.testing.assert_close(d, 3 * h.detach() ** 2)
    dd, = torch.autograd.grad(d.sum(), r)
    torch.testing.assert_close(dd, 6 * h.detach())
