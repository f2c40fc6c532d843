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
