"""Slopes of the gate's activations over the whole range of float32."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_slopes_far_out(act):
    """Wg the identity and Wu zero: dX is dG, U act'(G) dH with U = dH = 1, rounded once to bfloat16.  Up to |G| = 10 the slope has the error of a handful of
    fp32 operations and of an exponential that is within (G^2 / 2 + 8) 2**-23; from some tens on it is 0 or 1."""
    import paralleltnnlayers_b200 as P
    n = 64
    far = torch.cat([10.0 ** torch.arange(1.5, 38.6, 0.5), torch.tensor([3.0e38])]).to(torch.float32)
    near = torch.linspace(0, 10, 2 * n)
    G = torch.cat([far, -far, near, -near])
    G = torch.nn.functional.pad(G, (0, -G.numel() % n)).view(-1, n).contiguous().cuda()
    rows = G.shape[0]
    b16 = dict(dtype=torch.bfloat16, device="cuda")
    dx, dWg, dWu = P.dense_gated_backward(torch.ones(rows, n, **b16), torch.zeros(rows, n, **b16), torch.eye(n, **b16), torch.zeros(n, n, **b16), G,
                                          torch.ones_like(G), act)
    g = G.double().cpu()
    if act == "silu":
        s = torch.sigmoid(g)
        want = s + g * s * torch.sigmoid(-g)
    elif act == "gelu":
        want = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5) + g * torch.exp(-0.5 * g * g) * (0.5 / torch.pi) ** 0.5
    else:
        c = (2 / torch.pi) ** 0.5
        q = c * (g + 0.044715 * g ** 3)
        s, t = torch.sigmoid(2 * q), torch.sigmoid(-2 * q)
        want = s + torch.where(s * t > 0, 2 * g * s * t * c * (1 + 3 * 0.044715 * g * g), 0.0)
    assert bool(torch.isfinite(want).all())
    err = (dx.double().cpu() - want).abs()
    bound = 2.0 ** -8 * want.abs() + (g.abs().clamp(max=100) ** 2 / 2 + 16) * 2.0 ** -22
    worst = float((err / bound).max())
    assert worst <= 1, worst   # (a NaN is not)
    assert not bool(dWg.any()) and not bool(dWu.any())
