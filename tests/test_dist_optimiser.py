"""One optimiser over several layers, handed to the data-parallel step of each."""
import pytest
import torch


def _two(**kw):
    return [torch.nn.Parameter(torch.zeros(3, **kw)) for _ in range(2)]


@pytest.mark.parametrize("make", [lambda p: torch.optim.SGD(p, lr=1.0), lambda p: torch.optim.SGD([{"params": [p[0]]}, {"params": [p[1]]}], lr=1.0)])
def test_a_step_leaves_the_other_layers_alone(make):
    from paralleltnnlayers_b200.dist import _update
    a, b = _two()
    opt = make([a, b])
    one, two = torch.ones(3), 2 * torch.ones(3)
    _update(opt, [a], [one])
    assert torch.equal(a.detach(), -one) and not bool(b.detach().any())
    _update(opt, [b], [two])
    assert torch.equal(a.detach(), -one) and torch.equal(b.detach(), -two)
    assert a.grad is one and b.grad is two   # as each step left them
    with pytest.raises(ValueError, match="over the factors"):
        _update(opt, [torch.nn.Parameter(torch.zeros(3))], [one])
    assert a.grad is one and torch.equal(a.detach(), -one)


def test_gradients_come_back_where_the_optimiser_fails():
    from paralleltnnlayers_b200.dist import _update
    a, b = _two()

    class Fails(torch.optim.SGD):
        def step(self, closure=None):
            raise RuntimeError("no step")

    a.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="no step"):
        _update(Fails([a, b], lr=1.0), [b], [torch.ones(3)])
    assert torch.equal(a.grad, torch.ones(3))


@pytest.mark.gpu
def test_two_layers_under_one_optimiser():
    """Each layer's first step is the rate times its gradient's sign, once."""
    from paralleltnnlayers_b200 import dist as D
    from paralleltnnlayers_b200.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    layers = [[torch.nn.Parameter(n(4, 4, 3)), torch.nn.Parameter(n(4, 2, 3))] for _ in range(2)]
    start = [[p.detach().clone() for p in F] for F in layers]
    opt = AdamW([p for F in layers for p in F], lr=1e-2, weight_decay=0.0)
    grads = [D.dense_data_parallel_step(n(7, 16), n(7, 8), F, optimizer=opt)[2] for F in layers]
    for F, before, gs in zip(layers, start, grads):
        for p, b, g in zip(F, before, gs):
            big = g.abs() > 1e-3
            assert bool(((p.detach() - b + 1e-2 * g.sign())[big].abs() < 1e-6 + 2.0 ** -22 * b.abs()[big]).all())
            assert opt.state[p]["step"] == 1
