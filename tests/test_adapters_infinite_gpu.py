"""Infinities in the rows of the adapters' operands: the sums that the definition gives, at ranks below and at a tile of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rank", [1, 4, 16, 17, 24, 40, 100, 128])
@pytest.mark.parametrize("rows", [10, 200])
def test_an_infinite_value_gives_an_infinite_row(rows, rank, dtype):
    """Factors above zero: a row with one infinity has infinite V, and so an infinite result in every column; the other rows are finite.  A scale below zero turns
    the sign."""
    import paralleltnnlayers_b200 as P
    gen = torch.Generator(device="cuda").manual_seed(rows + rank)
    r = lambda *s: (torch.rand(*s, generator=gen, device="cuda") + 0.5).to(dtype)  # noqa: E731
    I, O = 72, 48
    x, y, A, B, dy = r(rows, I), r(rows, O), r(2, I, rank), r(2, rank, O), r(rows, O)
    which = torch.arange(rows, device="cuda", dtype=torch.int32) % 2
    scale = torch.tensor([0.5, -0.25], device="cuda")
    x[3, 5] = x[6, 70] = dy[2, 47] = dy[9, 0] = float("inf")
    leaves = [t.requires_grad_() for t in (y, x, A, B)]
    out = P.DenseAdaptersFunction.apply(*leaves, which, scale)
    _, dx, dA, dB = torch.autograd.grad(out, leaves, dy)
    bare = P.dense_adapters(y.detach(), x.detach(), A.detach(), B.detach(), which, scale)
    for got in (out.detach(), bare):
        sign = torch.where(which % 2 == 0, 1.0, -1.0).view(-1, 1)
        want = torch.zeros(rows, O, device="cuda")
        want[3], want[6] = float("inf"), float("inf")
        infinite = torch.isinf(got)
        assert torch.equal(infinite, torch.isinf(want)) and not bool(torch.isnan(got).any())
        assert torch.equal(got.float()[infinite] > 0, (want * sign)[infinite] > 0)
    want = torch.zeros(rows, I, device="cuda")
    want[2], want[9] = float("inf"), -float("inf")
    assert torch.equal(torch.isinf(dx), torch.isinf(want)) and not bool(torch.isnan(dx).any())
    assert bool((dx[2] > 0).all()) and bool((dx[9] < 0).all())
    # dA sums x over an adapter's rows with an infinite W, dB the infinite V with dY: infinite in all its places, none of them NaN
    for g in (dA, dB):
        assert bool(torch.isinf(g).all())
    assert bool((dA[0] > 0).all()) and bool((dA[1] < 0).all()) and bool((dB[1] < 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_a_value_that_is_not_finite_in_the_gradient_stays_in_its_column(dtype):
    """dY at (row, column): dB of that row's adapter in that column alone, dA of that adapter; every other adapter is what it is without."""
    import paralleltnnlayers_b200 as P
    gen = torch.Generator(device="cuda").manual_seed(5)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    rows, I, O, R, count = 150, 136, 72, 16, 5
    x, y, A, B, dy = n(rows, I), n(rows, O), n(count, I, R), n(count, R, O), n(rows, O)
    which = torch.randint(count, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    row = int((which == 1).nonzero()[0])

    def grads(d):
        leaves = [t.clone().requires_grad_() for t in (y, x, A, B)]
        return torch.autograd.grad(P.DenseAdaptersFunction.apply(*leaves, which), leaves[1:], d)

    clean = grads(dy)
    bad = dy.clone()
    bad[row, 7] = float("nan")
    dx, dA, dB = grads(bad)
    rest = torch.arange(count, device="cuda") != 1
    columns = torch.arange(O, device="cuda") != 7
    others = torch.arange(rows, device="cuda") != row
    assert torch.equal(dx[others], clean[0][others]) and bool(torch.isnan(dx[row]).all())
    assert torch.equal(dA[rest], clean[1][rest]) and bool(torch.isnan(dA[1]).all())
    assert torch.equal(dB[rest], clean[2][rest]) and torch.equal(dB[1][:, columns], clean[2][1][:, columns]) and bool(torch.isnan(dB[1][:, 7]).all())
