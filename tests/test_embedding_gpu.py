"""Embedding and its gradient against their definition in 64 bits.

A result is rounded once to its type (half a step: eps / 2 of the value) after one product in fp32 (half a step of fp32).  A gradient is a sum of n terms in
fp32, each of n additions off by at most 2**-24 of the largest partial sum, which is at most the sum of magnitudes, then scaled (2**-24) and rounded to the type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
NUMBERS = [torch.int32, torch.int64]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the spacing of the subnormal numbers: what rounding adds near zero."""
    return torch.finfo(dtype).tiny * half(dtype)


def draw(S, V, D, dtype, numbers, seed=0, bare=0.1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    W = torch.randn(V, D, generator=gen, device="cuda").to(dtype)
    t = torch.randint(V, (S,), generator=gen, device="cuda")
    t[torch.rand(S, generator=gen, device="cuda") < bare] = -1
    return t.to(numbers), W, torch.randn(S, D, generator=gen, device="cuda").to(dtype)


def check_gradient(dW, tokens, dY, scale):
    V, dtype = dW.shape[0], dW.dtype
    t, d = tokens.reshape(-1).long(), dY.reshape(-1, dY.shape[-1]).double()
    inside = (t >= 0) & (t < V)
    want = torch.zeros(dW.shape, dtype=torch.float64, device=dW.device).index_add_(0, t[inside], d[inside]) * scale
    sizes = torch.zeros(dW.shape, dtype=torch.float64, device=dW.device).index_add_(0, t[inside], d[inside].abs()) * abs(scale)
    n = torch.zeros(V, dtype=torch.float64, device=dW.device).index_add_(0, t[inside], torch.ones_like(t[inside], dtype=torch.float64))
    fp32 = 2.0 ** -24
    bound = (n.view(-1, 1) + 2) * fp32 * sizes
    bound = bound + half(dtype) * (want.abs() + bound) + least(dtype)
    assert dW.shape == want.shape and bool(((dW.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("numbers", NUMBERS)
@pytest.mark.parametrize("S,V,D", [(1, 1, 1), (1, 16, 8), (2, 7, 3), (31, 1000, 65), (1000, 31, 256), (257, 5, 513), (40, 70000, 24), (3000, 1023, 40), (2048, 1024, 2056)])
def test_forward_and_gradient(S, V, D, numbers, dtype):
    import paralleltnnlayers_b200 as P
    t, W, dY = draw(S, V, D, dtype, numbers, seed=S + D)
    scale = 1.7
    W.requires_grad_()
    out = P.EmbeddingFunction.apply(t, W, scale)
    held = (t >= 0).view(-1, 1)
    want = torch.where(held, W.detach().double()[t.clamp(min=0).long()] * scale, 0)
    bound = (half(dtype) + 2.0 ** -23) * want.abs() + least(dtype)   # (scale itself is rounded to fp32)
    assert bool(((out.detach().double() - want).abs() <= bound).all())
    dW, = torch.autograd.grad(out, W, dY)
    check_gradient(dW, t, dY, scale)
    assert torch.equal(out.detach(), P.embedding(t, W.detach(), scale))
    assert torch.equal(dW, P.embedding_backward(dY, t, V, scale))


def test_scale_one_copies_rows():
    import paralleltnnlayers_b200 as P
    for dtype in TYPES:
        t, W, _ = draw(300, 50, 72, dtype, torch.int64, bare=0.0)
        W[7, 3] = float("inf")
        W[8, 4] = float("nan")
        t[0], t[1] = 7, 8
        assert torch.equal(P.embedding(t, W).nan_to_num(5.0), W[t].nan_to_num(5.0))


@pytest.mark.parametrize("numbers", NUMBERS)
def test_numbers_outside_are_none(numbers):
    import paralleltnnlayers_b200 as P
    big = torch.iinfo(numbers).max
    t = torch.tensor([[0, -1, 4, 5], [big, -big, 3, 6]], device="cuda", dtype=numbers)
    W = torch.randn(5, 16, device="cuda")
    out = P.embedding(t, W, 2.0)
    assert out.shape == (2, 4, 16)
    held = (t >= 0) & (t < 5)
    assert torch.equal(out[held], 2 * W[t[held].long()]) and not out[~held].any()
    dY = torch.randn(2, 4, 16, device="cuda")
    dY[~held] = float("nan")   # (what comes to a place without a token is not read into a sum)
    dW = P.embedding_backward(dY, t, 5, 2.0)
    want = torch.zeros(5, 16, device="cuda")
    want[t[held].long()] = 2 * dY[held]
    assert torch.equal(dW, want)
    assert not P.embedding_backward(dY, torch.full_like(t, -1), 5).any()


@pytest.mark.parametrize("S,D", [(5000, 40), (70001, 8), (4096, 1032)])
@pytest.mark.parametrize("kind", ["one", "two", "runs", "skewed"])
def test_tokens_of_many_places(S, D, kind):
    """A token's places reach over many parts of the sorted batch."""
    import paralleltnnlayers_b200 as P
    gen = torch.Generator(device="cuda").manual_seed(S)
    i = torch.arange(S, device="cuda")
    t = {"one": torch.full_like(i, 3), "two": i % 2 * 4, "runs": i // 777, "skewed": (torch.rand(S, generator=gen, device="cuda") ** 8 * 600).long()}[kind]
    dY = torch.randn(S, D, generator=gen, device="cuda")
    dW = P.embedding_backward(dY, t, 601, 0.5)
    check_gradient(dW, t, dY, 0.5)
    assert torch.equal(dW, P.embedding_backward(dY, t.int(), 601, 0.5))


def test_large_tables_take_several_digits():
    import paralleltnnlayers_b200 as P
    for V in (1023, 1024, 1 << 20, (1 << 21) + 5):
        t = torch.tensor([V - 1, 0, 5, V - 1, 1000, V // 2, 0], device="cuda")
        dY = torch.randn(7, 4, device="cuda")
        dW = P.embedding_backward(dY, t, V)
        rows = torch.tensor(sorted(set(t.tolist())), device="cuda")
        want = torch.stack([sum(dY[k] for k in range(7) if int(t[k]) == int(r)) for r in rows])
        assert torch.allclose(dW[rows], want, rtol=2.0 ** -22, atol=2.0 ** -22)
        dW[rows] = 0
        assert not dW.any()


def test_no_rows_and_views():
    import paralleltnnlayers_b200 as P
    W = torch.randn(9, 20, device="cuda", dtype=torch.bfloat16)
    none = torch.zeros(0, 3, device="cuda", dtype=torch.int64)
    assert P.embedding(none, W).shape == (0, 3, 20)
    assert not P.embedding_backward(torch.zeros(0, 3, 20, device="cuda"), none, 9).any()
    t = torch.randint(9, (6, 10), device="cuda")
    assert torch.equal(P.embedding(t.t(), W), W[t.t()])
    wide = torch.randn(9, 41, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(P.embedding(t[:, ::2], wide[:, 1:21]), wide[:, 1:21][t[:, ::2]])   # (rows off their boundaries)
    flat = torch.randn(9 * 24 + 1, device="cuda")[1:].view(9, 24)
    assert torch.equal(P.embedding(t, flat), flat[t])
    dY = torch.randn(10, 6, 24, device="cuda")
    check_gradient(P.embedding_backward(dY.transpose(0, 1), t, 9), t, dY.transpose(0, 1), 1.0)


def test_streams_graphs_and_the_same_bits():
    import paralleltnnlayers_b200 as P
    t, W, dY = draw(4000, 900, 136, torch.float32, torch.int64, seed=3)
    want = P.embedding_backward(dY, t, 900)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(P.embedding_backward(dY, t, 900), want)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):   # two graphs of one pool
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
            got = P.embedding_backward(dY, t, 900)
            out = P.embedding(t, W, 3.0)
        graphs.append((g, got, out))
    for k in range(3):
        g, got, out = graphs[k % 2]
        g.replay()
        assert torch.equal(got, want) and torch.equal(out, P.embedding(t, W, 3.0))
    t.copy_(t.flip(0))
    graphs[0][0].replay()
    check_gradient(graphs[0][1], t, dY, 1.0)
