"""Gradients of tokens that make up much of a batch: their parts are added up in two steps, at the borders of chunks of 8 to 64 places and of 64 chunks."""
import pytest
import torch

from test_embedding_gpu import check_gradient

pytestmark = pytest.mark.gpu


def rows(S, D, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(S, D, generator=gen, device="cuda").to(dtype)


# rows of few values take chunks of eight places: 512 places are a group of chunks
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 8, 13, 64])
@pytest.mark.parametrize("lengths", [(1, 511), (512, 1), (511, 2), (7, 513, 8), (504, 1024), (505, 1031, 600), (512, 512, 512), (1024, 1536, 3, 2048), (20000, 1, 20000, 9000), (5, 40000)], ids=str)
def test_runs_at_borders(lengths, D, dtype):
    import paralleltnnlayers_b200 as P
    t = torch.cat([torch.full((n,), k, device="cuda") for k, n in enumerate(lengths)])
    dY = rows(len(t), D, dtype)
    V = len(lengths)
    check_gradient(P.embedding_backward(dY, t, V, 0.5), t, dY, 0.5)
    check_gradient(P.embedding_backward(dY, t, V - 1, 0.5), t, dY, 0.5)   # (the last ones are none)
    mixed = torch.randperm(len(t), generator=torch.Generator().manual_seed(1)).cuda()
    out = P.embedding_backward(dY, t[mixed], V + 5)
    check_gradient(out, t[mixed], dY, 1.0)
    assert torch.equal(out, P.embedding_backward(dY, t[mixed], V + 5))


@pytest.mark.parametrize("S,D", [(9000, 1024), (5000, 4100), (70000, 264)])
def test_runs_of_long_rows(S, D):
    import paralleltnnlayers_b200 as P
    dY = rows(S, D, torch.bfloat16)
    for share in (0.0, 0.5, 1.0):
        gen = torch.Generator(device="cuda").manual_seed(1)
        t = torch.randint(50, (S,), generator=gen, device="cuda")
        t[torch.rand(S, generator=gen, device="cuda") < share] = 17
        check_gradient(P.embedding_backward(dY, t, 50, 1.0), t, dY, 1.0)


@pytest.mark.parametrize("S,D", [(65536, 8), (65536, 64), (262144, 64)])
def test_time_of_one_token(S, D):
    """A batch of one token takes about as long as one of many (it took 10 to 17 times as long where one CTA had all parts): the best of several, with room."""
    import paralleltnnlayers_b200 as P
    dY = rows(S, D, torch.bfloat16)
    best = []
    for t in (torch.randint(50000, (S,), device="cuda"), torch.full((S,), 3, device="cuda")):
        took = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(4):
                P.embedding_backward(dY, t, 50000)
            b.record()
            b.synchronize()
            took.append(a.elapsed_time(b))
        best.append(min(took))
    assert best[1] < 4 * best[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S,D", [(300, 64), (3000, 8), (3000, 1024), (20000, 264), (1500, 4096), (2000, 513)])
def test_bits_wherever_the_rows_lie(S, D, dtype):
    import paralleltnnlayers_b200 as P
    dY = rows(S, D, dtype)
    off = torch.cat([dY.reshape(-1)[:1], dY.reshape(-1)])[1:].view(S, D)   # (off the boundary of a load)
    assert off.data_ptr() % 16 and torch.equal(off, dY)
    t = torch.randint(7, (S,), generator=torch.Generator().manual_seed(2)).cuda()
    assert torch.equal(P.embedding_backward(dY, t, 9), P.embedding_backward(off, t, 9))
