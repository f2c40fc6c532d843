"""Embedding, layer norm and the Muon step over arrays of more than 2^31 values: the rows at their far ends, against the same rows by themselves."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory():
    if torch.cuda.mem_get_info()[0] < 70 << 30:
        pytest.skip("takes 70 GB")
    yield
    torch.cuda.empty_cache()


def far(t, rows):
    """The first rows, some around 2^31 values, and the last ones."""
    per = t[0].numel()
    at = (1 << 31) // per
    return torch.cat([torch.arange(rows), torch.arange(at - rows, at + rows), torch.arange(len(t) - rows, len(t))]).cuda()


@pytest.mark.parametrize("D", [8192, 8191])
def test_embedding(D):
    import paralleltnnlayers_b200 as P
    S = V = (1 << 31) // D + 3000
    W = torch.empty(V, D, dtype=torch.bfloat16, device="cuda").normal_()
    t = torch.arange(V - 1, -1, -1, device="cuda")
    out = P.embedding(t, W, 2.0)
    at = far(out, 500)
    assert torch.equal(out[at], 2 * W[V - 1 - at])
    dW = P.embedding_backward(out, t, V, 0.5)
    assert torch.equal(dW[at], W[at])
    t[S // 2:] = 3
    dW = P.embedding_backward(out, t, V, 1.0)
    want = out[S // 2:].double().sum(0)
    # (a sum of 1.3e5 terms in fp32, and its rounding)
    assert bool(((dW[3].double() - want).abs() <= 2.0 ** -24 * (S + 2) * out[S // 2:].float().abs().sum(0).double() + 2.0 ** -8 * want.abs()).all())
    assert torch.equal(dW[V - 1 - S // 2 + 1:], out[:S // 2].flip(0)) and not dW[4:V - 1 - S // 2].any()


@pytest.mark.parametrize("D", [4096, 4095, 40000])
def test_layer_norm(D):
    import paralleltnnlayers_b200 as P
    S = (1 << 31) // D + 2000
    x, dy = (torch.empty(S, D, dtype=torch.bfloat16, device="cuda").normal_() for _ in range(2))
    w = torch.empty(D, dtype=torch.bfloat16, device="cuda").normal_()
    y, mean, rstd = P.layer_norm_save(x, w)
    dx, _, db = P.layer_norm_backward(dy, x, w, None, mean, rstd, need_dw=False)
    at = far(x, 300)
    y1, mean1, rstd1 = P.layer_norm_save(x[at], w)
    assert torch.equal(y[at], y1) and torch.equal(mean[at], mean1) and torch.equal(rstd[at], rstd1)
    dx1, _, _ = P.layer_norm_backward(dy[at], x[at], w, None, mean1, rstd1, need_dw=False)
    assert torch.equal(dx[at], dx1)
    sums, sizes = torch.zeros(D, dtype=torch.float64, device="cuda"), torch.zeros(D, dtype=torch.float64, device="cuda")
    for part in dy.split(20000):
        sums += part.double().sum(0)
        sizes += part.double().abs().sum(0)
    assert bool(((db.double() - sums).abs() <= S * 2.0 ** -24 * sizes + 2.0 ** -8 * sums.abs()).all())


@pytest.mark.parametrize("shape", [(40, 60, 900000), (35000, 256, 256)], ids=str)
def test_muon(shape):
    import paralleltnnlayers_b200 as P
    X = torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_()
    out = P.orthogonalise(X)
    for k in (0, shape[0] - 1, (1 << 31) // (shape[1] * shape[2])):
        alone = P.orthogonalise(X[k])
        # (a matrix by itself may be cut into other parts: 64-bit sums in another order)
        assert float((out[k].float() - alone.float()).norm()) <= 2.0 ** -8 * float(alone.float().norm())
    P.device_status()


def test_muon_one_matrix():
    import paralleltnnlayers_b200 as P
    X = torch.empty(72, 16700001, device="cuda").normal_()
    Y = torch.empty(130, 16700001, device="cuda", dtype=torch.bfloat16).normal_()
    for Z in (X, Y):
        out = P.orthogonalise(Z, steps=2)
        n = Z.shape[0]
        A = torch.zeros(n, n, dtype=torch.float64, device="cuda")
        G = torch.zeros(n, n, dtype=torch.float64, device="cuda")
        for a, b in zip(Z.split(1000000, 1), out.split(1000000, 1)):
            A += a.double() @ a.double().T
            G += b.double() @ b.double().T
        S = torch.linalg.eigvalsh(A / A.trace()).clamp(min=0).sqrt()
        for _ in range(2):
            S = 3.4445 * S - 4.7750 * S ** 3 + 2.0315 * S ** 5
        got = torch.linalg.eigvalsh(G).clamp(min=0).sqrt()
        assert bool(((got - S.sort().values).abs() <= 2.0 ** -7 * S.max()).all())
        # far columns, as the definition has them: X P with P of the Gram matrix
        A = A / A.trace()
        Q = torch.eye(n, dtype=torch.float64, device="cuda")
        B = A
        for _ in range(2):
            P1 = 3.4445 * torch.eye(n, dtype=torch.float64, device="cuda") - 4.7750 * B + 2.0315 * B @ B
            Q, B = P1 @ Q, P1 @ B @ P1
        norm = float(Z.float().norm())
        want = Q @ (Z[:, -5000:].double() / norm)
        off = out[:, -5000:].double() - want
        assert float(off.norm()) <= (2.0 ** -8 if Z.dtype == torch.bfloat16 else 2.0 ** -16) * float(want.norm())
