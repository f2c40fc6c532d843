"""What the Muon step's products are worth: results of 16 bits are those of float32, rounded once; sums of any length; the wide tiles, blocks of bands and
matrices that do not go together, which the small shapes of test_muon_gpu.py do not reach.  Bounds are that file's."""
import pytest
import torch

from test_muon_gpu import check, defined, matrices

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(40, 100), (64, 64), (65, 65), (300, 66), (257, 513), (640, 129), (3, 70, 90), (104, 6777)], ids=str)
def test_results_of_16_bits(shape, dtype):
    """The same values in float32 go through the same operations: the bits are those of its result, rounded."""
    import paralleltnnlayers_b200 as P
    X = matrices(*shape, seed=sum(shape)).to(dtype)
    assert torch.equal(P.orthogonalise(X), P.orthogonalise(X.float()).to(dtype))
    p, q = torch.zeros_like(X), torch.zeros(shape, device="cuda")
    P.muon_step([p], [X], [torch.zeros_like(q)], 1.0)
    P.muon_step([q], [X.float()], [torch.zeros_like(q)], 1.0)
    assert torch.equal(p, q.to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(80, 300001), (200003, 72)], ids=str)
def test_long_sums(shape, dtype):
    """An accumulator of the tensor cores holds 256 terms, however many a sum has: what they cut off does not grow with it."""
    import paralleltnnlayers_b200 as P
    X = matrices(*shape, seed=4).to(dtype)
    out = P.orthogonalise(X)
    check(out, *defined(X))
    assert torch.equal(out, P.orthogonalise(X.float()).to(dtype))


# tiles of 256 x 256 (A and B of the first two, X of the others), blocks of more than 16 rows of tiles, and matrices of 1.5 GB of planes and more
@pytest.mark.parametrize("shape", [(3, 1100, 1111), (3, 1111, 1100), (2, 1300, 1301), (2, 1301, 1290), (4500, 300), (300, 4500), (4300, 1400)], ids=str)
def test_wide_tiles_and_bands(shape):
    import paralleltnnlayers_b200 as P
    X = matrices(*shape, seed=6)
    out = P.orthogonalise(X)
    check(out, *defined(X))
    assert torch.equal(out, P.orthogonalise(X))
    P.device_status()


def test_more_than_goes_together():
    """Two of these fit the planes that share launches, the third does not; a smaller one joins it."""
    import paralleltnnlayers_b200 as P
    shapes = [(70, 1000064)] * 3 + [(100, 90)]
    g = [matrices(*s, seed=k) for k, s in enumerate(shapes)]
    p = [torch.zeros(*s, device="cuda") for s in shapes]
    P.muon_step(p, g, [torch.zeros_like(t) for t in p], 1.0, momentum=0.0, weight_decay=0.0, adjust=None)
    for a, b in zip(p, g):
        check(-a, *defined(b))
    P.device_status()
