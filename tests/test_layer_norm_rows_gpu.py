"""Rows whose statistics are at an edge: gradients of rows of one value, statistics of rows that are not finite."""
import pytest
import torch

from test_layer_norm_gpu import check, defined

pytestmark = pytest.mark.gpu
SIZES = [40, 256, 300, 1000, 1001, 4096, 4100, 8192, 9000, 9001]   # a size or two of each kernel


@pytest.mark.parametrize("D", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_rows_of_one_value(D, dtype):
    """Their deviations are exactly 0, and so is what they give to the weight's gradient.  (The mean is the value itself: a sum's rounding is corrected by the sum of the
    deviations, whose own rounding is far below a step of the mean.)"""
    import paralleltnnlayers_b200 as P
    gen = torch.Generator(device="cuda").manual_seed(D)
    x = torch.tensor([0.1, -3.5, 100.3, 12345.6, 0.0, -7e4], device="cuda").to(dtype).unsqueeze(1).expand(6, D).contiguous()
    dy, w = torch.randn(6, D, generator=gen, device="cuda").to(dtype), torch.randn(D, generator=gen, device="cuda").to(dtype)
    y, mean, rstd = P.layer_norm_save(x, w)
    dx, dw, db = P.layer_norm_backward(dy, x, w, None, mean, rstd)
    assert torch.equal(mean, x[:, 0].float()) and not y.any() and not dw.any()
    (_, want, _, sums), (_, bound, _, slack) = defined(x, w, None, 1e-5, dy, None)
    check(dx, want, bound, "dx")
    check(db, sums, slack, "db")


@pytest.mark.parametrize("D", [*SIZES, 40000])
def test_statistics_of_rows_that_are_not_finite(D):
    import paralleltnnlayers_b200 as P
    x = torch.randn(5, D, device="cuda")
    _, m, r = P.layer_norm_save(x)
    z = x.clone()
    z[1, D // 2], z[2, 1], z[3] = float("nan"), float("inf"), float("-inf")
    y, mean, rstd = P.layer_norm_save(z)
    assert y[1:4].isnan().all() and rstd[1:4].isnan().all() and not mean[1:4].isfinite().any()
    for k in (0, 4):
        assert torch.equal(mean[k], m[k]) and torch.equal(rstd[k], r[k])
    dx, dw, db = P.layer_norm_backward(torch.ones_like(z), z, torch.ones(D, device="cuda"), None, mean, rstd)
    assert dx[1:4].isnan().all() and dw.isnan().all() and bool((db == 5).all()) and dx[[0, 4]].isfinite().all()
