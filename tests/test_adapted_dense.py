"""The adapted layer as a module: its conversions."""
import pytest
import torch


def _layer(scale):
    from paralleltnnlayers_b200 import layers as L
    return L.AdaptedDense(torch.nn.Linear(6, 4), 3, 2, scale=scale)


@pytest.mark.parametrize("scale", [0.1, 1 / 3, 1e6, 1e-9])
def test_the_scales_keep_their_values_where_the_type_changes(scale):
    """Through 16 bits they would be off by 2**-9, or infinite, or nothing."""
    want = torch.full((3,), scale, dtype=torch.float32)
    for change in (lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: m.to("cpu", torch.float16).bfloat16().float(),
                   lambda m: torch.nn.Sequential(m).half()[0]):
        m = change(_layer(scale))
        assert m.scale.dtype == torch.float32 and torch.equal(m.scale, want)
        assert "scale" in m.state_dict() and m.A.dtype == m.B.dtype
    m = _layer(scale).to("meta")
    assert m.scale.is_meta and m.half().scale.dtype == torch.float32
    assert m.to_empty(device="cpu").scale.shape == (3,)


@pytest.mark.gpu
def test_the_scales_move_with_the_layer():
    m = _layer(0.1).to("cuda", torch.bfloat16)
    assert m.scale.is_cuda and torch.equal(m.scale.cpu(), torch.full((3,), 0.1))
    assert torch.equal(m.cpu().scale, torch.full((3,), 0.1)) and torch.equal(m.cuda().scale.cpu(), torch.full((3,), 0.1))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,launches", [(1, 1), (64, 1), (256, 1), (257, 2)])
def test_a_layer_that_serves_takes_the_launches_of_the_operator(rows, launches):
    """One launch beyond the shared layer's for up to 256 rows, as dense_adapters itself, where nothing is kept for a backward."""
    import paralleltnnlayers_b200 as P
    from paralleltnnlayers_b200 import layers as L
    torch.manual_seed(rows)
    m = L.AdaptedDense(L.CPDense(256, 64, rank=12, input_shape=(16, 16), output_shape=(8, 8)), count=3, rank=8, scale=0.5).cuda()
    with torch.no_grad():
        m.B.normal_(0, 0.2)
    x, which = torch.randn(rows, 256, device="cuda"), torch.randint(-1, 3, (rows,), device="cuda", dtype=torch.int32)
    y = m.shared(x).detach()

    def run(f):
        k = P.launch_count()
        return f(), P.launch_count() - k

    _, shared = run(lambda: m.shared(x))
    want, bare = run(lambda: P.dense_adapters(y, x, m.A, m.B, which, m.scale))
    assert bare == launches
    with torch.no_grad():
        out, n = run(lambda: m(x, which))
        assert n == shared + launches and torch.equal(out, want) and not out.requires_grad
        plan = P.adapter_plan(which, 3)
        out, n = run(lambda: m(x, plan))
        assert n == shared + 1 and torch.equal(out, want)
    m.requires_grad_(False)
    out, n = run(lambda: m(x, which))
    assert n == shared + launches and torch.equal(out, want) and not out.requires_grad
    m.B.requires_grad_()
    out, n = run(lambda: m(x, which))
    assert n == shared + 2 and torch.equal(out.detach(), want) and out.requires_grad   # a plan, which the backward needs
