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
