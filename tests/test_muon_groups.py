"""Parameter groups of the Muon optimiser."""
import pytest
import torch

from paralleltnnlayers_b200 import optim


@pytest.mark.parametrize("form", [lambda p: p, lambda p: [p], lambda p: (q for q in [torch.nn.Parameter(torch.zeros(2, 2)), p]), lambda p: [("name", p)]], ids=("one", "list", "generator", "named"))
def test_a_refused_group_is_not_kept(form):
    named = isinstance(form(None), list) and form(None)[0] == ("name", None)
    first, vector = torch.nn.Parameter(torch.zeros(3, 4)), torch.nn.Parameter(torch.zeros(5))
    o = optim.Muon([("first", first)] if named else [first])
    groups = [dict(g) for g in o.param_groups]
    with pytest.raises(ValueError, match="Muon is for matrices"):
        o.add_param_group({"params": form(vector)})
    assert o.param_groups == groups
    o.add_param_group({"params": form(torch.nn.Parameter(torch.zeros(5, 6))), "lr": 0.5})
    assert len(o.param_groups) == 2 and o.param_groups[1]["lr"] == 0.5


def test_a_vector_among_the_first_parameters():
    with pytest.raises(ValueError, match="Muon is for matrices"):
        optim.Muon([torch.nn.Parameter(torch.zeros(3, 4)), torch.nn.Parameter(torch.zeros(()))])
