"""The counts of steps of a capturable optimiser: every parameter is corrected by the steps that it has taken itself."""
import copy
import pickle

import pytest
import torch


@pytest.fixture
def calls(lib_built, monkeypatch):
    """The optimiser's own work on the CPU: what it hands to the step, in place of the launch."""
    from paralleltnnlayers_b200 import ops
    seen = []

    def step(params, grads, exp_avg, exp_avg_sq, step, lr, *rest):
        seen.append((len(params), int(step)))

    monkeypatch.setattr(ops, "adamw_step", step)
    return seen


def _optimiser(n=3, **kw):
    from paralleltnnlayers_b200.optim import AdamW
    p = [torch.nn.Parameter(torch.zeros(4)) for _ in range(n)]
    return p, AdamW(p, capturable=True, **kw)


def _grads(params, have):
    for k, p in enumerate(params):
        p.grad = torch.ones(4) if k in have else None


@pytest.mark.parametrize("schedule,want", [
    ([{0, 1, 2}] * 3, [3, 3, 3]),
    ([{0, 1}, {0, 1}, {0, 1, 2}], [3, 3, 1]),          # one that comes later
    ([{0, 1, 2}, {0}, {0, 1, 2}], [3, 2, 2]),          # two that miss a step
    ([{0}, {1}, {0}, {1}, {2}], [2, 2, 1]),            # a step of each layer in turn
    ([{0, 1, 2}, {1, 2}, {1}, {0, 1, 2}], [2, 4, 3]),
])
def test_a_parameter_counts_its_own_steps(calls, schedule, want):
    p, opt = _optimiser()
    counts = [0, 0, 0]
    for have in schedule:
        _grads(p, have)
        calls.clear()
        opt.step()
        for k in have:
            counts[k] += 1
        assert sorted(t for m, t in calls for _ in range(m)) == sorted(counts[k] for k in have)
    assert [int(opt.state[q]["step"]) for q in p] == counts == want


def test_parameters_that_step_together_share_a_count_and_a_launch(calls):
    p, opt = _optimiser()
    for _ in range(3):
        _grads(p, {0, 1, 2})
        opt.step()
    assert calls == [(3, 1), (3, 2), (3, 3)] and len({id(opt.state[q]["step"]) for q in p}) == 1


def test_copies_and_saved_states_keep_the_counts(calls):
    p, opt = _optimiser()
    for have in ({0, 1}, {0, 1, 2}):
        _grads(p, have)
        opt.step()
    q, loaded = _optimiser()
    loaded.load_state_dict(opt.state_dict())
    _grads(q, {0, 1, 2})
    for other, ps in ((loaded, q), (copy.deepcopy(opt), None), (pickle.loads(pickle.dumps(opt)), None)):
        ps = ps or other.param_groups[0]["params"]
        _grads(ps, {0, 1, 2})
        assert other.state[ps[0]]["step"] is other.state[ps[1]]["step"]
        other.step()
        assert [int(other.state[a]["step"]) for a in ps] == [3, 3, 2] and other.state[ps[0]]["step"].dtype == torch.int64
    assert [int(opt.state[a]["step"]) for a in p] == [2, 2, 1]
    # between an optimiser that is captured and one that is not
    from paralleltnnlayers_b200.optim import AdamW
    r = [torch.nn.Parameter(torch.zeros(4)) for _ in range(3)]
    eager = AdamW(r)
    _grads(r, {0, 2})
    eager.step()
    assert [eager.state[a]["step"] for a in (r[0], r[2])] == [1, 1]


@pytest.mark.gpu
def test_late_parameters_are_updated_as_by_an_eager_optimiser():
    from paralleltnnlayers_b200.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(0)
    start = [torch.randn(s, generator=gen, device="cuda") for s in (40, 300, 7)]
    twins = [[torch.nn.Parameter(a.clone()) for a in start] for _ in range(2)]
    opts = [AdamW(p, lr=1e-2, capturable=c) for p, c in zip(twins, (False, True))]
    for have in ({0, 1}, {0, 1}, {0, 1, 2}, {1}, {0, 1, 2}):
        grads = [torch.randn(a.shape, generator=gen, device="cuda") for a in start]
        for p, opt in zip(twins, opts):
            for k, q in enumerate(p):
                q.grad = grads[k].clone() if k in have else None
            opt.step()
        for a, b in ((a.detach(), b.detach()) for a, b in zip(*twins)):   # a rate that is rounded the other way moves a sum by one place at most, in each of five steps
            assert float((a - b).abs().max()) <= 6 * 2.0 ** -23 * float(a.abs().max())


@pytest.mark.gpu
def test_a_capture_begins_and_divides_nothing():
    """Refused while a stream is captured; the capture itself ends in order and the optimiser goes on."""
    from paralleltnnlayers_b200.optim import AdamW
    p = [torch.nn.Parameter(torch.ones(5, device="cuda")) for _ in range(2)]
    for q in p:
        q.grad = torch.ones_like(q)

    def refused(opt, match):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match=match):
                opt.step()
            torch.zeros(1, device="cuda")   # something to capture

    opt = AdamW(p, capturable=True)
    refused(opt, "begins no state")
    refused(AdamW(p), "capturable=True alone")
    opt.step()
    p[1].grad = None
    refused(opt, "divides no count")
    p[1].grad = torch.ones_like(p[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    assert [int(opt.state[q]["step"]) for q in p] == [2, 2]
