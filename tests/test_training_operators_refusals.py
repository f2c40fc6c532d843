"""What the embedding, layer norm and the Muon step refuse, before anything is launched, and their layers and optimiser on the host."""
import ctypes as C

import pytest
import torch

BF16, I64 = torch.bfloat16, torch.int64


@pytest.fixture
def fake(lib_built):
    """Fake CUDA tensors: nothing can be launched."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        yield lambda *size, dev=0, dtype=torch.float32: torch.empty(*size, device=f"cuda:{dev}", dtype=dtype)


CALLS = {
    "tokens type": (TypeError, lambda P, c: P.embedding(c(3), c(5, 4))),
    "tokens device": (ValueError, lambda P, c: P.embedding(c(3, dtype=I64, dev=1), c(5, 4))),
    "tokens on the host": (TypeError, lambda P, c: P.embedding(torch.zeros(3, dtype=I64), c(5, 4))),
    "table type": (TypeError, lambda P, c: P.embedding(c(3, dtype=I64), c(5, 4, dtype=torch.float64))),
    "table shape": (ValueError, lambda P, c: P.embedding(c(3, dtype=I64), c(5, 4, 2))),
    "empty table": (ValueError, lambda P, c: P.embedding(c(3, dtype=I64), c(0, 4))),
    "gradient shape": (ValueError, lambda P, c: P.embedding_backward(c(4, 4), c(3, dtype=I64), 5)),
    "gradient of no table": (ValueError, lambda P, c: P.embedding_backward(c(3, 4), c(3, dtype=I64), 0)),
    "no scale": (TypeError, lambda P, c: P.embedding(c(3, dtype=I64), c(5, 4), None)),
    "norm type": (TypeError, lambda P, c: P.layer_norm(c(3, 4, dtype=torch.float64))),
    "norm weight type": (TypeError, lambda P, c: P.layer_norm(c(3, 4), c(4, dtype=BF16))),
    "norm weight and bias": (TypeError, lambda P, c: P.layer_norm(c(3, 4, dtype=BF16), c(4, dtype=BF16), c(4))),
    "norm weight shape": (ValueError, lambda P, c: P.layer_norm(c(3, 4), c(3))),
    "norm bias shape": (ValueError, lambda P, c: P.layer_norm(c(3, 4), None, c(1, 4))),
    "norm weight device": (ValueError, lambda P, c: P.layer_norm(c(3, 4), c(4, dev=1))),
    "norm eps": (ValueError, lambda P, c: P.layer_norm(c(3, 4), eps=-1.0)),
    "norm residual shape": (ValueError, lambda P, c: P.layer_norm(c(3, 4), residual=c(4))),
    "norm residual type": (TypeError, lambda P, c: P.layer_norm(c(3, 4), residual=c(3, 4, dtype=BF16))),
    "norm without features": (ValueError, lambda P, c: P.layer_norm(c(3, 0))),
    "norm statistics": (ValueError, lambda P, c: P.layer_norm_backward(c(3, 4), c(3, 4), c(4), None, c(2), c(3))),
    "norm statistics type": (TypeError, lambda P, c: P.layer_norm_backward(c(3, 4), c(3, 4), c(4), None, c(3, dtype=BF16), c(3))),
    "norm gradient": (ValueError, lambda P, c: P.layer_norm_backward(c(3, 5), c(3, 4), c(4), None, c(3), c(3))),
    "norm gradient of the sum": (ValueError, lambda P, c: P.layer_norm_backward(c(3, 4), c(3, 4), c(4), None, c(3), c(3), c(12))),
    "muon grads missing": (ValueError, lambda P, c: P.muon_step([c(4, 4)], [], [c(4, 4)], 0.1)),
    "muon vector": (ValueError, lambda P, c: P.muon_step([c(4)], [c(4)], [c(4)], 0.1)),
    "muon grad shape": (ValueError, lambda P, c: P.muon_step([c(4, 2)], [c(2, 4)], [c(4, 2)], 0.1)),
    "muon momentum type": (TypeError, lambda P, c: P.muon_step([c(4, 2, dtype=BF16)], [c(4, 2, dtype=BF16)], [c(4, 2, dtype=BF16)], 0.1)),
    "muon param type": (TypeError, lambda P, c: P.muon_step([c(4, 2, dtype=torch.float64)], [c(4, 2)], [c(4, 2)], 0.1)),
    "muon grad type": (TypeError, lambda P, c: P.muon_step([c(4, 2)], [c(4, 2, dtype=BF16)], [c(4, 2)], 0.1)),
    "muon strided": (ValueError, lambda P, c: P.muon_step([c(4, 2).t()], [c(2, 4)], [c(2, 4)], 0.1)),
    "muon device": (ValueError, lambda P, c: P.muon_step([c(4, 2)], [c(4, 2, dev=1)], [c(4, 2)], 0.1)),
    "muon master": (ValueError, lambda P, c: P.muon_step([c(4, 2)], [c(4, 2)], [c(4, 2)], 0.1, master=[c(4, 2)])),
    "muon lr": (TypeError, lambda P, c: P.muon_step([c(4, 2)], [c(4, 2)], [c(4, 2)], c(2))),
    "muon lr device": (ValueError, lambda P, c: P.muon_step([c(4, 2)], [c(4, 2)], [c(4, 2)], c(1, dev=1))),
    "muon adjust": (ValueError, lambda P, c: P.muon_step([c(4, 2)], [c(4, 2)], [c(4, 2)], 0.1, adjust="other")),
    "muon coefficients": (ValueError, lambda P, c: P.muon_step([c(4, 2)], [c(4, 2)], [c(4, 2)], 0.1, coefficients=(1.0, 2.0))),
    "muon triples": (ValueError, lambda P, c: P.muon_step([c(4, 2)], [c(4, 2)], [c(4, 2)], 0.1, coefficients=((1.0, 2.0, 3.0), (1.0, 2.0)))),
    "muon not a list": (TypeError, lambda P, c: P.muon_step(c(4, 2), [c(4, 2)], [c(4, 2)], 0.1)),
    "orthogonalise a vector": (ValueError, lambda P, c: P.orthogonalise(c(4))),
    "orthogonalise type": (TypeError, lambda P, c: P.orthogonalise(c(4, 4, dtype=torch.float64))),
    "orthogonalise coefficients": (ValueError, lambda P, c: P.orthogonalise(c(4, 4), ())),
}


@pytest.mark.parametrize("what", CALLS)
def test_refused(fake, what):
    import paralleltnnlayers_b200 as P
    error, call = CALLS[what]
    with pytest.raises(error):
        call(P, fake)


class Hyper(C.Structure):
    _fields_ = [(k, C.c_double) for k in ("lr", "momentum", "wd", "eps")] + [(k, C.c_int) for k in ("nesterov", "steps", "adjust", "count")] + \
        [("coefficients", C.POINTER(C.c_double)), ("device_lr", C.c_void_p)]


class Matrix(C.Structure):
    _fields_ = [(k, C.c_void_p) for k in ("param", "grad", "momentum", "master")] + [(k, C.c_int) for k in ("stack", "rows", "cols")]


def test_the_library_refuses(lib_built):
    from paralleltnnlayers_b200 import _lib
    lib = _lib.lib
    invalid, unsupported = -1, -2
    abc = (C.c_double * 3)(3.4445, -4.7750, 2.0315)

    def step(matrices=(), types=(0, 0), **k):
        v = dict(lr=0.1, momentum=0.9, wd=0.0, eps=1e-7, nesterov=1, steps=5, adjust=1, count=1, coefficients=abc)
        v.update(k)
        ms = (Matrix * max(1, len(matrices)))(*[Matrix(*m) for m in matrices])
        return lib.b200cp_muon_step(ms, len(matrices), *types, C.byref(Hyper(**v)), None, 0, None)
    assert step() == 0   # nothing to do
    assert step(matrices=[(0, 0, 0, 0, 0, 5, 5)]) == 0
    for bad in (dict(momentum=-0.1), dict(momentum=1.5), dict(eps=0.0), dict(eps=float("nan")), dict(steps=-1), dict(steps=101), dict(count=2), dict(adjust=3),
                dict(coefficients=None), dict(matrices=[(0, 0, 0, 0, 1, 5, 5)]), dict(matrices=[(0, 0, 0, 0, 1, -5, 5)])):
        assert step(**bad) == invalid, bad
    assert step(types=(0, 1)) == unsupported
    assert step(coefficients=(C.c_double * 3)(20.0, 30.0, 40.0)) == unsupported
    assert step(matrices=[(0, 0, 0, 0, 1, 1 << 18, 1 << 18)]) == unsupported
    # addresses are looked at by no kernel: every call is refused before
    at = 4096
    assert lib.b200cp_embedding(3, 0, 4, 0, 0, at, at, 1.0, at, None) == invalid
    assert lib.b200cp_embedding(3, 5, 4, 7, 0, at, at, 1.0, at, None) == invalid
    assert lib.b200cp_embedding(3, 5, 4, 0, 2, at, at, 1.0, at, None) == invalid
    assert lib.b200cp_embedding(3, 5, 4, 0, 0, None, at, 1.0, at, None) == invalid
    assert lib.b200cp_embedding(0, 5, 4, 0, 0, None, None, 1.0, None, None) == 0
    assert lib.b200cp_embedding_bwd(3, 5, 4, 0, 0, at, at, 1.0, None, None, 0, None) == invalid
    assert lib.b200cp_embedding_bwd(3, 5, 4, 0, 0, None, at, 1.0, at, None, 0, None) == invalid
    assert lib.b200cp_embedding_bwd(-1, 5, 4, 0, 0, at, at, 1.0, at, None, 0, None) == invalid
    assert lib.b200cp_layer_norm(3, 4, 0, 1, at, None, at, None, 1e-5, at, None, None, None, None) == unsupported
    assert lib.b200cp_layer_norm(3, 4, 0, 0, at, at, at, None, 1e-5, at, None, None, None, None) == invalid   # a residual without a place for the sum
    assert lib.b200cp_layer_norm(3, 4, 0, 0, at, None, at, None, -1.0, at, None, None, None, None) == invalid
    assert lib.b200cp_layer_norm(3, 4, 0, 0, at, None, at, None, 1e-5, at, None, at, None, None) == invalid
    assert lib.b200cp_layer_norm(0, 4, 0, 0, None, None, None, None, 1e-5, None, None, None, None, None) == 0
    assert lib.b200cp_layer_norm_bwd(3, 4, 0, 0, at, None, None, at, at, at, at, None, None, None, 0, None) == invalid
    assert lib.b200cp_layer_norm_bwd(3, 0, 0, 0, at, None, at, at, at, at, at, None, None, None, 0, None) == invalid


def test_layers_and_optimiser_on_the_host():
    from paralleltnnlayers_b200.layers import Embedding, LayerNorm
    from paralleltnnlayers_b200.optim import Muon
    e, n = Embedding(7, 4, scale=2.0, dtype=BF16), LayerNorm(4, bias=False)
    assert e.W.shape == (7, 4) and e.W.dtype == BF16 and n.bias is None and n.weight.dtype == torch.float32
    assert LayerNorm(4, affine=False).weight is None
    for bad in (lambda: Embedding(0, 4), lambda: Embedding(4, 4, dtype=torch.float64), lambda: LayerNorm(0), lambda: LayerNorm(4, eps=-1.0)):
        with pytest.raises(ValueError):
            bad()
    p = [torch.nn.Parameter(torch.zeros(3, 2))]
    for bad in (dict(lr=-1.0), dict(momentum=1.5), dict(eps=0.0), dict(weight_decay=-1.0), dict(ns_steps=101), dict(adjust_lr_fn="other")):
        with pytest.raises(ValueError):
            Muon(p, **bad)
    with pytest.raises(ValueError, match="matrices"):
        Muon([torch.nn.Parameter(torch.zeros(3))])
    q = [torch.nn.Parameter(torch.zeros(3, 2, dtype=BF16))]
    opt = Muon(q)
    opt.state[q[0]] = {"momentum_buffer": torch.ones(3, 2), "master": torch.full((3, 2), 0.1)}
    other = Muon([torch.nn.Parameter(torch.zeros(3, 2, dtype=BF16))])
    other.load_state_dict(opt.state_dict())
    s = next(iter(other.state.values()))
    assert s["momentum_buffer"].dtype == torch.float32 and torch.equal(s["master"], torch.full((3, 2), 0.1))


def test_the_optimiser_calls_the_step(monkeypatch, lib_built):
    """A call per type; parameters without a gradient are left out."""
    from paralleltnnlayers_b200 import ops
    from paralleltnnlayers_b200.optim import Muon
    calls = []
    monkeypatch.setattr(ops, "muon_step", lambda *a: calls.append(a))
    p = [torch.nn.Parameter(torch.zeros(3, 2)), torch.nn.Parameter(torch.zeros(2, 2, dtype=BF16)), torch.nn.Parameter(torch.zeros(5, 2)), torch.nn.Parameter(torch.zeros(4, 2))]
    for t in (p[0], p[1], p[3]):
        t.grad = torch.ones_like(t)
    opt = Muon(p, lr=0.5, momentum=0.8, adjust_lr_fn="match_rms_adamw")
    opt.step()
    opt.step()
    assert [len(c[0]) for c in calls] == [2, 1, 2, 1]
    assert calls[0][3:11] == (0.5, 0.8, True, 0.1, (3.4445, -4.7750, 2.0315), 1e-7, 5, "match_rms_adamw") and calls[0][11] is None
    assert calls[1][11][0].dtype == torch.float32 and calls[1][2][0].dtype == torch.float32
    assert calls[1][11][0] is calls[3][11][0] and p[2] not in opt.state


def test_the_state_of_torchs_muon_is_loaded(monkeypatch, lib_built):
    """Buffers of the parameter's type become float32, float32 copies are taken at the first step, and groups without ``master`` have them."""
    from paralleltnnlayers_b200 import ops
    from paralleltnnlayers_b200.optim import Muon
    p = [torch.nn.Parameter(torch.full((3, 2), 0.5, dtype=BF16)), torch.nn.Parameter(torch.full((2, 4), 0.25))]
    theirs = torch.optim.Muon(p, lr=0.3, momentum=0.8, ns_steps=4)
    theirs.state[p[0]] = {"momentum_buffer": torch.full((3, 2), 1.5, dtype=BF16)}
    theirs.state[p[1]] = {"momentum_buffer": torch.full((2, 4), 2.5)}
    opt = Muon(p)
    opt.load_state_dict(theirs.state_dict())
    calls = []
    monkeypatch.setattr(ops, "muon_step", lambda *a: calls.append(a))
    for t in p:
        t.grad = torch.ones_like(t)
    opt.step()
    assert len(calls) == 2 and all(c[3:5] == (0.3, 0.8) and c[9] == 4 for c in calls)
    assert torch.equal(calls[0][2][0], torch.full((3, 2), 1.5)) and torch.equal(calls[1][2][0], torch.full((2, 4), 2.5))
    assert torch.equal(calls[0][11][0], torch.full((3, 2), 0.5)) and calls[1][11] is None


def test_too_many_rows_are_refused(lib_built):
    from paralleltnnlayers_b200 import _lib
    lib, at, rows = _lib.lib, 4096, (1 << 31) - 1
    assert lib.b200cp_layer_norm(rows, 4, 0, 0, at, None, at, None, 1e-5, at, None, None, None, None) == -2
    assert lib.b200cp_layer_norm_bwd(rows, 4, 0, 0, at, None, at, at, at, at, at, None, None, None, 0, None) == -2
    assert lib.b200cp_embedding(rows, 5, 4, 0, 0, at, at, 1.0, at, None) == -2
    assert lib.b200cp_embedding_bwd(rows, 5, 4, 0, 0, at, at, 1.0, at, None, 0, None) == -2
