"""What the operators beside the factored layers refuse, before anything is launched."""
import pytest
import torch


@pytest.fixture
def fake(lib_built):
    """Fake CUDA tensors: nothing can be launched."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        yield lambda *size, dev=0, dtype=torch.float32: torch.empty(*size, device=f"cuda:{dev}", dtype=dtype)


ADAMW = {
    "grads missing": (ValueError, lambda c: ([c(4)], [], [c(4)], [c(4)], 1, 0.1)),
    "grad size": (ValueError, lambda c: ([c(4)], [c(5)], [c(4)], [c(4)], 1, 0.1)),
    "grad device": (ValueError, lambda c: ([c(4)], [c(4, dev=1)], [c(4)], [c(4)], 1, 0.1)),
    "moment type": (TypeError, lambda c: ([c(4)], [c(4)], [c(4, dtype=torch.bfloat16)], [c(4)], 1, 0.1)),
    "param type": (TypeError, lambda c: ([c(4, dtype=torch.float64)], [c(4)], [c(4)], [c(4)], 1, 0.1)),
    "two param types": (TypeError, lambda c: ([c(4), c(4, dtype=torch.float16)], [c(4), c(4)], [c(4), c(4)], [c(4), c(4)], 1, 0.1)),
    "grad type": (TypeError, lambda c: ([c(4)], [c(4, dtype=torch.bfloat16)], [c(4)], [c(4)], 1, 0.1)),
    "strided param": (ValueError, lambda c: ([c(4, 2)[:, 0]], [c(4)], [c(4)], [c(4)], 1, 0.1)),
    "step tensor": (TypeError, lambda c: ([c(4)], [c(4)], [c(4)], [c(4)], c(1), 0.1)),
    "step device": (ValueError, lambda c: ([c(4)], [c(4)], [c(4)], [c(4)], c(1, dev=1, dtype=torch.int64), 0.1)),
    "lr tensor": (TypeError, lambda c: ([c(4)], [c(4)], [c(4)], [c(4)], 1, c(2))),
    "not a list": (TypeError, lambda c: (3, [c(4)], [c(4)], [c(4)], 1, 0.1)),
    "not tensors": (TypeError, lambda c: ([3], [c(4)], [c(4)], [c(4)], 1, 0.1)),
}


@pytest.mark.parametrize("what", ADAMW)
def test_adamw_refuses(fake, what):
    import paralleltnnlayers_b200 as P
    error, args = ADAMW[what]
    with pytest.raises(error):
        P.adamw_step(*args(fake))


def test_adamw_refuses_scales_and_copies_that_do_not_fit(fake):
    import paralleltnnlayers_b200 as P
    c, i8, u8 = fake, torch.int8, torch.uint8
    with pytest.raises(ValueError, match="values where 2 are needed"):
        P.adamw_step([c(257)], [c(257)], [c(257, dtype=i8)], [c(257, dtype=u8)], 1, 0.1, scales=([c(1)], [c(2)]))
    with pytest.raises(ValueError, match="16-bit parameters"):
        P.adamw_step([c(4)], [c(4)], [c(4)], [c(4)], 1, 0.1, master=[c(4)])
    with pytest.raises(ValueError):
        P.adamw_moments(c(257, dtype=i8), c(257, dtype=u8), (c(2), c(1)))


def test_adamw_refuses_rates_out_of_range(lib_built):
    import ctypes as C

    from paralleltnnlayers_b200 import _lib
    from paralleltnnlayers_b200.optim import AdamW

    class H(C.Structure):
        _fields_ = [(k, C.c_double) for k in ("lr", "b1", "b2", "eps", "wd")] + [("step", C.c_longlong), ("t", C.c_void_p), ("d", C.c_void_p)]

    call = lambda bits=32, **k: _lib.lib.b200cp_adamw_step(None, 0, 0, 0, bits, C.byref(H(**{**dict(lr=1, b1=0.9, b2=0.9, step=1), **k})), None)  # noqa: E731
    assert call() == 0   # nothing to do
    for bad in (dict(b1=1.0), dict(b2=-0.1), dict(b1=float("nan")), dict(eps=-1), dict(step=0), dict(bits=16)):
        assert call(**bad) == -1
    p = [torch.nn.Parameter(torch.zeros(3))]
    for bad in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(bits=4), dict(eps=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            AdamW(p, **bad)
