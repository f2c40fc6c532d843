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


ADAPTERS = {
    "x type": (TypeError, lambda c: (c(2, 4), c(2, 8, dtype=torch.float64), c(3, 8, 2), c(3, 2, 4), c(2, dtype=torch.int32))),
    "y type": (TypeError, lambda c: (c(2, 4), c(2, 8, dtype=torch.float16), c(3, 8, 2, dtype=torch.float16), c(3, 2, 4, dtype=torch.float16), c(2, dtype=torch.int32))),
    "A type": (TypeError, lambda c: (c(2, 4), c(2, 8), c(3, 8, 2, dtype=torch.bfloat16), c(3, 2, 4), c(2, dtype=torch.int32))),
    "A features": (ValueError, lambda c: (c(2, 4), c(2, 8), c(3, 7, 2), c(3, 2, 4), c(2, dtype=torch.int32))),
    "rank": (ValueError, lambda c: (c(2, 4), c(2, 8), c(3, 8, 2), c(3, 3, 4), c(2, dtype=torch.int32))),
    "count": (ValueError, lambda c: (c(2, 4), c(2, 8), c(3, 8, 2), c(4, 2, 4), c(2, dtype=torch.int32))),
    "y features": (ValueError, lambda c: (c(2, 5), c(2, 8), c(3, 8, 2), c(3, 2, 4), c(2, dtype=torch.int32))),
    "y rows": (ValueError, lambda c: (c(3, 4), c(2, 8), c(3, 8, 2), c(3, 2, 4), c(2, dtype=torch.int32))),
    "numbers": (ValueError, lambda c: (c(2, 4), c(2, 8), c(3, 8, 2), c(3, 2, 4), c(3, dtype=torch.int32))),
    "numbers type": (TypeError, lambda c: (c(2, 4), c(2, 8), c(3, 8, 2), c(3, 2, 4), c(2))),
    "numbers device": (ValueError, lambda c: (c(2, 4), c(2, 8), c(3, 8, 2), c(3, 2, 4), c(2, dtype=torch.int32, dev=1))),
    "B device": (ValueError, lambda c: (c(2, 4), c(2, 8), c(3, 8, 2), c(3, 2, 4, dev=1), c(2, dtype=torch.int32))),
    "scale size": (ValueError, lambda c: (c(2, 4), c(2, 8), c(3, 8, 2), c(3, 2, 4), c(2, dtype=torch.int32), c(2))),
    "scale type": (TypeError, lambda c: (c(2, 4), c(2, 8), c(3, 8, 2), c(3, 2, 4), c(2, dtype=torch.int32), c(3, dtype=torch.float16))),
    "empty": (ValueError, lambda c: (c(2, 4), c(2, 8), c(0, 8, 2), c(0, 2, 4), c(2, dtype=torch.int32))),
    "not a tensor": (TypeError, lambda c: (c(2, 4), None, c(3, 8, 2), c(3, 2, 4), c(2, dtype=torch.int32))),
}


@pytest.mark.parametrize("what", ADAPTERS)
def test_adapters_refuse(fake, what):
    import paralleltnnlayers_b200 as P
    error, args = ADAPTERS[what]
    with pytest.raises(error):
        P.dense_adapters(*args(fake))
    with pytest.raises(error):
        P.DenseAdaptersFunction.apply(*args(fake))


def test_adapters_refuse_an_out_that_does_not_fit(fake):
    import paralleltnnlayers_b200 as P
    args = (fake(2, 4), fake(2, 4), fake(3, 4, 2), fake(3, 2, 4), fake(2, dtype=torch.int32))
    for out in (fake(3, 4), fake(2, 4, dtype=torch.float16), fake(2, 4, dev=1)):
        with pytest.raises((TypeError, ValueError)):
            P.dense_adapters(*args, out=out)


def test_adapter_sizes_the_library_refuses(lib_built):
    from paralleltnnlayers_b200 import _lib
    lib = _lib.lib
    assert lib.b200cp_adapter_plan_bytes(4, 0) == 0 and lib.b200cp_adapter_plan_bytes(4, 16385) == 0 and lib.b200cp_adapter_plan_bytes(-1, 3) == 0
    assert lib.b200cp_adapter_plan_bytes(0, 1) > 0
    assert lib.b200cp_adapter_plan(4, 3, None, None, 0, None) == -1
    assert lib.b200cp_adapter_plan(4, 3, 16, 16, 8, None) == -3        # too small a plan
    assert lib.b200cp_adapter_plan(4, 3, 16, 24, 1 << 20, None) == -3  # not on sixteen bytes
    fwd = lambda *a, by=(16, None): lib.b200cp_dense_adapters(*a, *[16] * 4, None, *by, 16, None, None)  # noqa: E731
    assert fwd(0, 4, 4, 4, 1, 0) == 0
    assert fwd(4, 4, 4, 129, 1, 0) == -2 and fwd(4, 4, 4, 4, 16385, 0) == -2
    assert fwd(4, 0, 4, 4, 1, 0) == -1 and fwd(4, 4, 4, 4, 1, 3) == -1 and fwd(-1, 4, 4, 4, 1, 0) == -1
    assert fwd(257, 4, 4, 4, 1, 0) == -2 and fwd(4, 4, 4, 4, 1, 0, by=(None, None)) == -1   # too many rows without a plan; neither
    assert lib.b200cp_dense_adapters(4, 4, 4, 4, 1, 0, *[None] * 10) == -1
    assert lib.b200cp_dense_adapters_bwd(4, 4, 4, 4, 1, 0, *[16] * 5, None, 16, 16, 16, 16, 16, 4, None) == -3
    assert lib.b200cp_dense_adapters_bwd(4, 4, 4, 4, 1, 0, *[None] * 5, None, 16, 16, 16, 16, 16, 1 << 20, None) == -1


B16 = torch.bfloat16
GATED = {
    "x type": (TypeError, lambda c: (c(2, 8), c(8, 4), c(8, 4))),
    "Wg type": (TypeError, lambda c: (c(2, 8, dtype=B16), c(8, 4, dtype=torch.float16), c(8, 4, dtype=B16))),
    "Wu type": (TypeError, lambda c: (c(2, 8, dtype=B16), c(8, 4, dtype=B16), c(8, 4))),
    "Wu size": (ValueError, lambda c: (c(2, 8, dtype=B16), c(8, 4, dtype=B16), c(8, 5, dtype=B16))),
    "features": (ValueError, lambda c: (c(2, 7, dtype=B16), c(8, 4, dtype=B16), c(8, 4, dtype=B16))),
    "device": (ValueError, lambda c: (c(2, 8, dtype=B16), c(8, 4, dtype=B16), c(8, 4, dtype=B16, dev=1))),
    "dimensions": (ValueError, lambda c: (c(2, 8, dtype=B16), c(1, 8, 4, dtype=B16), c(1, 8, 4, dtype=B16))),
    "empty": (ValueError, lambda c: (c(2, 8, dtype=B16), c(8, 0, dtype=B16), c(8, 0, dtype=B16))),
    "not a tensor": (TypeError, lambda c: (c(2, 8, dtype=B16), None, c(8, 4, dtype=B16))),
    "activation": (ValueError, lambda c: (c(2, 8, dtype=B16), c(8, 4, dtype=B16), c(8, 4, dtype=B16), "relu")),
}


@pytest.mark.parametrize("what", GATED)
def test_gated_refuses(fake, what):
    import paralleltnnlayers_b200 as P
    error, args = GATED[what]
    for call in (P.dense_gated, P.dense_gated_save, P.DenseGatedFunction.apply):
        with pytest.raises(error):
            call(*args(fake))


def test_gated_backward_refuses_what_does_not_fit(fake):
    import paralleltnnlayers_b200 as P
    c = fake
    good = dict(dH=c(2, 4, dtype=B16), X=c(2, 8, dtype=B16), Wg=c(8, 4, dtype=B16), Wu=c(8, 4, dtype=B16), G=c(2, 4), U=c(2, 4))
    for name, bad, error in (("dH", c(2, 5, dtype=B16), ValueError), ("dH", c(2, 4), TypeError), ("G", c(2, 5), ValueError), ("U", c(2, 4, dtype=B16), TypeError),
                             ("U", c(2, 4, dev=1), ValueError)):
        with pytest.raises(error):
            P.dense_gated_backward(**{**good, name: bad})


def test_gated_sizes_the_library_refuses(lib_built):
    from paralleltnnlayers_b200 import _lib
    lib = _lib.lib
    assert lib.b200cp_dense_gated_workspace_bytes(4, 8, 8, 1) == 0 and lib.b200cp_dense_gated_workspace_bytes(4, 8, 9, 1) > 0
    assert lib.b200cp_dense_gated_workspace_bytes(4, 8, 9, 0) == 0
    fwd = lambda *a: lib.b200cp_dense_gated(*a, None, 0, None)  # noqa: E731
    assert fwd(0, 8, 8, 1, 0, None, None, None, None, None, None) == 0
    assert fwd(4, 8, 8, 0, 0, 16, 16, 16, 16, None, None) == -2      # fp32
    assert fwd(4, 8, 8, 1, 3, 16, 16, 16, 16, None, None) == -1      # no such activation
    assert fwd(4, 8, 8, 1, 0, 16, 16, 16, 16, 16, None) == -1        # G without U
    assert fwd(4, 8, 8, 1, 0, 16, 24, 16, 16, None, None) == -1      # not on sixteen bytes
    assert fwd(4, 8, 9, 1, 0, 16, 16, 16, 16, None, None) == -3      # no workspace
    bwd = lambda *a: lib.b200cp_dense_gated_bwd(*a, None, 0, None)  # noqa: E731
    assert bwd(4, 8, 8, 1, 0, 16, 16, 16, 16, 16, 16, 16, 16, None) == -1
    assert bwd(4, 8, 8, 1, 0, 16, 16, 16, 16, 16, 16, 16, 16, 16) == -3
