"""A plan is one of its rows and its number of adapters, also where the plan of another number has the same size."""
import ctypes as C

import pytest
import torch

SAME_SIZE = [(1, 1, 2), (1, 3, 2), (64, 31, 32), (100, 3, 4), (100, 4, 3), (300, 4, 3), (4096, 7, 8)]   # rows, adapters of the plan and of the factors


def test_the_sizes_are_the_same(lib_built):
    from paralleltnnlayers_b200 import _lib
    for rows, a, b in SAME_SIZE:
        assert _lib.lib.b200cp_adapter_plan_bytes(rows, a) == _lib.lib.b200cp_adapter_plan_bytes(rows, b)


@pytest.mark.parametrize("rows,planned,count", SAME_SIZE)
def test_a_plan_of_another_count_is_refused(lib_built, rows, planned, count):
    """Fake CUDA tensors: nothing can be launched."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    import paralleltnnlayers_b200 as P
    from paralleltnnlayers_b200 import _lib
    with FakeTensorMode():
        c = lambda *s, dtype=torch.float32: torch.empty(*s, device="cuda:0", dtype=dtype)  # noqa: E731
        plan = object.__new__(P.AdapterPlan)
        plan.data, plan.shape, plan.count = c(_lib.lib.b200cp_adapter_plan_bytes(rows, planned), dtype=torch.uint8), (rows,), planned
        y, x, A, B, V = c(rows, 8), c(rows, 16), c(count, 16, 4), c(count, 4, 8), c(rows, 4)
        match = f"one of {planned} adapters, A and B are of {count}"
        with pytest.raises(ValueError, match=match):
            P.dense_adapters(y, x, A, B, plan)
        with pytest.raises(ValueError, match=match):
            P.DenseAdaptersFunction.apply(y, x, A, B, plan)
        with pytest.raises(ValueError, match=match):
            P.dense_adapters_backward(y, x, V, A, B, plan)


def test_a_plan_off_sixteen_bytes_is_refused_by_the_library(lib_built):
    from paralleltnnlayers_b200 import _lib
    lib = _lib.lib
    assert lib.b200cp_dense_adapters(4, 4, 4, 4, 1, 0, *[16] * 4, None, None, 24, 16, None, None) == -1
    assert lib.b200cp_dense_adapters_bwd(4, 4, 4, 4, 1, 0, *[16] * 5, None, 24, 16, 16, 16, 16, 1 << 20, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("rows,planned,count", SAME_SIZE)
def test_the_library_computes_nothing_from_a_plan_of_another_count(rows, planned, count):
    """Through the C entry points, which have the plan's address alone: the kernels compare what it says of itself."""
    import paralleltnnlayers_b200 as P
    from paralleltnnlayers_b200 import _lib
    lib, I, O, R = _lib.lib, 16, 8, 4
    gen = torch.Generator(device="cuda").manual_seed(rows)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    which = torch.randint(0, min(planned, count), (rows,), generator=gen, device="cuda", dtype=torch.int32)
    y, x, A, B, V = n(rows, O), n(rows, I), n(count, I, R), n(count, R, O), n(rows, R)
    ws = torch.empty(lib.b200cp_dense_adapters_bwd_workspace_bytes(rows, I, O, R, count, 0), dtype=torch.uint8, device="cuda")
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)

    def run(plan):
        outs = [torch.full_like(t, 7.0) for t in (y, x, A, B)]
        out, dx, dA, dB = outs
        assert lib.b200cp_dense_adapters(rows, I, O, R, count, 0, p(y), p(x), p(A), p(B), None, None, p(plan), p(out), None, st) == 0
        assert lib.b200cp_dense_adapters_bwd(rows, I, O, R, count, 0, p(y), p(x), p(V), p(A), p(B), None, p(plan), p(dx), p(dA), p(dB), p(ws),
                                             ws.numel(), st) == 0
        return outs

    P.device_status()
    for plan in (P.adapter_plan(which, planned), P.adapter_plan(which[:rows - 1].contiguous(), count)):   # another count, other rows
        outs = run(plan.data)
        with pytest.raises(_lib.B200CPError, match="a plan of other rows"):
            P.device_status()
        P.device_status()   # the record is cleared
        assert all(bool((t == 7).all()) for t in outs)
    outs = run(P.adapter_plan(which, count).data)
    P.device_status()
    assert all(not bool((t == 7).any()) for t in outs)


@pytest.mark.gpu
def test_an_output_over_the_numbers_the_plan_or_the_scales_is_refused():
    """CTAs that are done would write what others still read."""
    import paralleltnnlayers_b200 as P
    rows, I, O, R, count = 32, 16, 8, 4, 8
    n = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    y, x, A, B, scale = n(rows, O), n(rows, I), n(count, I, R), n(count, R, O), torch.ones(count, device="cuda")
    which = torch.zeros(rows, dtype=torch.int32, device="cuda")
    buf = torch.zeros(rows * O, device="cuda")
    over = lambda t: buf[100:100 + t.numel()].view(t.dtype).copy_(t)  # noqa: E731
    plan = P.adapter_plan(which, count)
    size = plan.data.numel() // 4
    room = torch.zeros(rows * O + size, device="cuda")
    plan.data = room[16:16 + size].view(torch.uint8).copy_(plan.data)
    with pytest.raises(ValueError, match="share memory"):
        P.dense_adapters(y, x, A, B, over(which), scale, out=buf.view(rows, O))
    with pytest.raises(ValueError, match="share memory"):
        P.dense_adapters(y, x, A, B, which, over(scale), out=buf.view(rows, O))
    with pytest.raises(ValueError, match="share memory"):
        P.dense_adapters(y, x, A, B, plan, scale, out=room[:rows * O].view(rows, O))
    out = P.dense_adapters(y, x, A, B, which, scale, out=buf.view(rows, O))
    assert torch.equal(out, P.dense_adapters(y, x, A, B, which, scale))
