"""Low-rank adapters beside a shared projection against the definition in 64 bits.

Bounds, for each entry.  e = finfo(type).eps / 2 is a rounding to the type, u = 2**-23 an addition of the tensor core (which may cut its sum off: a whole
unit of fp32; FFMA half of that).  V = c X A is a sum of I products: (I + 2) u |c| |X| |A|, and is rounded once, e |V|.  out = Y + V B: those errors times |B|,
(R + 2) u |V| |B| of its own sum, one rounding e |out|.  The gradients are the same with their own lengths; sums over an adapter's rows have at most `rows`
terms.  (float32: the roundings to the type are fp32's own.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _p():
    import paralleltnnlayers_b200 as P
    return P


def inputs(rows, I, O, R, count, dtype, which, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s, std=1.0: (torch.randn(*s, generator=gen, device="cuda") * std).to(dtype)  # noqa: E731
    if which == "each":
        a = torch.randint(-1, count, (rows,), generator=gen, device="cuda")
    elif which == "runs":
        a = torch.arange(rows, device="cuda") * count // max(rows, 1)
    elif which == "one":
        a = torch.full((rows,), count - 1, device="cuda")
    elif which == "none":
        a = torch.full((rows,), -1, device="cuda")
    else:   # numbers far out of the range: no adapter
        a = torch.randint(-2, count + 2, (rows,), generator=gen, device="cuda")
        a[::3] = 2 ** 31 - 1
        a[1::7] = -2 ** 31
    return {"x": n(rows, I), "y": n(rows, O), "A": n(count, I, R, std=I ** -0.5), "B": n(count, R, O, std=R ** -0.5), "dy": n(rows, O),
            "which": a.to(torch.int32), "scale": torch.rand(count, generator=gen, device="cuda") * 2 - 0.5}


def definition(t, scale=True):
    """Results and bounds of the forward and of the gradients."""
    d = {k: v.double() for k, v in t.items() if k != "which"}
    rows, I = t["x"].shape
    count, R, O = t["B"].shape
    e = torch.finfo(t["x"].dtype).eps / 2
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device="cuda")  # noqa: E731
    out, bout, dx, bdx, V = d["y"].clone(), z(rows, O), z(rows, I), z(rows, I), z(rows, R)
    dA, bdA, dB, bdB = z(count, I, R), z(count, I, R), z(count, R, O), z(count, R, O)
    for a in range(count):
        s = (t["which"] == a).nonzero().view(-1)
        if not len(s):
            continue
        c = d["scale"][a] if scale else torch.ones((), dtype=torch.float64, device="cuda")
        x, dy, A, B = d["x"][s], d["dy"][s], d["A"][a], d["B"][a]
        v, w = c * x @ A, c * dy @ B.t()
        ev = (I + 2) * U * abs(c) * x.abs() @ A.abs() + e * v.abs()
        ew = (O + 2) * U * abs(c) * dy.abs() @ B.abs().t() + e * w.abs()
        V[s] = v
        out[s] = d["y"][s] + v @ B
        bout[s] = ev @ B.abs() + (R + 2) * U * v.abs() @ B.abs() + (e + U) * (out[s].abs() + U * d["y"][s].abs())
        dx[s] = w @ A.t()
        bdx[s] = ew @ A.abs().t() + (R + 2) * U * w.abs() @ A.abs().t() + e * dx[s].abs()
        n = len(s) + 2
        dA[a], dB[a] = x.t() @ w, v.t() @ dy
        bdA[a] = x.abs().t() @ ew + n * U * x.abs().t() @ w.abs() + e * dA[a].abs()
        bdB[a] = ev.t() @ dy.abs() + n * U * v.abs().t() @ dy.abs() + e * dB[a].abs()
    # below the smallest normal number a rounding is off by half of the smallest one
    tiny = torch.finfo(t["x"].dtype).smallest_normal * e * 2
    return {"out": (out, bout + tiny), "dx": (dx, bdx + tiny), "dA": (dA, bdA + tiny), "dB": (dB, bdB + tiny)}, V


def near(got, want, what):
    ref, bound = want
    assert got.shape == ref.shape and bool(torch.isfinite(got).all()), what
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), f"{what}: worst {float((err / bound).nan_to_num().max()):.3f} of the bound"


def check(t, scale=True):
    P = _p()
    want, _ = definition(t, scale)
    c = t["scale"] if scale else None
    near(P.dense_adapters(t["y"], t["x"], t["A"], t["B"], t["which"], c), want["out"], "forward")
    leaves = [t[k].clone().requires_grad_() for k in ("y", "x", "A", "B")]
    out = P.DenseAdaptersFunction.apply(*leaves, t["which"], c)
    near(out.detach(), want["out"], "forward under autograd")
    dy, dx, dA, dB = torch.autograd.grad(out, leaves, t["dy"])
    assert torch.equal(dy, t["dy"])
    near(dx, want["dx"], "dX")
    near(dA, want["dA"], "dA")
    near(dB, want["dB"], "dB")


CASES = [(1, 64, 64, 16, 1, "one"), (1, 8, 8, 1, 3, "one"), (3, 1, 1, 1, 2, "each"), (5, 130, 257, 7, 4, "each"), (64, 512, 384, 16, 32, "each"),
         (200, 1000, 72, 64, 3, "runs"), (333, 96, 1033, 33, 5, "each"), (257, 264, 520, 128, 2, "runs"), (700, 256, 128, 8, 1, "one"),
         (1000, 136, 264, 24, 7, "far"), (40, 64, 64, 16, 5, "none"), (129, 2048, 2056, 16, 2, "runs"), (1500, 72, 40, 16, 300, "each"),
         (2100, 1024, 1024, 32, 6, "runs")]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_forward_and_gradients(case, dtype):
    rows, I, O, R, count, which = case
    check(inputs(rows, I, O, R, count, dtype, which, seed=rows))


def test_without_scales():
    check(inputs(70, 96, 64, 16, 4, BF16, "each"), scale=False)


def test_gradients_against_differences():
    """float32 gradients against central differences of the definition's own forward: <dout, d out / d theta> along random directions."""
    P = _p()
    t = inputs(60, 40, 24, 8, 3, F32, "each", seed=9)
    leaves = [t[k].clone().requires_grad_() for k in ("y", "x", "A", "B")]
    grads = torch.autograd.grad(P.DenseAdaptersFunction.apply(*leaves, t["which"], t["scale"]), leaves, t["dy"])
    gen = torch.Generator(device="cuda").manual_seed(10)
    for k, g in zip(("y", "x", "A", "B"), grads):
        d, h = torch.randn(t[k].shape, generator=gen, device="cuda").double(), 1e-4
        up, down = ({**t, k: t[k].double() + s * h * d} for s in (1, -1))
        diff = ((definition(up)[0]["out"][0] - definition(down)[0]["out"][0]) * t["dy"].double()).sum() / (2 * h)
        # the forward is quadratic in no single operand: the difference is exact but for 64-bit rounding
        assert abs(float((g.double() * d).sum() - diff)) <= 1e-4 * float((g.double() * d).abs().sum())


def test_shapes_strides_and_out():
    P = _p()
    t = inputs(48, 72, 40, 12, 4, BF16, "each")
    want = definition(t)[0]["out"]
    x3, y3, w3 = t["x"].view(4, 12, 72), t["y"].view(4, 12, 40), t["which"].view(4, 12)
    near(P.dense_adapters(y3, x3, t["A"], t["B"], w3.long(), t["scale"]).view(48, 40), want, "three dimensions")
    wide = torch.zeros(48, 144, dtype=BF16, device="cuda")
    wide[:, ::2] = t["x"]
    near(P.dense_adapters(t["y"].t().contiguous().t(), wide[:, ::2], t["A"].transpose(1, 2).contiguous().transpose(1, 2), t["B"], t["which"], t["scale"]),
         want, "strides")
    y = t["y"].clone()
    assert P.dense_adapters(y, t["x"], t["A"], t["B"], t["which"], t["scale"], out=y) is y
    near(y, want, "in place")
    assert torch.equal(y[t["which"] < 0], t["y"][t["which"] < 0])
    # views off sixteen bytes, and what lies around the output
    buf = torch.full((48 * 40 + 16,), 7.0, dtype=BF16, device="cuda")
    out = buf[3:3 + 48 * 40].view(48, 40)
    xb = torch.zeros(48 * 72 + 8, dtype=BF16, device="cuda")
    x = xb[1:1 + 48 * 72].view(48, 72)
    x.copy_(t["x"])
    P.dense_adapters(t["y"], x, t["A"], t["B"], t["which"], t["scale"], out=out)
    near(out, want, "off sixteen bytes")
    assert bool((buf[:3] == 7).all()) and bool((buf[3 + 48 * 40:] == 7).all())
    # operands and output as parts of one buffer
    one = torch.zeros(48, 72 + 40, dtype=BF16, device="cuda").view(-1)
    xs, os_ = one[:48 * 72].view(48, 72), one[48 * 72:].view(48, 40)
    xs.copy_(t["x"])
    near(P.dense_adapters(t["y"], xs, t["A"], t["B"], t["which"], t["scale"], out=os_), want, "parts of one buffer")
    for bad in (one[48 * 40:48 * 80].view(48, 40), one[:48 * 40].view(48, 40)):
        with pytest.raises(ValueError, match="share memory"):
            P.dense_adapters(t["y"], xs, t["A"], t["B"], t["which"], out=bad)
    with pytest.raises(ValueError, match="out may be Y"):
        P.dense_adapters(one[8:8 + 48 * 40].view(48, 40), t["x"], t["A"], t["B"], t["which"], out=one[:48 * 40].view(48, 40))
    none = P.dense_adapters(t["y"][:0], t["x"][:0], t["A"], t["B"], t["which"][:0])
    assert none.shape == (0, 40)


def test_no_rows_give_zero_gradients():
    P = _p()
    A, B = (torch.randn(3, 8, 8, device="cuda", requires_grad=True) for _ in range(2))
    x, y = torch.zeros(0, 8, device="cuda", requires_grad=True), torch.zeros(0, 8, device="cuda", requires_grad=True)
    out = P.DenseAdaptersFunction.apply(y, x, A, B, torch.zeros(0, dtype=torch.int32, device="cuda"))
    g = torch.autograd.grad(out, (x, A, B), torch.zeros(0, 8, device="cuda"))
    assert g[0].shape == (0, 8) and not bool(g[1].any()) and not bool(g[2].any())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_what_is_not_finite_stays_with_its_rows_and_adapters(dtype):
    P = _p()
    rows, count = 150, 5
    t = inputs(rows, 136, 72, 16, count, dtype, "each", seed=4)
    clean = definition(t)[0]
    bad = {k: v.clone() for k, v in t.items()}
    bad["A"][2, 5] = float("nan")
    bad["B"][2, :, 3] = float("inf")
    row = int((t["which"] == 1).nonzero()[0])
    bad["x"][row, 7] = float("inf")
    bad["x"][t["which"] == -1] = float("nan")
    bad["dy"][t["which"] == -1] = float("nan")
    fine = (t["which"] != 2) & (torch.arange(rows, device="cuda") != row)
    leaves = [bad[k].clone().requires_grad_() for k in ("y", "x", "A", "B")]
    out = P.DenseAdaptersFunction.apply(*leaves, t["which"], t["scale"])
    _, dx, dA, dB = torch.autograd.grad(out, leaves, bad["dy"])
    near(out.detach()[fine], tuple(a[fine] for a in clean["out"]), "forward")
    assert not bool(torch.isfinite(out.detach()[row]).all()) and bool(torch.isnan(out.detach()[t["which"] == 2]).all())
    keep = t["which"] != 2
    near(dx[keep], tuple(a[keep] for a in clean["dx"]), "dX")
    for a in (0, 3, 4):
        near(dA[a], tuple(q[a] for q in clean["dA"]), "dA")
        near(dB[a], tuple(q[a] for q in clean["dB"]), "dB")
    near(dB[1][:, :0], tuple(q[1][:, :0] for q in clean["dB"]), "dB")
    assert not bool(torch.isfinite(dA[1][7]).all()) and bool(torch.isfinite(dA[1][8]).all())


def test_an_infinite_row_of_the_gradient():
    P = _p()
    t = inputs(100, 64, 64, 16, 2, BF16, "runs")
    t["dy"][3, 5] = float("inf")
    leaves = [t[k].clone().requires_grad_() for k in ("y", "x", "A", "B")]
    dx, dA, dB = torch.autograd.grad(P.DenseAdaptersFunction.apply(*leaves, t["which"], t["scale"]), leaves[1:], t["dy"])
    assert bool(torch.isfinite(dx[:3]).all()) and bool(torch.isfinite(dx[4:]).all()) and not bool(torch.isfinite(dx[3]).all())
    assert bool(torch.isfinite(dA[1]).all()) and bool(torch.isfinite(dB[1]).all())


def test_a_plan_serves_many_layers_and_is_one_of_its_batch():
    P = _p()
    t = inputs(90, 64, 48, 8, 6, F16, "each")
    u = inputs(90, 200, 64, 20, 6, F16, "each", seed=1)
    plan = P.adapter_plan(t["which"], 6)
    u["which"] = t["which"]
    for v in (t, u):
        near(P.dense_adapters(v["y"], v["x"], v["A"], v["B"], plan, v["scale"]), definition(v)[0]["out"], "planned")
    want, V = definition(u)
    dx, dA, dB = P.dense_adapters_backward(u["dy"], u["x"], V.to(F16), u["A"], u["B"], plan, u["scale"])
    near(dx, want["dx"], "dX")
    near(dA, want["dA"], "dA")
    near(dB, want["dB"], "dB")
    assert P.dense_adapters_backward(u["dy"], u["x"], V.to(F16), u["A"], u["B"], plan, u["scale"], need_dx=False, need_da=False)[:2] == (None, None)
    only = P.dense_adapters_backward(u["dy"], u["x"], V.to(F16), u["A"], u["B"], plan, u["scale"], need_dx=False, need_db=False)
    assert torch.equal(only[1], dA)
    with pytest.raises(ValueError):
        P.dense_adapters(t["y"][:80], t["x"][:80], t["A"], t["B"], plan)
    with pytest.raises(ValueError):
        P.dense_adapters(t["y"], t["x"], t["A"][:5], t["B"][:5], plan)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows", [3, 200])
def test_the_product_with_the_adapter_is_not_rounded_between(dtype, rows):
    """V as two 16-bit parts: out and dX carry their own rounding and 2**-8 of another (bf16: e * e relative to V, and fp16's second part may fall below its
    smallest number, 2**-25)."""
    P = _p()
    t = inputs(rows, 256, 512, 4, 3, dtype, "each", seed=rows)
    want, V = definition(t)
    e = torch.finfo(dtype).eps / 2
    a = t["which"].long().clamp(min=0)
    B, A = t["B"].double()[a].abs(), t["A"].double()[a].abs()
    sums = (t["x"].double().abs().unsqueeze(1) @ A) * t["scale"].double().abs()[a].view(-1, 1, 1)
    ev = 258 * U * sums + e * e * V.abs().unsqueeze(1) + 2.0 ** -25
    bound = ((ev + 2 * 6 * U * V.abs().unsqueeze(1)) @ B).squeeze(1) + (e + 2 * U) * want["out"][0].abs() + U * t["y"].double().abs()
    near(P.dense_adapters(t["y"], t["x"], t["A"], t["B"], t["which"], t["scale"]), (want["out"][0], bound), "forward")


def test_the_same_bits_each_time_and_for_any_order_of_calls():
    P = _p()
    t = inputs(3000, 256, 256, 16, 3, BF16, "each")
    def once():
        leaves = [t[k].clone().requires_grad_() for k in ("y", "x", "A", "B")]
        out = P.DenseAdaptersFunction.apply(*leaves, t["which"], t["scale"])
        return (out.detach(), *torch.autograd.grad(out, leaves, t["dy"]))
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_other_streams_and_captured_calls():
    P = _p()
    t, u = inputs(100, 128, 128, 16, 4, BF16, "each"), inputs(100, 128, 128, 16, 4, BF16, "each", seed=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = P.dense_adapters(t["y"], t["x"], t["A"], t["B"], t["which"], t["scale"])
    torch.cuda.current_stream().wait_stream(side)
    near(out, definition(t)[0]["out"], "side stream")
    # two graphs of the same call on other inputs, replayed in turn: the adapters' numbers are read at each replay
    held = [{k: v.clone() for k, v in s.items()} for s in (t, u)]
    graphs = []
    for s in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s["out"] = P.dense_adapters(s["y"], s["x"], s["A"], s["B"], s["which"], s["scale"])
        graphs.append(g)
    for _ in range(2):
        for g in graphs:
            g.replay()
        for s, v in zip(held, (t, u)):
            near(s["out"], definition({k: s[k] for k in v})[0]["out"], "replayed")
            s["which"].copy_(s["which"].roll(1))


def test_training_pass_captured_into_a_graph():
    P = _p()
    t = inputs(300, 128, 192, 16, 3, BF16, "each")
    want = definition(t)[0]
    leaves = [t[k].clone().requires_grad_() for k in ("y", "x", "A", "B")]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.autograd.grad(P.DenseAdaptersFunction.apply(*leaves, t["which"], t["scale"]), leaves, t["dy"])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = P.DenseAdaptersFunction.apply(*leaves, t["which"], t["scale"])
        grads = torch.autograd.grad(out, leaves, t["dy"])
    g.replay()
    near(out.detach(), want["out"], "forward")
    for k, q in zip(("dx", "dA", "dB"), grads[1:]):
        near(q, want[k], k)


def test_offsets_past_32_bits():
    P = _p()
    rows, I, O, R = 270000, 8192, 16, 8
    x = torch.zeros(rows, I, dtype=BF16, device="cuda")
    which = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    pick = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device="cuda")
    t = inputs(5, I, O, R, 2, BF16, "one")
    x[pick] = t["x"]
    which[pick] = 1
    y = torch.ones(rows, O, dtype=BF16, device="cuda")
    t["y"], t["which"] = y[pick], which[pick]
    want = definition(t)[0]
    leaves = [a.requires_grad_() for a in (y, x, t["A"].clone(), t["B"].clone())]
    out = P.DenseAdaptersFunction.apply(*leaves, which, t["scale"])
    near(out.detach()[pick], want["out"], "forward")
    assert bool((out.detach()[which < 0] == 1).all())
    dy = torch.zeros(rows, O, dtype=BF16, device="cuda")
    dy[pick] = t["dy"]
    dx, dA, dB = torch.autograd.grad(out, leaves[1:], dy)
    near(dx[pick], want["dx"], "dX")
    near(dA, want["dA"], "dA")
    near(dB, want["dB"], "dB")
    assert int(torch.count_nonzero(dx)) == int(torch.count_nonzero(dx[pick]))   # the other rows are zero


def test_many_adapters():
    P = _p()
    count, rows = 16384, 400
    gen = torch.Generator(device="cuda").manual_seed(3)
    which = torch.randint(count, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    x, y = torch.randn(rows, 16, device="cuda"), torch.randn(rows, 8, device="cuda")
    A, B = torch.randn(count, 16, 4, device="cuda"), torch.randn(count, 4, 8, device="cuda")
    out = P.dense_adapters(y, x, A, B, which)
    w = which.long()
    want = y.double() + ((x.double().unsqueeze(1) @ A.double()[w]) @ B.double()[w]).squeeze(1)
    size = y.double().abs() + ((x.double().abs().unsqueeze(1) @ A.double().abs()[w]) @ B.double().abs()[w]).squeeze(1)
    near(out, (want, 24 * U * size), "many adapters")
