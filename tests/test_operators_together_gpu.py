"""The adapters, the gated block and the AdamW step as they are used together: a block served and trained, and the data-parallel steps that hand
their gradients to the optimiser."""
import pytest
import torch

BF16 = torch.bfloat16


class Block(torch.nn.Module):
    """x -> gated half in bfloat16 -> a CP dense layer shared by all requests, with an adapter for each."""

    def __init__(self):
        super().__init__()
        from paralleltnnlayers_b200 import layers as L
        torch.manual_seed(0)
        self.gated = L.GatedDense(96, 256)
        self.down = L.AdaptedDense(L.CPDense(256, 64, rank=12, input_shape=(16, 16), output_shape=(8, 8)), count=3, rank=8, scale=0.5)
        with torch.no_grad():
            self.down.B.normal_(0, 0.2)

    def forward(self, x, adapters):
        return self.down(self.gated(x).float(), adapters)


def exact(block, x, which, d):
    """The block's output and gradients in 64 bits, from the values that its parameters have."""
    p = {n: q.detach().double().requires_grad_() for n, q in block.named_parameters()}
    F = [p[f"down.shared.factors.{k}"] for k in range(2)]
    M = torch.einsum("abr,cdr->acbd", *F).reshape(256, 64)
    h = torch.nn.functional.silu(x.double() @ p["gated.Wg"]) * (x.double() @ p["gated.Wu"])
    y = h @ M
    for a in range(3):
        rows = (which == a).double().unsqueeze(1)
        y = y + rows * 0.5 * (h @ p["down.A"][a]) @ p["down.B"][a]
    names = [n for n in p if "shared" not in n]
    return y, dict(zip(names, torch.autograd.grad(y, [p[n] for n in names], d.double())))


def batch(rows, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, 96, generator=gen, device="cuda").to(BF16), torch.randint(-1, 3, (rows,), generator=gen, device="cuda", dtype=torch.int32),
            torch.randn(rows, 64, generator=gen, device="cuda"))


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_block_is_trained(bits):
    """bfloat16 inside: outputs and gradients carry the rounding of h (2**-9 of each value) and, in the gated half, of dh, dG and dU, four in all: 4 * 2**-9 of
    the norm at most.  The update is checked against the formula with the gradients that the backward gave."""
    import paralleltnnlayers_b200 as P
    from paralleltnnlayers_b200.optim import AdamW
    block = Block().cuda()
    opt = AdamW([p for p in block.parameters() if p.requires_grad], lr=1e-2, weight_decay=0.1, bits=bits)
    assert not any(p.requires_grad for n, p in block.named_parameters() if "shared" in n)
    moments = {}
    for t in (1, 2, 3):
        x, which, d = batch(200, t)
        y, grads = exact(block, x, which, d)
        out = block(x, which)
        assert off(out.detach(), y.detach()) < 4 * 2.0 ** -9
        opt.zero_grad()
        out.backward(d)
        params = {n: p for n, p in block.named_parameters() if p.requires_grad}
        for n, p in params.items():
            assert off(p.grad, grads[n]) < 4 * 2.0 ** -9, n
        before = {n: (opt.state[p]["master"] if t > 1 and "master" in opt.state[p] else p.detach().float()).double() for n, p in params.items()}
        opt.step()
        for n, p in params.items():
            g, s = p.grad.double(), opt.state[p]
            m, v = moments.get(n, (torch.zeros_like(g), torch.zeros_like(g)))
            m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
            want = before[n] * (1 - 1e-3) - 1e-2 * (m / (1 - 0.9 ** t)) / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8)
            now = s.get("master", p.detach()).double()
            assert float((now - want).abs().max()) < 1e-5, n
            if "master" in s:
                assert torch.equal(p.detach(), s["master"].to(BF16))
            if bits == 8:
                m, v = (q.double() for q in P.adamw_moments(s["exp_avg"], s["exp_avg_sq"], (s["scale_avg"], s["scale_sq"]), torch.float32))
            moments[n] = (m, v)
    P.device_status()


@pytest.mark.gpu
def test_a_block_is_served():
    """A batch of prompts, then single tokens of its requests, eagerly and from a captured graph: rows are what they are in any batch."""
    import paralleltnnlayers_b200 as P
    block = Block().cuda()
    x, which, d = batch(300, 9)
    with torch.no_grad():
        y, _ = exact_rows(block, x, which)
        plan = P.adapter_plan(which, 3)
        full = block(x, plan)
        assert off(full, y) < 4 * 2.0 ** -9
        for rows in (1, 5, 40, 130):
            assert off(block(x[:rows], which[:rows]), y[:rows]) < 4 * 2.0 ** -9
        tokens, numbers = x[:24].clone(), which[:24].clone()
        block(tokens, numbers)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(tokens, numbers)
        for at in (0, 24, 276):
            tokens.copy_(x[at:at + 24])
            numbers.copy_(which[at:at + 24])
            graph.replay()
            assert off(out, y[at:at + 24]) < 4 * 2.0 ** -9
    P.device_status()


def exact_rows(block, x, which):
    with torch.enable_grad():
        y, g = exact(block, x, which, torch.zeros(x.shape[0], 64, device="cuda"))
    return y.detach(), g


@pytest.mark.gpu
def test_a_captured_training_step():
    """Forward, backward and update in one graph: replays go on where the last one stopped, as eager steps of a twin do."""
    from paralleltnnlayers_b200.optim import AdamW
    one, two = Block().cuda(), Block().cuda()
    x, which, d = batch(64, 3)
    opts = [AdamW([p for p in b.parameters() if p.requires_grad], lr=1e-2, capturable=True) for b in (one, two)]

    def step(block, opt):
        opt.zero_grad(set_to_none=True)
        block(x, which).backward(d)
        opt.step()

    for _ in range(4):
        step(two, opts[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(one, opts[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    opts[0].zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(one, opts[0])
    for _ in range(3):
        graph.replay()
    for a, b in zip(one.parameters(), two.parameters()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_data_parallel_steps_hand_their_gradients_to_the_optimiser():
    from paralleltnnlayers_b200 import dist as D
    from paralleltnnlayers_b200.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    F = [torch.nn.Parameter(n(4, 4, 3)), torch.nn.Parameter(n(4, 2, 3))]
    K = [torch.nn.Parameter(n(d, 4) * 0.3) for d in (6, 5, 3, 3)]
    A = [torch.nn.Parameter(n(2, 3, 4)), torch.nn.Parameter(n(2, 2, 4))]
    S = torch.nn.Parameter(n(3, 3, 4))
    runs = [(F, lambda o: D.dense_data_parallel_step(n(7, 16), n(7, 8), F, optimizer=o)[2]),
            (K, lambda o: D.cp4_data_parallel_step(n(2, 5, 8, 8), n(2, 6, 8, 8), *K, optimizer=o)[2]),
            ([*A, S], lambda o: (lambda r: [*r[2], r[3]])(D.rcp_data_parallel_step(n(2, 4, 8, 8), n(2, 6, 8, 8), A, S, optimizer=o)))]
    for params, run in runs:
        before = [p.detach().clone() for p in params]
        grads = run(AdamW(params, lr=1e-2, weight_decay=0.0))
        for p, b, g in zip(params, before, grads):   # the first step is lr times the sign of the gradient
            assert torch.equal(p.grad, g)
            big = g.abs() > 1e-3
            assert bool(((p.detach() - b + 1e-2 * g.sign())[big].abs() < 1e-6 + 2.0 ** -22 * b.abs()[big]).all())
        with pytest.raises(ValueError, match="over the factors"):
            run(AdamW([torch.nn.Parameter(n(3))]))


def test_layers_refuse_what_does_not_fit():
    from paralleltnnlayers_b200 import layers as L
    shared = L.CPDense(16, 8, rank=2, input_shape=(4, 4), output_shape=(4, 2))
    m = L.AdaptedDense(shared, 2, 4)
    assert m.A.shape == (2, 16, 4) and m.B.shape == (2, 4, 8) and not bool(m.B.any()) and not any(p.requires_grad for p in shared.parameters())
    assert L.AdaptedDense(torch.nn.Linear(5, 3), 1, 2, freeze=False).B.shape == (1, 2, 3)
    assert m.to(torch.float16).scale.dtype == torch.float32
    for bad in (lambda: L.AdaptedDense(torch.nn.ReLU(), 2, 4), lambda: L.AdaptedDense(shared, 0, 4), lambda: L.AdaptedDense(shared, 2, 129),
                lambda: L.GatedDense(8, 8, activation="relu"), lambda: L.GatedDense(8, 8, dtype=torch.float32)):
        with pytest.raises(ValueError):
            bad()
