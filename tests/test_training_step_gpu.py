"""The embedding, layer norm and the Muon step as they are used together: a small language model trained, served, and stepped by a captured graph."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


class Model(torch.nn.Module):
    """tokens -> embedding -> (norm -> gated half -> dense layer with adapters, added to the stream) -> norm -> rows of the same width."""

    def __init__(self):
        super().__init__()
        from paralleltnnlayers_b200 import layers as L
        torch.manual_seed(0)
        self.embed = L.Embedding(101, 64, scale=8.0, dtype=BF16)
        self.first, self.last = L.LayerNorm(64), L.LayerNorm(64, bias=False)
        self.gated = L.GatedDense(64, 256)
        self.down = L.AdaptedDense(L.CPDense(256, 64, rank=12, input_shape=(16, 16), output_shape=(8, 8)), count=3, rank=8)
        with torch.no_grad():
            self.down.B.normal_(0, 0.2)

    def forward(self, tokens, adapters):
        x = self.embed(tokens)
        y = self.down(self.gated(self.first(x)).float(), adapters).to(BF16)
        return self.last(y, x)


def exact(model, tokens, which, d):
    """The results and the trained parameters' gradients in 64 bits."""
    p = {n: q.detach().double().requires_grad_() for n, q in model.named_parameters()}
    norm = lambda x, n: (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * p[n + ".weight"] + p.get(n + ".bias", 0.0)  # noqa: E731
    F = [p[f"down.shared.factors.{k}"] for k in range(2)]
    M = torch.einsum("abr,cdr->acbd", *F).reshape(256, 64)
    held = (tokens >= 0).unsqueeze(-1)
    x = torch.where(held, 8.0 * p["embed.W"][tokens.clamp(min=0)], 0)
    u = norm(x, "first")
    h = torch.nn.functional.silu(u @ p["gated.Wg"]) * (u @ p["gated.Wu"])
    y = h @ M
    for a in range(3):
        y = y + (which == a).double().unsqueeze(-1) * (h @ p["down.A"][a]) @ p["down.B"][a]
    s = x + y
    out = norm(s, "last")
    names = [n for n in p if "shared" not in n]
    return out, s, dict(zip(names, torch.autograd.grad((out, s), [p[n] for n in names], (d[0].double(), d[1].double()))))


def batch(seed, shape=(4, 70)):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    tokens = torch.randint(-1, 101, shape, generator=gen, device="cuda")
    return tokens, torch.randint(-1, 3, shape, generator=gen, device="cuda"), [torch.randn(*shape, 64, generator=gen, device="cuda").to(BF16) for _ in range(2)]


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


def optimisers(model):
    from paralleltnnlayers_b200.optim import AdamW, Muon
    trained = {n: p for n, p in model.named_parameters() if p.requires_grad}
    matrices = [p for n, p in trained.items() if n.split(".")[0] in ("gated", "down")]
    rest = [p for n, p in trained.items() if n.split(".")[0] not in ("gated", "down")]
    return Muon(matrices, lr=0.02, momentum=0.9), AdamW(rest, lr=1e-3, capturable=True), trained


def test_a_model_is_trained():
    """bfloat16 between the operators: a result carries up to eight roundings of 2**-9 (embedding, both norms, gated half with its kept sums, the dense
    layer's result, the stream), 8 * 2**-9 of the norm; the gradients twice that (forward and backward)."""
    import paralleltnnlayers_b200 as P
    model = Model().cuda()
    muon, adamw, trained = optimisers(model)
    momentum = {}
    for t in (1, 2, 3):
        tokens, which, d = batch(t)
        want, stream, grads = exact(model, tokens, which, d)
        out, h = model(tokens, which)
        assert off(out.detach(), want.detach()) < 8 * 2.0 ** -9 and off(h.detach(), stream.detach()) < 8 * 2.0 ** -9
        muon.zero_grad()
        adamw.zero_grad()
        torch.autograd.backward((out, h), d)
        for n, p in trained.items():
            assert off(p.grad, grads[n]) < 16 * 2.0 ** -9, n
        assert not model.embed.W.grad[[k for k in range(101) if not bool((tokens == k).any())]].any()
        before = {p: muon.state[p]["master"] if "master" in muon.state.get(p, {}) else p.detach().float() for p in muon.param_groups[0]["params"]}
        before = {p: v.double().clone() for p, v in before.items()}
        muon.step()
        adamw.step()
        for p, w in before.items():
            g = p.grad.double()
            m = momentum[p] = 0.9 * momentum.get(p, torch.zeros_like(g)) + 0.1 * g
            X = P.orthogonalise((0.1 * g + 0.9 * m).float()).double()   # (checked by itself elsewhere; here: what the step makes of it)
            r, c = p.shape[-2:]
            step = 0.02 * max(1.0, r / c) ** 0.5 * X
            now = muon.state[p].get("master", p.detach()).double()
            # the direction here and there differ by roundings of fp32, which the steps raise by less than 4**5
            assert off(now - 0.998 * w, -step) < 4 ** 5 * 2.0 ** -22 + 2.0 ** -22 * float(w.norm() / step.norm())
            if p.dtype == BF16:
                assert torch.equal(p.detach(), muon.state[p]["master"].to(BF16))
    P.device_status()


def test_a_model_is_served():
    import paralleltnnlayers_b200 as P
    model = Model().cuda()
    tokens, which, d = batch(9)
    with torch.no_grad():
        want = exact_rows(model, tokens, which)
        assert off(model(tokens, which)[0], want) < 8 * 2.0 ** -9
        for rows in (1, 3, 40):
            t, w = tokens.flatten()[:rows], which.flatten()[:rows]
            assert off(model(t, w)[0], want.flatten(0, 1)[:rows]) < 8 * 2.0 ** -9
        t, w = tokens.flatten()[:24].clone(), which.flatten()[:24].clone()
        model(t, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, _ = model(t, w)
        for at in (0, 24, 200):
            t.copy_(tokens.flatten()[at:at + 24])
            w.copy_(which.flatten()[at:at + 24])
            graph.replay()
            assert off(out, want.flatten(0, 1)[at:at + 24]) < 8 * 2.0 ** -9
    P.device_status()


def exact_rows(model, tokens, which):
    zero = [torch.zeros(*tokens.shape, 64, device="cuda") for _ in range(2)]
    with torch.enable_grad():
        return exact(model, tokens, which, zero)[0].detach()


def test_a_captured_step_is_the_eager_one():
    models = [Model().cuda() for _ in range(2)]
    tokens, which, d = batch(1)
    held = []
    for model in models:
        muon, adamw, trained = optimisers(model)

        def step(model=model, muon=muon, adamw=adamw, trained=trained):
            out = model(tokens, which)
            for p, g in zip(trained.values(), torch.autograd.grad(out, list(trained.values()), d)):
                p.grad = g
            muon.step()
            adamw.step()
        held.append(step)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held[0]()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held[0]()
    held[1]()
    for seed in (2, 3):
        for t, v in zip((tokens, which, *d), (lambda b: (b[0], b[1], *b[2]))(batch(seed))):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        held[1]()
        for a, b in zip(models[0].parameters(), models[1].parameters()):
            assert torch.equal(a, b)


def test_a_capture_begins_no_state():
    from paralleltnnlayers_b200.optim import Muon
    p = torch.nn.Parameter(torch.randn(8, 12, device="cuda"))
    p.grad = torch.randn(8, 12, device="cuda")
    opt = Muon([p], lr=torch.tensor(0.1, device="cuda"))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="begins no state"):
        with torch.cuda.graph(graph):
            opt.step()


def test_a_data_parallel_step_takes_the_optimiser():
    """One rank: the step's own factors are updated by Muon with the gradients that it gives."""
    import paralleltnnlayers_b200 as P
    from paralleltnnlayers_b200 import dist
    from paralleltnnlayers_b200.optim import Muon
    torch.manual_seed(3)
    F = [torch.nn.Parameter(torch.randn(8, 8, 6, device="cuda") * 0.3) for _ in range(2)]
    X, dY = torch.randn(32, 64, device="cuda"), torch.randn(32, 64, device="cuda")
    _, dF = P.dense_cp_backward(X, dY, *[f.detach() for f in F])
    want, m = [f.detach().clone() for f in F], [torch.zeros_like(f) for f in F]
    P.muon_step(want, list(dF), m, 0.05, 0.95)
    dist.dense_data_parallel_step(X, dY, F, allreduce=lambda t: t, optimizer=Muon(F, lr=0.05))
    for f, w in zip(F, want):
        assert torch.equal(f.detach(), w)


SCRIPT = """
import torch, paralleltnnlayers_b200 as P
gen = torch.Generator(device="cuda").manual_seed(0)
n = lambda *s: torch.randn(*s, generator=gen, device="cuda")
t, W, x, r, w = torch.randint(50, (400,), generator=gen, device="cuda"), n(50, 64), n(3000, 512), n(3000, 512), n(512)
out = [P.embedding(t, W, 2.0), P.embedding_backward(n(400, 64), t, 50)]
y, h, mean, rstd = P.layer_norm_save(x, w, None, 1e-5, r)
out += [y, h, *P.layer_norm_backward(r, h, w, None, mean, rstd, x)]
out += [P.orthogonalise(n(3, 20, 40)), P.orthogonalise(n(150, 300))]
P.device_status()
print("sums", *[repr(float(o.double().abs().sum())) for o in out])
"""


def test_plain_launches_give_the_same():
    """B200CP_PDL=0: every launch waits for the one before it to end."""
    root, lines = os.path.dirname(os.path.dirname(os.path.abspath(__file__))), []
    for value in ("0", "1"):
        run = subprocess.run([sys.executable, "-c", SCRIPT], cwd=root, env={**os.environ, "B200CP_PDL": value}, capture_output=True, text=True, timeout=120)
        assert run.returncode == 0, run.stderr[-2000:]
        lines.append(run.stdout.split("sums")[1])
    assert lines[0] == lines[1]


def test_a_trained_model_uses_every_type():
    """A step of each type of parameter: the layers in bfloat16 and float16 under norms of float32, and all of it in float32."""
    from paralleltnnlayers_b200 import layers as L
    from paralleltnnlayers_b200.optim import Muon
    for dtype in (torch.float32, BF16, torch.float16):
        torch.manual_seed(1)
        embed, norm, dense = L.Embedding(30, 48, dtype=dtype).cuda(), L.LayerNorm(48).cuda(), torch.nn.Linear(48, 80, bias=False).cuda().to(dtype)
        opt = Muon(dense.parameters(), lr=0.01, master=dtype != torch.float32)
        kept = dense.weight.detach().clone()
        tokens = torch.randint(30, (64,), device="cuda")
        dense(norm(embed(tokens))).float().square().mean().backward()
        assert embed.W.grad.dtype == dtype and norm.weight.grad.dtype == torch.float32
        opt.step()
        step = (dense.weight.detach() - kept).float()
        assert step.isfinite().all() and bool(step.any())
