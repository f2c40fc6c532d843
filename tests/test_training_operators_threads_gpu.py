"""The operators around the blocks from two host threads at once, each on a stream of its own, and in graphs that share their memory."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def inputs(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    S, V, D = 1500 + seed, 700, 520
    return {"t": torch.randint(-1, V, (S,), generator=gen, device="cuda"), "W": n(V, D).bfloat16(), "dy": n(S, D).bfloat16(), "x": n(S, D).bfloat16(),
            "r": n(S, D).bfloat16(), "w": n(D), "g": [n(*s) for s in ((200, 300), (64, 90), (3, 16, 40), (70, 66))]}


def work(i, steps=5):
    import paralleltnnlayers_b200 as P
    out = [P.embedding(i["t"], i["W"], 2.0), P.embedding_backward(i["dy"], i["t"], 700, 2.0)]
    y, h, mean, rstd = P.layer_norm_save(i["x"], i["w"], None, 1e-5, i["r"])
    out += [y, h, *P.layer_norm_backward(i["dy"], h, i["w"], None, mean, rstd, i["r"])]
    p, m = [torch.zeros_like(g) for g in i["g"]], [torch.zeros_like(g) for g in i["g"]]
    P.muon_step(p, i["g"], m, 0.1, steps=steps)
    return out + p + m


def same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b))


def test_two_threads():
    import paralleltnnlayers_b200 as P
    given = [inputs(k) for k in range(2)]
    want = [work(i) for i in given]
    torch.cuda.synchronize()
    bad, start = [], threading.Barrier(2)

    def run(k):
        try:
            side = torch.cuda.Stream()
            start.wait(60)
            with torch.cuda.stream(side):
                outs = [work(given[k]) for _ in range(20)]
            side.synchronize()
            bad.extend(k for o in outs if not same(o, want[k]))
        except Exception as e:   # noqa: BLE001
            bad.append(e)
    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad
    P.device_status()


@pytest.mark.parametrize("steps", [5, 12])
def test_graphs_that_share_memory(steps):
    given = [inputs(k) for k in range(2)]
    want = [work(i, steps) for i in given]
    graphs = []
    for i in given:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
            out = work(i, steps)
        graphs.append((g, out))
    for k in (0, 1, 1, 0):
        graphs[k][0].replay()
        assert same(graphs[k][1], want[k])
