"""Operators around the blocks of a language model, as cases that can be timed and compared: the embedding with its gradient, layer norm with its
gradients, and the Muon step, which orthogonalises the update of a matrix by Newton-Schulz products.

``listed()`` holds the named cases, ``draw(rng)`` more of the same ranges:

    embedding  1-65536 tokens (some of them none: padding) of 16-100000, rows of 8-8192 values; float32, bfloat16, float16
    norm       1-16384 rows of 8-16384 features, with or without the residual that is added first, with or without a bias
    muon       1-60 matrices or stacks of them, sides of 1 to 10240; float32, or 16-bit types with or without a float32 copy
    orthogonal the orthogonalisation alone, a matrix or a stack of them

Each computes in its plain form (``own = False``) with elementary tensor operations in 32 bits, or (``own = True``) by this package.
"""
import math

import torch

own = False

# the most of a drawn case: the work of the largest listed ones
MAX_FLOPS, MAX_BYTES = 8.7e12, 2.7e9
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS, NS_EPS, COEFFICIENTS, STEPS = 1e-5, 1e-7, (3.4445, -4.7750, 2.0315), 5
RATE, MOMENTUM, DECAY = 0.02, 0.95, 0.1


def _embedding(name, mode, S, V, D, bare, dtype, numbers):
    return {"name": name, "op": "embedding", "mode": mode, "S": S, "V": V, "D": D, "bare": bare, "dtype": dtype, "numbers": numbers}


def _norm(name, mode, S, D, residual, bias, dtype):
    return {"name": name, "op": "norm", "mode": mode, "S": S, "D": D, "residual": residual, "bias": bias, "dtype": dtype}


def _muon(name, sizes, dtype, master, adjust):
    return {"name": name, "op": "muon", "sizes": sizes, "dtype": dtype, "master": master, "adjust": adjust}


def _orthogonal(name, sizes, dtype):
    return {"name": name, "op": "orthogonal", "sizes": sizes, "dtype": dtype}


def listed():
    return [
        # one token of one request: the latency of a call
        _embedding("embedding_one_token", "forward", 1, 32000, 1024, 0.0, "bfloat16", "int64"),
        # a batch of sequences in training, with the gradient of the whole table; some tokens are padding
        _embedding("embedding_train", "train", 8192, 50021, 4096, 0.05, "bfloat16", "int64"),
        # a small table in float32, with sizes that are no multiples of anything
        _embedding("embedding_train_odd", "train", 1500, 1001, 513, 0.2, "float32", "int32"),
        # one token through a norm
        _norm("norm_one_token", "forward", 1, 1024, False, True, "bfloat16"),
        # prompts: the block's output is added to the stream, and the sum is normed for the next block
        _norm("norm_prompts", "forward", 5003, 4096, True, False, "float16"),
        # training, a batch of sequences
        _norm("norm_train", "train", 8192, 4096, True, True, "bfloat16"),
        # beside a float32 dense layer of this package, with sizes that are no multiples of anything
        _norm("norm_train_odd", "train", 1021, 1001, False, True, "float32"),
        # the factors of a network of CP layers (the benchmark's channel counts): many small matrices
        _muon("muon_factors", "64x16*6,128x32*8,256x32*8,512x64*8,3x16*12,8x8x32*4", "float32", False, "match_rms_adamw"),
        # the adapters of a layer: stacks of tall and of wide matrices
        _muon("muon_adapters", "32x4096x16*1,32x16x4096*1", "bfloat16", True, "original"),
        # the weights of a gated block and of the projection behind it, bfloat16 with float32 copies
        _muon("muon_block", "4096x10240*2,10240x4096*1", "bfloat16", True, "match_rms_adamw"),
        # 16-bit parameters alone, odd sizes
        _muon("muon_odd", "1030x2051*2,513x1001*1,77x300*2", "float16", False, "original"),
        # the orthogonalisation of one large weight, in float32
        _orthogonal("orthogonal_weight", "4096x4096*1", "float32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _features(rng, lo, hi):
    """Feature counts are mostly multiples of 8; some are not."""
    n = _log_int(rng, lo, hi)
    return max(8, n // 64 * 64 if n >= 256 else n // 8 * 8) if rng.random() < 0.7 else n


def draw(rng):
    while True:
        op = rng.choice(["embedding", "norm", "norm", "muon", "muon", "orthogonal"])
        dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
        mode = rng.choice(["forward", "train", "train"])
        if op == "embedding":
            case = {"op": op, "mode": mode, "S": _log_int(rng, 1, 65536), "V": _log_int(rng, 16, 100000), "D": _features(rng, 8, 8192),
                    "bare": rng.choice([0.0, 0.05, 0.5]), "dtype": dtype, "numbers": rng.choice(["int32", "int64"])}
        elif op == "norm":
            case = {"op": op, "mode": mode, "S": _log_int(rng, 1, 16384), "D": _features(rng, 8, 16384), "residual": rng.random() < 0.5,
                    "bias": rng.random() < 0.6, "dtype": dtype}
        else:
            groups = []
            for _ in range(rng.randint(1, 4) if op == "muon" else 1):
                r, c = _features(rng, 1, 4096), _features(rng, 8, 10240)
                if rng.random() < 0.4:
                    r, c = c, r
                stack = _log_int(rng, 1, 40) if rng.random() < 0.3 else 0
                groups.append(("%dx" % stack if stack else "") + "%dx%d*%d" % (r, c, _log_int(rng, 1, 12) if op == "muon" else 1))
            case = {"op": op, "sizes": ",".join(groups), "dtype": dtype}
            if op == "muon":
                case.update(master=dtype != "float32" and rng.random() < 0.6, adjust=rng.choice(["original", "match_rms_adamw"]))
        w = work(case)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return case


def _shapes(case):
    """Shape of each tensor of a Muon or orthogonalisation case: [.., rows, columns]."""
    out = []
    for group in case["sizes"].split(","):
        shape, times = group.split("*")
        out += [tuple(int(v) for v in shape.split("x"))] * int(times)
    return out


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(dtype)

    dtype = TYPES[case["dtype"]]
    if case["op"] == "embedding":
        S, V, D = case["S"], case["V"], case["D"]
        # a few tokens are frequent and most are rare: their numbers are uniform on the scale of logarithms
        tokens = (torch.rand(S, generator=gen, device="cuda", dtype=torch.float64) * math.log(V + 1)).exp().long().sub(1).clamp(0, V - 1)
        bare = torch.rand(S, generator=gen, device="cuda") < case["bare"]
        s = {"case": case, "tokens": torch.where(bare, -1, tokens).to(getattr(torch, case["numbers"])), "W": normal(V, D, dtype=dtype),
             "scale": D ** 0.5}
        if case["mode"] == "train":
            s["dy"] = normal(S, D, dtype=dtype)
            s["W"].requires_grad_()
        return s
    if case["op"] == "norm":
        S, D = case["S"], case["D"]
        s = {"case": case, "x": normal(S, D, std=2.0, mean=0.3, dtype=dtype), "w": normal(D, std=0.2, mean=1.0, dtype=dtype),
             "b": normal(D, std=0.2, dtype=dtype) if case["bias"] else None, "r": normal(S, D, dtype=dtype) if case["residual"] else None}
        if case["mode"] == "train":
            s["dy"] = normal(S, D, dtype=dtype)
            if case["residual"]:
                s["dh"] = normal(S, D, dtype=dtype)
            for k in ("x", "r", "w", "b"):
                if s[k] is not None:
                    s[k].requires_grad_()
        return s
    # gradients of matrices have a few large directions and many small ones
    shapes = _shapes(case)
    starts, total = [], 0
    for shape in shapes:
        starts.append(total)
        total += (math.prod(shape) + 255) // 256 * 256
    cut = lambda t: [t[a: a + math.prod(shape)].view(shape) for a, shape in zip(starts, shapes)]  # noqa: E731

    def matrices(std):
        t = torch.zeros(total, device="cuda")
        for part in cut(t):
            part.copy_(normal(*part.shape) + 4 * normal(*part.shape[:-1], 1) * normal(*part.shape[:-2], 1, part.shape[-1]))
        return t.mul_(std)

    if case["op"] == "orthogonal":
        return {"case": case, "X": cut(matrices(1e-2))[0].to(dtype)}
    s = {"case": case, "g": matrices(1e-2).to(dtype), "m": matrices(1e-2), "w": normal(total, std=0.05)}
    s["p"] = s["w"] if dtype == torch.float32 else s["w"].to(dtype)
    if not case["master"]:
        del s["w"]
    s["lists"] = {k: cut(s[k]) for k in ("g", "m", "w", "p") if k in s}
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    with torch.set_grad_enabled(own):   # (the plain forms write their gradients out)
        return {"embedding": _run_embedding, "norm": _run_norm, "muon": _run_muon, "orthogonal": _run_orthogonal}[op](state)


def _run_embedding(s):
    train, t, W, c = s["case"]["mode"] == "train", s["tokens"], s["W"], s["scale"]
    if own:
        import paralleltnnlayers_b200 as P
        if not train:
            return P.embedding(t, W, c)
        out = P.EmbeddingFunction.apply(t, W, c)
        return (out, *torch.autograd.grad(out, W, s["dy"]))
    held = ((t >= 0) & (t < W.shape[0])).unsqueeze(1)
    t = torch.where(held.squeeze(1), t, 0).long()
    out = torch.where(held, W[t].float() * c, 0).to(W.dtype)
    if not train:
        return out
    dW = torch.zeros(W.shape, device="cuda").index_add_(0, t, torch.where(held, s["dy"].float(), 0)) * c
    return out, dW.to(W.dtype)


def _run_norm(s):
    train, x, r, w, b = s["case"]["mode"] == "train", s["x"], s["r"], s["w"], s["b"]
    if own:
        import paralleltnnlayers_b200 as P
        if not train:
            return P.layer_norm(x, w, b, EPS, residual=r)
        out = P.LayerNormFunction.apply(x, w, b, EPS, r)
        leaves = [t for t in (x, r, w, b) if t is not None]
        if r is None:
            return (out, *torch.autograd.grad(out, leaves, s["dy"]))
        return (*out, *torch.autograd.grad(out, leaves, (s["dy"], s["dh"])))
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    f = h.float()
    d = f - f.mean(1, keepdim=True)
    rstd = 1 / ((d * d).mean(1, keepdim=True) + EPS).sqrt()
    n = d * rstd
    y = n * w.float()
    if b is not None:
        y = y + b.float()
    y = y.to(x.dtype)
    outs = (y,) if r is None else (y, h)
    if not train:
        return outs if len(outs) > 1 else y
    dy = s["dy"].float()
    g = dy * w.float()
    dx = rstd * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    if r is not None:
        dx = dx + s["dh"].float()
    dx = dx.to(x.dtype)
    grads = [dx] if r is None else [dx, dx]
    grads.append((dy * n).sum(0).to(w.dtype))
    if b is not None:
        grads.append(dy.sum(0).to(w.dtype))
    return (*outs, *grads)


def _newton_schulz(X):
    X = X / X.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=NS_EPS)
    tall = X.shape[-2] > X.shape[-1]
    if tall:
        X = X.mT
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        A = X @ X.mT
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.mT if tall else X


def _lr_factor(shape, adjust):
    r, c = shape[-2:]
    return 0.2 * max(r, c) ** 0.5 if adjust == "match_rms_adamw" else max(1.0, r / c) ** 0.5


def _run_muon(s):
    case, L = s["case"], s["lists"]
    if own:
        import paralleltnnlayers_b200 as P
        P.muon_step(L["p"], L["g"], L["m"], RATE, MOMENTUM, True, DECAY, COEFFICIENTS, NS_EPS, STEPS, case["adjust"], master=L.get("w"))
    else:
        for i, (p, g, m) in enumerate(zip(L["p"], L["g"], L["m"])):
            g = g.float()
            m.add_(g - m, alpha=1 - MOMENTUM)
            X = _newton_schulz(g + MOMENTUM * (m - g))
            w = L["w"][i] if "w" in L else p
            w.copy_(w.float() * (1 - RATE * DECAY) - RATE * _lr_factor(p.shape, case["adjust"]) * X)
            if "w" in L:
                p.copy_(w)
    return (s["p"], s["m"], s["w"]) if "w" in s else (s["p"], s["m"])


def _run_orthogonal(s):
    if own:
        import paralleltnnlayers_b200 as P
        return P.orthogonalise(s["X"], COEFFICIENTS, NS_EPS, STEPS)
    return _newton_schulz(s["X"].float()).to(s["X"].dtype)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    train = case.get("mode") == "train"
    if case["op"] == "embedding":
        S, V, D = case["S"], case["V"], case["D"]
        met = sum(1 - math.exp(-S * (1 - case["bare"]) * p) for p in _shares(V))   # rows of the table that are met
        numbers = S * (8 if case["numbers"] == "int64" else 4)
        return {"bytes": numbers + size * D * (S + met) + (size * D * (S + V) if train else 0), "flops": S * D * (2 if train else 1)}
    if case["op"] == "norm":
        S, D = case["S"], case["D"]
        forward = 4 if case["residual"] else 2
        backward = 3 if case["residual"] else 2   # the inputs have been read
        return {"bytes": size * S * D * (forward + (backward if train else 0)) + 2 * size * D, "flops": S * D * (18 if train else 8)}
    n = flops = 0
    for shape in _shapes(case):
        a, b = sorted(shape[-2:])
        n += math.prod(shape)
        flops += math.prod(shape[:-2]) * STEPS * (a * a * (a + b) + 2 * a * a * b)   # the first two products are symmetric
    return {"bytes": n * (2 * size if case["op"] == "orthogonal" else 8 + 3 * size + (8 if case["master"] else 0)), "flops": flops}


def _shares(V):
    """The share of each token, by ranges of tokens that are alike."""
    last, out = 0, []
    while last < V:
        step = max(1, last // 16)
        end = min(V, last + step)
        out += [math.log((end + 1) / (last + 1)) / math.log(V + 1) / (end - last)] * (end - last)
        last = end
    return out


# ---- the definitions, in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d = lambda t: t.detach().double()  # noqa: E731
    if case["op"] == "embedding":
        W, c, V = d(s["W"]), s["scale"], case["V"]
        t = s["tokens"].long()
        inside = (t >= 0) & (t < V)
        out = torch.zeros(case["S"], case["D"], dtype=torch.float64, device="cuda")
        out[inside] = c * W[t[inside]]
        if case["mode"] == "forward":
            return out
        dW = torch.zeros_like(W)
        dW.index_put_((t[inside],), c * d(s["dy"])[inside], accumulate=True)
        return out, dW
    if case["op"] == "norm":
        x, w = d(s["x"]), d(s["w"])
        b = d(s["b"]) if case["bias"] else None
        train = case["mode"] == "train"
        h = x if not case["residual"] else (s["x"].detach().float() + s["r"].detach().float()).to(s["x"].dtype).double()
        leaves = [t for t in (h, w, b) if t is not None]
        for t in leaves:
            t.requires_grad_(train)
        y = torch.nn.functional.layer_norm(h, (case["D"],), w, b, EPS)
        # (the sum before the norm is rounded to its type: that rounding is part of the definition)
        outs = (y.detach(),) if not case["residual"] else (y.detach(), h.detach())
        if not train:
            return outs if len(outs) > 1 else outs[0]
        grads = list(torch.autograd.grad(y, leaves, d(s["dy"])))
        if case["residual"]:
            grads[0] = grads[0] + d(s["dh"])
            grads.insert(1, grads[0])
        return (*outs, *grads)
    # 3.6e13 operations in 64 bits are about a second
    if work(case)["flops"] > 6e13:
        return None

    def polar(X):   # the polynomial on the singular values
        small = min(X.shape[-2:])
        X = X / torch.linalg.matrix_norm(X, keepdim=True).clamp(min=NS_EPS)
        I = torch.eye(small, dtype=torch.float64, device="cuda")  # noqa: E741
        a, b, c = COEFFICIENTS
        for _ in range(STEPS):
            if X.shape[-2] <= X.shape[-1]:
                A = X @ X.mT
                X = (a * I + A @ (b * I + c * A)) @ X
            else:
                A = X.mT @ X
                X = X @ (a * I + A @ (b * I + c * A))
        return X

    if case["op"] == "orthogonal":
        return polar(d(s["X"]))
    L = s["lists"]
    for i, g in enumerate(L["g"]):
        g, m = d(g), d(L["m"][i])
        m = MOMENTUM * m + (1 - MOMENTUM) * g
        X = polar((1 - MOMENTUM) * g + MOMENTUM * m)
        w = d(L["w" if case["master"] else "p"][i])
        L["m"][i] = m
        L["p"][i] = w - RATE * DECAY * w - RATE * _lr_factor(g.shape, case["adjust"]) * X
    # laid out as the buffers are, the gaps between tensors as they were
    outs = []
    for k in ("p", "m"):
        flat, at = d(s["w" if k == "p" and case["master"] else k]).clone(), 0
        for t in L[k]:
            flat[at: at + t.numel()] = t.reshape(-1)
            at += (t.numel() + 255) // 256 * 256
        outs.append(flat)
    return (outs[0], outs[1], outs[0]) if case["master"] else tuple(outs)
