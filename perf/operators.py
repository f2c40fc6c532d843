"""Operators beside the factored dense layers, as cases that can be timed and compared: low-rank adapters of many requests beside a shared
projection, the gated feed-forward product, and the AdamW step over many tensors.

``listed()`` holds the named cases, ``draw(rng)`` more of the same ranges:

    adapters   1-8192 rows (one per request while tokens are generated, runs of rows in prompts and training), 64-8192 features,
               rank 4-64, 1-64 adapters, some rows without one; float32, bfloat16, float16
    gated      1-8192 rows, 64-10240 features, bfloat16 and float16, silu or gelu
    adamw      1-300 tensors of 16 to 2**26 values, moments in 32 or 8 bits, parameters in float32 or bfloat16 with a float32 copy

Each computes in its plain form (``own = False``) with elementary tensor operations in 32 bits, or (``own = True``) by this package.
"""
import math

import torch

own = False

# the most of a drawn case: the work of the largest listed ones
MAX_FLOPS, MAX_BYTES = 2.1e12, 2.2e9
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BETAS, EPS, DECAY, RATE, BLOCK = (0.9, 0.999), 1e-8, 0.01, 1e-3, 256


def _adapters(name, mode, S, I, O, R, count, rows, bare, dtype):
    return {"name": name, "op": "adapters", "mode": mode, "S": S, "I": I, "O": O, "R": R, "count": count, "rows": rows, "bare": bare,
            "dtype": dtype}


def _gated(name, mode, S, I, F, act, dtype):
    return {"name": name, "op": "gated", "mode": mode, "S": S, "I": I, "F": F, "act": act, "dtype": dtype}


def _adamw(name, sizes, bits, dtype):
    return {"name": name, "op": "adamw", "sizes": sizes, "bits": bits, "dtype": dtype}


def listed():
    return [
        # one token of one request: the latency of a call
        _adapters("adapters_one_token", "forward", 1, 1024, 1024, 16, 4, "each", 0.0, "bfloat16"),
        # generation for 64 requests, each with an adapter of its own choice, some with none
        _adapters("adapters_generate_64", "forward", 64, 4096, 4096, 16, 32, "each", 0.1, "bfloat16"),
        # prompts of a few requests, of uneven lengths
        _adapters("adapters_prompts", "forward", 5003, 4096, 1024, 32, 8, "runs", 0.1, "float16"),
        # two adapters trained on one batch
        _adapters("adapters_train", "train", 4096, 4096, 4096, 16, 2, "runs", 0.0, "bfloat16"),
        # an adapter beside a float32 dense layer of this package, with sizes that are no multiples of anything
        _adapters("adapters_train_float32", "train", 1021, 1001, 513, 12, 3, "each", 0.05, "float32"),
        # one token through a small block
        _gated("gated_one_token", "forward", 1, 1024, 2816, "silu", "bfloat16"),
        # generation for 48 requests: the weights are what is read
        _gated("gated_generate_48", "forward", 48, 4096, 10240, "silu", "bfloat16"),
        # training, a batch of sequences
        _gated("gated_train", "train", 4096, 4096, 10240, "silu", "bfloat16"),
        # training of a smaller block with odd sizes
        _gated("gated_train_odd", "train", 1500, 1030, 2051, "gelu", "float16"),
        # the factors of a network of CP layers (the benchmark's channel counts): many small tensors
        _adamw("adamw_factors", "64x16*6,128x32*8,256x32*8,512x64*8,3x16*12,3x32*16,8x8x32*16,4096*4", 32, "float32"),
        # the weights of dense blocks, parameters in 16 bits with their float32 copy
        _adamw("adamw_weights", "4096x4096*2,4096x1024*2,4096*9", 32, "bfloat16"),
        # the same in float32 with moments in 8 bits
        _adamw("adamw_8bit", "4096x10240*1,4096x4096*1,1001x77*3,4096*5", 8, "float32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _features(rng, lo, hi):
    """Feature counts are mostly multiples of 8; some are not."""
    n = _log_int(rng, lo, hi)
    return max(8, n // 64 * 64 if n >= 256 else n // 8 * 8) if rng.random() < 0.8 else n


def draw(rng):
    while True:
        op = rng.choice(["adapters", "adapters", "gated", "gated", "adamw"])
        if op == "adapters":
            mode = rng.choice(["forward", "train"])
            rows = rng.choice(["each", "runs"])
            S = _log_int(rng, 1, 256) if mode == "forward" and rows == "each" else _log_int(rng, 16, 8192)
            case = {"op": op, "mode": mode, "S": S, "I": _features(rng, 64, 8192), "O": _features(rng, 64, 8192),
                    "R": rng.choice([4, 8, 8, 12, 16, 16, 32, 64, 5 + rng.randrange(40)]), "count": _log_int(rng, 1, 64), "rows": rows,
                    "bare": rng.choice([0.0, 0.1, 0.5]), "dtype": rng.choice(["float32", "bfloat16", "bfloat16", "float16"])}
        elif op == "gated":
            mode = rng.choice(["forward", "forward", "train"])
            S = _log_int(rng, 1, 8192) if mode == "forward" else _log_int(rng, 64, 8192)
            case = {"op": op, "mode": mode, "S": S, "I": _features(rng, 64, 8192), "F": _features(rng, 64, 10240),
                    "act": rng.choice(["silu", "gelu"]), "dtype": rng.choice(["bfloat16", "bfloat16", "float16"])}
        else:
            kinds, groups = rng.randint(1, 6), []
            for _ in range(kinds):
                n = _log_int(rng, 16, 1 << 26)
                times = max(1, min(50, _log_int(rng, 1, 50), (1 << 26) // n))
                groups.append("%d*%d" % (n, times) if rng.random() < 0.5 else "%dx%d*%d" % (max(1, n // 16), 16, times))
            case = {"op": op, "sizes": ",".join(groups), "bits": rng.choice([8, 32]), "dtype": rng.choice(["float32", "float32", "bfloat16"])}
        w = work(case)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return case


def _sizes(case):
    """Values of each tensor of an AdamW case."""
    out = []
    for group in case["sizes"].split(","):
        shape, times = group.split("*")
        out += [math.prod(int(v) for v in shape.split("x"))] * int(times)
    return out


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    dtype = TYPES[case["dtype"]]
    if case["op"] == "adapters":
        S, I, O, R, n = case["S"], case["I"], case["O"], case["R"], case["count"]
        which = torch.randint(n, (S,), generator=gen, device="cuda", dtype=torch.int32)
        if case["rows"] == "runs":   # requests of uneven lengths, about four per adapter: each row has the draw of its request's first row
            first = torch.rand(S, generator=gen, device="cuda") < min(1.0, 4.0 * n / S)
            first[0] = True
            at = torch.cummax(torch.where(first, torch.arange(S, device="cuda"), 0), 0).values
            bare = (torch.rand(S, generator=gen, device="cuda") < case["bare"])[at]
            which = which[at]
        else:
            bare = torch.rand(S, generator=gen, device="cuda") < case["bare"]
        s = {"case": case, "x": normal(S, I, dtype=dtype), "y": normal(S, O, dtype=dtype), "which": torch.where(bare, -1, which).to(torch.int32),
             "A": normal(n, I, R, std=I ** -0.5, dtype=dtype), "B": normal(n, R, O, std=R ** -0.5, dtype=dtype),
             "scale": torch.rand(n, generator=gen, device="cuda") + 0.5}
        if case["mode"] == "train":
            s["dy"] = normal(S, O, dtype=dtype)
            for k in ("x", "y", "A", "B"):
                s[k].requires_grad_()
        return s
    if case["op"] == "gated":
        S, I, F = case["S"], case["I"], case["F"]
        s = {"case": case, "x": normal(S, I, dtype=dtype), "Wg": normal(I, F, std=I ** -0.5, dtype=dtype), "Wu": normal(I, F, std=I ** -0.5, dtype=dtype)}
        if case["mode"] == "train":
            s["dh"] = normal(S, F, dtype=dtype)
            for k in ("x", "Wg", "Wu"):
                s[k].requires_grad_()
        return s
    # the tensors lie in one buffer, each from a multiple of 256 values on
    sizes = _sizes(case)
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += (n + BLOCK - 1) // BLOCK * BLOCK
    held = torch.zeros(total, dtype=torch.bool, device="cuda")
    cut = lambda t, step=1: [t[a // step: a // step + (n + step - 1) // step] for a, n in zip(starts, sizes)]  # noqa: E731
    for part in cut(held):
        part.fill_(True)
    w = normal(total, std=0.05) * held
    s = {"case": case, "step": 100, "held": held, "g": (normal(total, std=1e-2, dtype=dtype) * held).to(dtype), "w": w, "master": case["dtype"] != "float32"}
    s["p"] = w.to(dtype) if s["master"] else w
    m, v = normal(total, std=1e-3) * held, normal(total, std=1e-2).square() * held
    if case["bits"] == 8:
        m, s["ms"] = _to_codes(m, True)
        v, s["vs"] = _to_codes(v, False)
    s["m"], s["v"] = m, v
    s["lists"] = {k: cut(s[k], BLOCK if k in ("ms", "vs") else 1) for k in ("p", "g", "w", "m", "v", "ms", "vs") if k in s}
    return s


def _to_codes(x, signed):
    """8-bit codes of blocks of 256 values and the largest magnitude of each: |x| = s (c / 127)**2 with x's sign, or (not signed) s (c / 254)**4,
    where a value above zero has a code of one at least."""
    b = x.view(-1, BLOCK)
    s = b.abs().amax(1, keepdim=True)
    q = (b.abs() / torch.where(s > 0, s, 1)).sqrt()
    if signed:
        return (torch.round(127 * q) * b.sign()).to(torch.int8).view(-1), s.float().view(-1)
    return torch.where(b > 0, torch.round(254 * q.sqrt()).clamp(min=1), 0).to(torch.uint8).view(-1), s.float().view(-1)


def _of_codes(c, s, signed, dtype):
    c = c.view(-1, BLOCK).to(dtype)
    q = (c / 127).square() * c.sign() if signed else (c / 254).square().square()
    return (q * s.view(-1, 1).to(dtype)).view(-1)


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    with torch.set_grad_enabled(own):   # (the plain forms write their gradients out)
        return (_run_adapters if op == "adapters" else _run_gated if op == "gated" else _run_adamw)(state)


def _run_adapters(s):
    train = s["case"]["mode"] == "train"
    if own:
        import paralleltnnlayers_b200 as P
        if not train:
            return P.dense_adapters(s["y"], s["x"], s["A"], s["B"], s["which"], s["scale"])
        out = P.DenseAdaptersFunction.apply(s["y"], s["x"], s["A"], s["B"], s["which"], s["scale"])
        return (out, *torch.autograd.grad(out, (s["x"], s["A"], s["B"]), s["dy"]))
    # all adapters side by side, and each row's own kept
    n, I, R = s["A"].shape
    dtype = s["x"].dtype
    x, A, B = s["x"].float(), s["A"].float().transpose(0, 1).reshape(I, n * R), s["B"].float().view(n * R, -1)
    mine = (s["which"].view(-1, 1) == torch.arange(n, device="cuda")) * s["scale"]
    mine = mine.repeat_interleave(R, 1)
    V = (x @ A) * mine
    out = (s["y"].float() + V @ B).to(dtype)
    if not train:
        return out
    dy = s["dy"].float()
    dV = (dy @ B.t()) * mine
    dA = (x.t() @ dV).view(I, n, R).transpose(0, 1).contiguous()
    return out, (dV @ A.t()).to(dtype), dA.to(dtype), (V.t() @ dy).view(n, R, -1).to(dtype)


def _run_gated(s):
    train, act, dtype = s["case"]["mode"] == "train", s["case"]["act"], s["x"].dtype
    if own:
        import paralleltnnlayers_b200 as P
        if not train:
            return P.dense_gated(s["x"], s["Wg"], s["Wu"], act)
        h = P.DenseGatedFunction.apply(s["x"], s["Wg"], s["Wu"], act)
        return (h, *torch.autograd.grad(h, (s["x"], s["Wg"], s["Wu"]), s["dh"]))
    x, Wg, Wu = s["x"].float(), s["Wg"].float(), s["Wu"].float()
    G, U = x @ Wg, x @ Wu
    gate = torch.sigmoid(G) if act == "silu" else 0.5 * (1 + torch.erf(G * 0.5 ** 0.5))
    h = (G * gate * U).to(dtype)
    if not train:
        return h
    slope = gate * (1 + G * (1 - gate)) if act == "silu" else gate + G * torch.exp(-0.5 * G * G) * (2 * math.pi) ** -0.5
    dh = s["dh"].float()
    dG, dU = dh * U * slope, dh * G * gate
    return h, (dG @ Wg.t() + dU @ Wu.t()).to(dtype), (x.t() @ dG).to(dtype), (x.t() @ dU).to(dtype)


def _run_adamw(s):
    s["step"] += 1
    t, (b1, b2), small = s["step"], BETAS, s["case"]["bits"] == 8
    if own:
        import paralleltnnlayers_b200 as P
        L = s["lists"]
        P.adamw_step(L["p"], L["g"], L["m"], L["v"], t, RATE, betas=BETAS, eps=EPS, weight_decay=DECAY, master=L["w"] if s["master"] else None,
                     scales=(L["ms"], L["vs"]) if small else None)
        m, v = P.adamw_moments(s["m"], s["v"], (s["ms"], s["vs"])) if small else (s["m"], s["v"])
    else:
        g, w = s["g"].float(), s["w"]
        m, v = (_of_codes(s["m"], s["ms"], True, torch.float32), _of_codes(s["v"], s["vs"], False, torch.float32)) if small else (s["m"], s["v"])
        m.mul_(b1).add_(g, alpha=1 - b1)
        v.mul_(b2).add_(g * g, alpha=1 - b2)
        w.mul_(1 - RATE * DECAY).sub_((m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS), alpha=RATE)
        if s["master"]:
            s["p"].copy_(w)
        if small:
            for k, x, signed in (("m", m, True), ("v", v, False)):
                codes, scale = _to_codes(x, signed)
                s[k].copy_(codes)
                s[k + "s"].copy_(scale)
            m, v = (_of_codes(s["m"], s["ms"], True, torch.float32).bfloat16(), _of_codes(s["v"], s["vs"], False, torch.float32).bfloat16())
    return (s["p"], s["w"], m, v) if s["master"] else (s["p"], m, v)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "adapters":
        S, I, O, R, n = case["S"], case["I"], case["O"], case["R"], case["count"]
        met = n * (1 - (1 - 1 / n) ** max(1.0, min(S, 4 * n) if case["rows"] == "runs" else S * (1 - case["bare"])))   # adapters that have a row
        fwd = 2 * S * (1 - case["bare"]) * R * (I + O)
        if case["mode"] == "forward":
            return {"bytes": size * (S * (I + 2 * O) + met * R * (I + O)), "flops": fwd}
        # x, y, dy and the adapters read, the output, dx and all adapters' gradients written
        return {"bytes": size * (S * (2 * I + 3 * O) + (met + n) * R * (I + O)), "flops": 3 * fwd}
    if case["op"] == "gated":
        S, I, F = case["S"], case["I"], case["F"]
        if case["mode"] == "forward":
            return {"bytes": size * (S * (I + F) + 2 * I * F), "flops": 4 * S * I * F}
        return {"bytes": size * (2 * S * (I + F) + 4 * I * F), "flops": 12 * S * I * F}
    n = sum(_sizes(case))
    moments = 2 * 2 * (1 + 4 / BLOCK) + 2 * 2 if case["bits"] == 8 else 16   # read and written; of 8 bits also given back as values
    return {"bytes": n * (moments + size + (2 + 8 if case["dtype"] != "float32" else 8)), "flops": 16 * n}


# ---- the definitions, in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d = lambda t: t.detach().double()  # noqa: E731
    if case["op"] == "adapters":
        train = case["mode"] == "train"
        out, dx = d(s["y"]), torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
        dA, dB = torch.zeros(s["A"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["B"].shape, dtype=torch.float64, device="cuda")
        for a in range(case["count"]):
            rows = (s["which"] == a).nonzero().view(-1)
            if not len(rows):
                continue
            x, A, B, c = d(s["x"])[rows], d(s["A"][a]), d(s["B"][a]), float(s["scale"][a])
            out[rows] += c * (x @ A) @ B
            if train:
                dy = d(s["dy"])[rows]
                dx[rows] = c * (dy @ B.t()) @ A.t()
                dA[a], dB[a] = c * x.t() @ (dy @ B.t()), c * (x @ A).t() @ dy
        return (out, dx, dA, dB) if train else out
    if case["op"] == "gated":
        if case["S"] * case["I"] * case["F"] > 2e11:
            return None
        x, Wg, Wu = d(s["x"]), d(s["Wg"]), d(s["Wu"])
        if case["mode"] == "train":
            for t in (x, Wg, Wu):
                t.requires_grad_()
        G = x @ Wg
        h = (torch.nn.functional.silu if case["act"] == "silu" else torch.nn.functional.gelu)(G) * (x @ Wu)
        if case["mode"] == "forward":
            return h
        return (h.detach(), *torch.autograd.grad(h, (x, Wg, Wu), d(s["dh"])))
    t, (b1, b2), small = s["step"] + 1, BETAS, case["bits"] == 8
    m = _of_codes(s["m"], s["ms"], True, torch.float64) if small else d(s["m"])
    v = _of_codes(s["v"], s["vs"], False, torch.float64) if small else d(s["v"])
    g, w = d(s["g"]), d(s["w"])
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
    w = w - RATE * DECAY * w - RATE * m / (1 - b1 ** t) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    if small:
        m, v = (_of_codes(*_to_codes(x, signed), signed, torch.float64) for x, signed in ((m, True), (v, False)))
    return (w, w, m, v) if s["master"] else (w, m, v)
