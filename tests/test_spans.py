"""What an AdamW step writes may not meet anything else that it is given."""
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_spans_that_meet(tmp_path):
    exe = str(tmp_path / "test_spans")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-o", exe, os.path.join(ROOT, "tests", "cpp", "test_spans.cpp"),
                           "-I", os.path.join(ROOT, "paralleltnnlayers_b200", "csrc")])
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout


def _args(small, half):
    """Two tensors of 600 values in buffers with room beside them."""
    types = {"p": torch.bfloat16 if half else torch.float32, "g": torch.float32, "m": torch.int8 if small else torch.float32,
             "v": torch.uint8 if small else torch.float32, "w": torch.float32}
    t = {k: [torch.zeros(1024, dtype=d, device="cuda") for _ in range(2)] for k, d in types.items()}
    t["ms"], t["vs"] = ([torch.zeros(8, device="cuda") for _ in range(2)] for _ in range(2))
    return t


def _step(t, small, half, cut=lambda k, i, b: b[:3] if k in ("ms", "vs") else b[:600]):
    import paralleltnnlayers_b200 as P
    c = {k: [cut(k, i, b) for i, b in enumerate(bs)] for k, bs in t.items()}
    P.adamw_step(c["p"], c["g"], c["m"], c["v"], 1, 0.1, master=c["w"] if half else None, scales=(c["ms"], c["vs"]) if small else None)


@pytest.mark.gpu
@pytest.mark.parametrize("small", [False, True], ids=["32", "8"])
@pytest.mark.parametrize("half", [False, True], ids=["float32", "bfloat16"])
def test_a_tensor_that_meets_another_is_refused(small, half):
    kinds = ["p", "m", "v"] + (["ms", "vs"] if small else []) + (["w"] if half else [])
    for k in kinds:   # the same tensor twice, and a view that begins inside it
        n, off = (3, 2) if k in ("ms", "vs") else (600, 300)
        for at in (0, off):
            t = _args(small, half)
            t[k][1] = t[k][0]
            with pytest.raises(ValueError, match="occurs twice"):
                _step(t, small, half, lambda q, i, b: b[at * i:at * i + n] if q == k else b[:3] if q in ("ms", "vs") else b[:600])
            assert not any(bool(b.any()) for bs in t.values() for b in bs)
    if not small:   # a gradient that is a moment, and a moment that is the next parameter
        t = _args(small, half)
        t["g"][1] = t["m"][0]
        with pytest.raises(ValueError, match="occurs twice"):
            _step(t, small, half)
        if not half:
            t = _args(small, half)
            t["p"][1] = t["v"][0]
            with pytest.raises(ValueError, match="occurs twice"):
                _step(t, small, half)


@pytest.mark.gpu
@pytest.mark.parametrize("small", [False, True], ids=["32", "8"])
@pytest.mark.parametrize("half", [False, True], ids=["float32", "bfloat16"])
def test_tensors_beside_one_another_are_taken(small, half):
    """Views that end where the next begins, in any order, and one gradient for two parameters."""
    t = _args(small, half)
    for k, bs in t.items():
        n = 3 if k in ("ms", "vs") else 500
        t[k] = [bs[0][n:2 * n], bs[0][:n]]
    t["g"] = [t["g"][0].fill_(1.0)] * 2
    _step(t, small, half, lambda q, i, b: b[:2] if q in ("ms", "vs") else b)
    assert all(bool((p < 0).all()) for p in t["p"])
