"""How many clusters a device holds: asked once per kernel, device and size (csrc/raise_limit.hpp, csrc/cluster_util.cuh)."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "paralleltnnlayers_b200", "csrc")


def test_a_count_of_zero_is_an_answer(tmp_path):
    exe = str(tmp_path / "test_count")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-pthread", "-o", exe, os.path.join(ROOT, "tests", "cpp", "test_count.cpp"), "-I", CSRC])
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout


def test_the_counts_are_those_of_the_device():
    """Every kernel that asks says for which device, and the answers are held by device."""
    helper = open(os.path.join(CSRC, "cluster_util.cuh")).read()
    assert "remembered_count(counts.of[dev][c]" in helper
    for name in ("adapters.cu", "gated.cu"):
        source = open(os.path.join(CSRC, name)).read()
        calls = re.findall(r"resident_clusters\(([^()]*)\)", source)
        assert calls and all(c.split(", ")[3] == "dev" for c in calls)
        assert source.count("cudaGetDevice(&dev)") == len(calls)
