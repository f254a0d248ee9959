"""The choice of how many workgroups share a walk of the attention kernels for training (no GPU needed)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_shared_walks_fit_a_launch(tmp_path):
    """No choice starts more threads than a launch takes, shares a grid that fills the card, or keeps more sums than that needs."""
    exe = tmp_path / "share"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", os.path.join(ROOT, "tests", "cpp", "test_attn_share.cpp"), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    print(r.stdout[:4000])
    assert r.returncode == 0 and "ALL PASSED" in r.stdout
