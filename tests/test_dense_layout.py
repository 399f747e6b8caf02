"""How a dense layer's products are shared out (tests/cpp/test_dense_layout.cpp)."""
import os
import subprocess

from conftest import ROOT


def test_no_row_of_sums_behind_the_work(tmp_path):
    exe = str(tmp_path / "test_dense_layout")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "neutronbench_amd", "csrc"), "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "cpp", "test_dense_layout.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
