"""The C++ host mirror's 8-bit caches, windows and rotary positions with several axes (tests/cpp/cache8_cases.cpp)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _build(folder):
    from floneum_b200 import build
    lib = build.build()
    exe = str(folder / "cache8_cases")
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", "cache8_cases.cpp"), "-o", exe,
                    "-L", os.path.dirname(lib), "-lfusor_cuda", "-Wl,-rpath," + os.path.dirname(lib)], check=True)
    return exe


def test_it_compiles_and_its_host_checks_pass(tmp_path):
    res = subprocess.run([_build(tmp_path), "--no-gpu"], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr


@pytest.mark.gpu
def test_it_passes_on_a_gpu(tmp_path):
    res = subprocess.run([_build(tmp_path)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "all cache cases passed" in res.stdout
