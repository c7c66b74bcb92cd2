"""host/q4t/model/verify_head.h: compiles as host C++ (CPU test) and runs end to end on a GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXE = os.path.join(ROOT, "tests", "cpp", "verify_test")


def _build():
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    pkg = os.path.join(ROOT, "qwen4-thor_b200")
    cmd = ["g++", "-std=c++20", "-O1", "-Wall", f"-I{cuda}/include", f"-I{ROOT}/include", f"-I{pkg}/host",
           os.path.join(ROOT, "tests", "cpp", "verify_test.cpp"), "-o", EXE,
           f"-L{pkg}", "-lq4t_moe_b200", f"-Wl,-rpath,{pkg}", f"-L{cuda}/lib64", "-lcudart"]
    return subprocess.run(cmd, capture_output=True, text=True)


def test_compiles_and_links(q4t):
    if not os.path.exists(q4t.LIB_PATH):
        pytest.skip("library not built")
    r = _build()
    assert r.returncode == 0, r.stderr


@pytest.mark.gpu
def test_runs_on_gpu(q4t, gpu_lib):
    r = _build()
    assert r.returncode == 0, r.stderr
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "verify_test PASS" in r.stdout, r.stdout + r.stderr


def test_refusals_come_before_anything_is_enqueued(q4t, tmp_path):
    if not os.path.exists(q4t.LIB_PATH):
        pytest.skip("library not built")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    pkg = os.path.join(ROOT, "qwen4-thor_b200")
    exe = str(tmp_path / "verify_refusals")
    r = subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Werror", f"-I{cuda}/include", f"-I{ROOT}/include", f"-I{pkg}/host",
                        os.path.join(ROOT, "tests", "cpp", "verify_refusals.cpp"), "-o", exe, f"-L{pkg}", "-lq4t_moe_b200",
                        f"-Wl,-rpath,{pkg}", f"-L{cuda}/lib64", "-lcudart"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "verify_refusals PASS" in r.stdout, r.stdout + r.stderr
