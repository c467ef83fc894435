"""The C++ host's row operators (host/arrow_gpu.hpp, tests/cpp/test_rows.cpp): the program builds against the C ABI, fails loudly without a GPU and passes
on one."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "cpp", "test_rows.cpp")
EXE = os.path.join(ROOT, "tests", "cpp", "build", "test_rows")
LIBDIR = os.path.join(ROOT, "arrow_gpu_amd", "lib")


def build():
    os.makedirs(os.path.dirname(EXE), exist_ok=True)
    deps = [SRC, os.path.join(ROOT, "host", "arrow_gpu.hpp"), os.path.join(ROOT, "include", "arrow_gpu.h")]
    if os.path.exists(EXE) and all(os.path.getmtime(EXE) >= os.path.getmtime(d) for d in deps):
        return
    cmd = ["/opt/rocm/bin/hipcc", "-std=c++17", "-O1", "-Wall", "-x", "c++", SRC, "-o", EXE, f"-L{LIBDIR}", "-larrow_gpu_hip", "-Wl,-rpath," + LIBDIR]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]


def test_cpp_rows_compile_and_fail_loudly_without_gpu():
    import torch

    build()
    if torch.cuda.device_count() > 0:
        pytest.skip("a GPU is present; the run is covered by the gpu-marked test")
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=120)
    assert r.returncode == 2 and "no device" in r.stdout


VIEWS = os.path.join(ROOT, "tests", "cpp", "test_rows_views.cpp")


def build_views():
    exe = os.path.join(ROOT, "tests", "cpp", "build", "test_rows_views")
    os.makedirs(os.path.dirname(exe), exist_ok=True)
    deps = [VIEWS, os.path.join(ROOT, "host", "arrow_gpu.hpp"), os.path.join(ROOT, "include", "arrow_gpu.h")]
    if not os.path.exists(exe) or any(os.path.getmtime(exe) < os.path.getmtime(d) for d in deps):
        cmd = ["/opt/rocm/bin/hipcc", "-std=c++17", "-O1", "-Wall", "-x", "c++", VIEWS, "-o", exe, f"-L{LIBDIR}", "-larrow_gpu_hip", "-Wl,-rpath," + LIBDIR]
        r = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stderr[-3000:]
    return exe


def test_cpp_row_views_compile_and_fail_loudly_without_gpu():
    import torch

    exe = build_views()
    if torch.cuda.device_count() > 0:
        pytest.skip("a GPU is present; the run is covered by the gpu-marked test")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 2 and "no device" in r.stdout


@pytest.mark.gpu
def test_cpp_row_views_on_gpu():
    r = subprocess.run([build_views()], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "ALL OK" in r.stdout, r.stdout[-3000:] + r.stderr[-2000:]


@pytest.mark.gpu
def test_cpp_rows_on_gpu():
    build()
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "ALL OK" in r.stdout, r.stdout[-3000:] + r.stderr[-2000:]
