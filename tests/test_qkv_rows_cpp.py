"""The row operators and the block-scaled cache from C++: tests/cpp/test_qkv_rows.cpp, compiled with g++ against the shipped
headers and run on the GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "cpp", "test_qkv_rows.cpp")
EXE = os.path.join(ROOT, "tests", "cpp", "test_qkv_rows")
LIBDIR = os.path.join(ROOT, "paged_attention_b200")


def build():
    headers = [os.path.join(LIBDIR, "include", "decode", f) for f in os.listdir(os.path.join(LIBDIR, "include", "decode"))]
    deps = [SRC, os.path.join(ROOT, "include", "pd_b200.h"), os.path.join(LIBDIR, "libpd_b200.so")] + headers
    if os.path.exists(EXE) and all(os.path.getmtime(EXE) >= os.path.getmtime(d) for d in deps):
        return
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.check_call(["g++", "-std=c++20", "-O2", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(LIBDIR, "include"),
                           "-I", os.path.join(cuda, "include"), SRC, "-o", EXE, "-L", LIBDIR, "-lpd_b200",
                           "-L", os.path.join(cuda, "lib64"), "-lcudart", "-Wl,-rpath," + LIBDIR])


def test_headers_compile(pa):
    build()
    assert os.path.exists(EXE)


@pytest.mark.gpu
def test_cpp_caller_runs(torch_cuda, pa):
    build()
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "all checks passed" in r.stdout, r.stdout[-3000:] + r.stderr[-2000:]
