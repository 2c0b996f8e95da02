"""Builds tests/cpp/bin/test_operators: the C++ classes of the quantiser, the scaled GEMM and the
orthogonalisation through the stand-in cudawrappers header, linked against the CUDA library."""
from __future__ import annotations

import importlib.util
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
BIN = os.path.join(HERE, "bin", "test_operators")
CUDA_HOME = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def build() -> str:
    spec = importlib.util.spec_from_file_location(
        "ccglib_b200_build_recipe", os.path.join(ROOT, "ccglib_b200", "build.py"))
    lib_build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(lib_build)
    lib = lib_build.build()
    src = os.path.join(HERE, "test_operators.cpp")
    deps = [src, lib, os.path.join(ROOT, "include", "ccglib", "b200_api.hpp"),
            os.path.join(HERE, "shim", "cudawrappers", "cu.hpp"), __file__]
    if os.path.exists(BIN) and all(os.path.getmtime(d) <= os.path.getmtime(BIN) for d in deps):
        return BIN
    os.makedirs(os.path.dirname(BIN), exist_ok=True)
    lib_dir = os.path.dirname(lib)
    driver_dir = next(d for d in ("/usr/lib/x86_64-linux-gnu",
                                  os.path.join(CUDA_HOME, "lib64", "stubs"))
                      if os.path.exists(os.path.join(d, "libcuda.so")))
    subprocess.run(
        ["g++", "-std=c++17", "-O2", "-Wall", "-I", os.path.join(ROOT, "include"),
         "-I", os.path.join(HERE, "shim"), "-I", os.path.join(CUDA_HOME, "include"), src, "-o", BIN,
         "-L", lib_dir, "-lccglib_b200", "-L", driver_dir, "-lcuda",
         "-Wl,-rpath,$ORIGIN/" + os.path.relpath(lib_dir, os.path.dirname(BIN))], check=True)
    return BIN


if __name__ == "__main__":
    print(build())
