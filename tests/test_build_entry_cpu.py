"""build() makes the library from a tree that holds the product but not the C++ test programs' recipes."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("recipes", [(), ("build_cpp_test.py",)], ids=["no-tests", "older-tests"])
def test_build_without_test_programs(recipes, tmp_path):
    for part in ("ccglib_b200", "include", "oracle"):
        # copies keep their times, so a library that is up to date here is not compiled again
        shutil.copytree(os.path.join(ROOT, part), tmp_path / part,
                        ignore=shutil.ignore_patterns("obj", "trace", "__pycache__"))
    shutil.copy2(os.path.join(ROOT, "__graft_entry__.py"), tmp_path)
    if recipes:
        shutil.copytree(os.path.join(ROOT, "tests", "cpp"), tmp_path / "tests" / "cpp",
                        ignore=shutil.ignore_patterns("build_operators_test.py", "test_operators*", "bin"))
    res = subprocess.run([sys.executable, "-c", "import __graft_entry__ as g; g.build()"], cwd=tmp_path,
                         capture_output=True, text=True, timeout=1200,
                         env={k: v for k, v in os.environ.items() if k not in ("PYTHONPATH", "CCGLIB_B200_LIB")})
    assert res.returncode == 0, res.stdout + res.stderr
    assert str(tmp_path / "ccglib_b200" / "lib" / "libccglib_b200.so") in res.stdout
