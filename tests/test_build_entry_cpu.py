"""build() makes the library from a tree that holds the product but not the C++ test programs' recipes, and
where those programs cannot be built."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _tree(tmp_path, with_tests):
    for part in ("ccglib_b200", "include", "oracle"):
        # copies keep their times, so a library that is up to date here is not compiled again
        shutil.copytree(os.path.join(ROOT, part), tmp_path / part,
                        ignore=shutil.ignore_patterns("obj", "trace", "__pycache__"))
    shutil.copy2(os.path.join(ROOT, "__graft_entry__.py"), tmp_path)
    if with_tests:
        shutil.copytree(os.path.join(ROOT, "tests", "cpp"), tmp_path / "tests" / "cpp",
                        ignore=shutil.ignore_patterns("bin"))


def _build(tmp_path):
    res = subprocess.run([sys.executable, "-c", "import __graft_entry__ as g; g.build()"], cwd=tmp_path,
                         capture_output=True, text=True, timeout=1200,
                         env={k: v for k, v in os.environ.items() if k not in ("PYTHONPATH", "CCGLIB_B200_LIB")})
    assert res.returncode == 0, res.stdout + res.stderr
    assert str(tmp_path / "ccglib_b200" / "lib" / "libccglib_b200.so") in res.stdout
    return res


@pytest.mark.parametrize("recipes", [(), ("build_cpp_test.py",)], ids=["no-tests", "older-tests"])
def test_build_without_test_programs(recipes, tmp_path):
    _tree(tmp_path, bool(recipes))
    if recipes:
        for name in ("build_operators_test.py", "test_operators.cpp"):
            os.unlink(tmp_path / "tests" / "cpp" / name)
    _build(tmp_path)


def test_build_where_a_test_program_cannot_be_built(tmp_path):
    _tree(tmp_path, True)
    with open(tmp_path / "tests" / "cpp" / "test_operators.cpp", "a") as f:
        f.write("#error cannot be built here\n")
    res = _build(tmp_path)
    assert "not built: build of tests/cpp/build_operators_test.py" in res.stderr
    assert "cannot be built here" in res.stderr and "built %s" % (tmp_path / "tests" / "cpp" / "bin" / "test_api") in res.stdout
