"""CPU suite of the attention calls: refusals of arguments at their ends (tests/test_attend_host.py has the plain ones)."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from test_attend_host import args, at  # noqa: F401  (at: the fixture)


@pytest.mark.parametrize("scale", [5e-324, 1e-300, 1e-50, 1e-46, 1e-39, 2.0 ** -126 * (1 - 2.0 ** -52)])
def test_scales_that_a_float_does_not_hold(gpx, at, scale):  # noqa: F811
    for which in range(3):
        assert at._entry(which)(args(at, scale=scale)) == gpx.E_BAD_ARG
        assert "scale" in gpx.lib().gpx_last_error().decode()


@pytest.mark.parametrize("scale", [2.0 ** -126, 1e-30, 1.0, 2.0 ** 127])
def test_scales_that_a_float_holds(gpx, at, scale):  # noqa: F811
    n = C.c_size_t(0)
    for which in range(3):
        assert at._entry(3)(args(at, scale=scale), which, C.byref(n)) == gpx.OK


def test_rows_that_overlap(tmp_path):
    """The rule by which outputs are refused, built by itself (csrc/gpx_overlap.hpp) and held to the list of all rows."""
    if not shutil.which("g++"):
        pytest.skip("no g++")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = str(tmp_path / "rows_overlap")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(root, "gaussian-object-modelling_amd", "csrc"),
                    os.path.join(root, "tests", "cpp", "rows_overlap.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
