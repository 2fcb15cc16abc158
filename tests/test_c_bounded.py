"""The entry points for bounded caches from C (tests/c/bounded_check.c): structure layouts
equal to the ctypes mirrors', argument errors, an empty call. CPU only."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from dsv4_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def test_bounded_structures_and_errors_from_c(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None or not os.path.exists(_lib.LIB_PATH):
        pytest.skip("gcc or libsas.so missing")
    exe = str(tmp_path / "bounded_check")
    libdir = os.path.dirname(_lib.LIB_PATH)
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"),
                    os.path.join(HERE, "c", "bounded_check.c"), "-o", exe, "-L", libdir, "-lsas", f"-Wl,-rpath,{libdir}",
                    "-Wl,--allow-shlib-undefined"], check=True)
    out = dict(line.split(" ", 1) for line in subprocess.run([exe], check=True, capture_output=True,
                                                             text=True).stdout.splitlines())
    for name, last in (("SasFwdFirstArgs", "ori_first"), ("SasBwdFirstArgs", "ori_first"),
                       ("SasRowWeightsArgs", "cmp_rows"), ("SasCacheEvictArgs", "keep_recent")):
        t = getattr(_lib, name)
        assert out[name] == f"{_lib.C.sizeof(t)} {getattr(t, last).offset}", name
    assert out["null"].split() == [str(_lib.SAS_EINVAL)] * 5
    assert out["errors"].split() == [str(_lib.SAS_EINVAL)] * 4 and out["message"] == "1"
    assert out["empty"] == "0"
