"""The norm, append and tree entry points from C (tests/c/step_check.c): structure
layouts equal to the ctypes mirrors', argument errors, empty calls. CPU only."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from dsv4_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def test_structures_and_errors_from_c(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None or not os.path.exists(_lib.LIB_PATH):
        pytest.skip("gcc or libsas.so missing")
    exe = str(tmp_path / "step_check")
    libdir = os.path.dirname(_lib.LIB_PATH)
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"),
                    os.path.join(HERE, "c", "step_check.c"), "-o", exe, "-L", libdir, "-lsas", f"-Wl,-rpath,{libdir}",
                    "-Wl,--allow-shlib-undefined"], check=True)
    out = dict(line.split(" ", 1) for line in subprocess.run([exe], check=True, capture_output=True,
                                                             text=True).stdout.splitlines())
    for name, last in (("SasNormRopeArgs", "reserved"), ("SasNormRopeBwdArgs", "dkv_out_stride_t"),
                       ("SasCacheAppendArgs", "reserved"), ("SasFwdTreeArgs", "tree_words")):
        t = getattr(_lib, name)
        assert out[name] == f"{_lib.C.sizeof(t)} {getattr(t, last).offset}", name
    assert out["errors"].split() == [str(_lib.SAS_EINVAL)] * 5 and out["message"] == "1"
    assert out["empty"] == "0 0 0"
