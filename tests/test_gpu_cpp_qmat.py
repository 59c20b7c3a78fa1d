"""RowQuantizer and QuantizedMatrix of the C++ facade (vq_b200/cpp/vq.hpp)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBDIR = os.path.join(ROOT, "vq_b200")


def _build(out):
    subprocess.check_call(["/usr/bin/g++", "-std=c++17", "-O1", "-Wall", "-Wno-format-extra-args", "-o", out, os.path.join(ROOT, "tests", "cpp", "test_facade_qmat.cpp"), "-L" + LIBDIR, "-lvqb",
                           "-Wl,-rpath," + LIBDIR])


def test_compiles_and_links(tmp_path):
    _build(os.path.join(str(tmp_path), "test_facade_qmat"))


@pytest.mark.gpu
def test_codes_and_products_through_the_cpp_facade(tmp_path):
    exe = os.path.join(str(tmp_path), "test_facade_qmat")
    _build(exe)
    res = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=120)
    out = res.stdout.decode()
    assert res.returncode == 0 and "all checks of codes and products passed" in out, out[-2000:]
