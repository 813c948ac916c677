"""The combine's gradient: which form the sizes take, by the rule of csrc/cx_shapes.h on the host,
at the sizes where both were measured."""
from __future__ import annotations

import ctypes as C
import subprocess

import pytest

from test_q4_shapes import CSRC

SOURCE = r"""
#include "cx_shapes.h"
extern "C" int routes(int64_t pairs, int vec) { return cx::combine_grad_routes(pairs, vec != 0); }
"""


@pytest.fixture(scope="module")
def routes(tmp_path_factory):
    d = tmp_path_factory.mktemp("grad")
    (d / "grad.cc").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(d / "grad.cc"),
                    "-o", str(d / "grad.so")], check=True)
    L = C.CDLL(str(d / "grad.so"))
    L.routes.argtypes = [C.c_int64, C.c_int]
    return L.routes


@pytest.mark.parametrize("T,K,vec,faster", [(128, 8, 1, 1), (384, 8, 1, 1), (640, 8, 1, 8), (2048, 8, 1, 8), (384, 16, 1, 8), (1024, 2, 1, 1),
                                            (128, 6, 0, 1), (256, 6, 0, 1), (320, 6, 0, 8), (384, 6, 0, 8), (509, 6, 0, 8), (96, 16, 0, 1),
                                            (128, 16, 0, 8), (1 << 24, 64, 1, 8)])
def test_the_faster_form(routes, T, K, vec, faster):
    assert routes(T * K, vec) == faster
