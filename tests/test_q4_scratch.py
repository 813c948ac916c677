"""What cx_q4_scratch and cx_q4_moe_scratch ask for covers every smaller call on the same
matrices.  No GPU: a call whose scratch is too small says what it needs before anything
touches a device."""
from __future__ import annotations

import ctypes as C
import re
import subprocess

import pytest

from constellation_amd._lib import BF16, CX_EINVAL, E4M3, FP16, lib
from test_q4_refusals import desc, held  # noqa: F401  (held is a fixture)
from test_q4_shapes import CSRC

SOURCE = r"""
#include "cx_shapes.h"
using namespace cx;
extern "C" {
int splits(int rt, int kt, int64_t rows, int mats, int item) { return q4_gemm_splits(rt, kt, rows, mats, item); }
int layer_dec(int cols, int inter) { return q4_layer_dec_rows(cols, inter); }
size_t dec_lds(int cols, int rows) { return q4_dec_lds(cols, rows); }
size_t sum_lds(int cols, int routes) { return q4_sum_lds(cols, routes); }
int routes(int k, int h, int i) { return q4_routes_ok(1, k, h, i, 0); }
int64_t part_rows(int rt, int kt, int64_t rows, int mats, int item) { return q4_gemm_part_rows(rt, kt, rows, mats, item); }
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("parts")
    (d / "parts.cc").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(d / "parts.cc"),
                    "-o", str(d / "parts.so")], check=True)
    L = C.CDLL(str(d / "parts.so"))
    L.part_rows.restype = C.c_int64
    L.dec_lds.restype = L.sum_lds.restype = C.c_size_t
    L.splits.argtypes = L.part_rows.argtypes = [C.c_int, C.c_int, C.c_int64, C.c_int, C.c_int]
    return L


SIZES = sorted({1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 66, 80, 96, 112, 127, 128, 129, 130, 256, 257, 448, 497, 498, 640, 641,
                1023, 1024, 1025, 1280, 1281, 1536, 2047, 2048, 2049, 2999, 3000, 4096, 6110, 6111, 6112, 8192, 20000, 1 << 17,
                *range(150, 1500, 53), *range(1500, 12000, 331)})


def needed(rc):
    """Bytes that a call refused for its scratch needs."""
    text = lib().cx_last_error().decode()
    m = re.search(r"scratch must be (\d+) bytes", text)
    assert rc == CX_EINVAL and m, (rc, text)
    return int(m.group(1))


def need_matmul(at, d, dt, rows, offsets):
    rc = lib().cx_q4_matmul(at, C.byref(d), at, dt, at if dt == E4M3 else None, rows, None, 1, at if offsets else None, rows, at, BF16, None, 0, None)
    # nothing needed: the call goes on to the device, which a fake context has not
    return needed(rc) if b"scratch" in lib().cx_last_error() else 0


@pytest.mark.parametrize("dt", [BF16, FP16, E4M3])
@pytest.mark.parametrize("mats,rows,cols", [(1, 18432, 7168), (1, 7168, 2048), (1, 4096, 7168), (1, 1000, 2048), (1, 512, 512), (1, 40, 1025),
                                            (1, 600, 1000), (1, 64, 9000), (8, 4096, 7168), (64, 1024, 2048), (64, 4096, 7168), (1024, 64, 264)])
def test_a_request_covers_smaller_products(held, mats, rows, cols, dt):
    _, at = held
    d = desc(at, mats, rows, cols)
    offsets = mats > 1
    most = last = 0
    for n in SIZES:
        lib().cx_ctx_sync(None, None)  # another error in the place of the last one
        asked = lib().cx_q4_scratch(C.byref(d), dt, n, n, int(offsets))
        most = max(most, need_matmul(at, d, dt, n, offsets))
        assert asked >= most and asked >= last, (n, asked, most, last)
        last = asked


@pytest.mark.parametrize("E,H,I,K,shared", [(64, 7168, 2048, 8, 0), (8, 1024, 704, 2, 1), (256, 7168, 2048, 8, 1), (4, 300, 70, 3, 0),
                                            (1, 4096, 14336, 1, 0), (2, 64, 33, 1, 1), (1024, 128, 64, 4, 0)])
def test_a_request_covers_smaller_layers(held, E, H, I, K, shared):
    _, at = held
    gu, dn = desc(at, E, 2 * I, H, 128, 1), desc(at, E, H, I, 128, 0)
    sg, sd = (C.byref(desc(at, 1, 2 * I, H, 128, 1)), C.byref(desc(at, 1, H, I, 128, 0))) if shared else (None, None)
    most = last = 0
    for n in SIZES:
        asked = lib().cx_q4_moe_scratch(C.byref(gu), C.byref(dn), shared, n, K)
        rc = lib().cx_q4_moe(at, C.byref(gu), C.byref(dn), sg, sd, at, BF16, n, at, at, K, at, BF16, None, None, 0, None)
        most = max(most, needed(rc))
        assert asked >= most and asked >= last, (n, asked, most, last)
        last = asked


def test_partial_rows_over_all_smaller_calls(rules):
    """The bound by intervals is no less than the largest need, row by row, and not much more."""
    for rt, kt in ((1, 2), (16, 9), (63, 16), (256, 56), (448, 16), (1152, 56), (5, 112)):
        for mats in (1, 3, 64):
            for item in (64, 128):
                most = 0
                for n in range(1, 9000):
                    s = rules.splits(rt, kt, n, mats, item)
                    if s > 1:
                        most = max(most, s * n)
                    if n % 97 == 0 or n in (1, 8999):
                        bound = rules.part_rows(rt, kt, n, mats, item)
                        assert most <= bound <= 16 * n, (rt, kt, mats, item, n, most, bound)
                for n in range(9001, 400000, 1117):  # nothing larger where the bound has stopped to look
                    s = rules.splits(rt, kt, n, mats, item)
                    assert s == 1 or s * n <= rules.part_rows(rt, kt, n, mats, item), (rt, kt, mats, item, n)


def test_both_planes_of_h_fit_the_lds(rules):
    for inter in [*range(1, 9000, 61), 2048, 4096, 7168, 8192, 8193]:
        rows = rules.layer_dec(max(64, inter), inter)
        assert 0 <= rows <= 4 and (rows > 0) == (inter <= 8192)
        assert rows == 0 or rules.dec_lds(inter, 2 * rows) <= 64 * 1024 - 256  # beside its static 144 bytes
        for k in (1, 9, 15, 16):
            if rules.routes(k, 7168, inter):
                # two planes of up to 4 column tiles, 16 sums and a weight per route
                assert rules.sum_lds(inter, k) == k * (2 * (min(-(-inter // 128), 4) * 256 + 64) + 68) <= 64 * 1024
    assert rules.routes(16, 7168, 2048) and not rules.routes(17, 7168, 2048) and not rules.routes(1, 7168, 2049)
