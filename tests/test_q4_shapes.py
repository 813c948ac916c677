"""The rules of csrc/cx_shapes.h for work items, staging and partial sums of the
4-bit products, over ranges of sizes on the host."""
from __future__ import annotations

import ctypes as C
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "constellation_amd" / "csrc"

SOURCE = r"""
#include "cx_shapes.h"
using namespace cx;
extern "C" {
int share(int n, int rows) { return q4_item_share(n, rows); }
int64_t most(int64_t rows, int mats, int item) { return q4_max_items(rows, mats, item); }
int item(int64_t rows, int mats, int n, int cols, int two) { return q4_item_rows(rows, mats, n, cols, two); }
int layer(int64_t rows, int mats, int cols) { return q4_layer_rows(rows, mats, cols); }
int dec_rows(int cols) { return q4_dec_rows(cols); }
size_t dec_lds(int cols, int rows) { return q4_dec_lds(cols, rows); }
int routes(int t, int k, int h, int i, int sh) { return q4_routes_ok(t, k, h, i, sh); }
size_t sum_lds(int cols, int routes) { return q4_sum_lds(cols, routes); }
int splits(int rt, int kt, int64_t rows, int mats, int item) { return q4_gemm_splits(rt, kt, rows, mats, item); }
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.cc").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(d / "rules.cc"), "-o", str(d / "rules.so")], check=True)
    L = C.CDLL(str(d / "rules.so"))
    L.most.restype = C.c_int64
    L.dec_lds.restype = L.sum_lds.restype = C.c_size_t
    L.most.argtypes = [C.c_int64, C.c_int, C.c_int]
    L.item.argtypes = [C.c_int64, C.c_int, C.c_int, C.c_int, C.c_int]
    L.layer.argtypes = [C.c_int64, C.c_int, C.c_int]
    L.splits.argtypes = [C.c_int, C.c_int, C.c_int64, C.c_int, C.c_int]
    return L


@pytest.mark.parametrize("cap", [1, 3, 4, 16, 64, 128])
def test_items_cover_the_rows_once(rules, cap):
    """n items of the share, the last with the rest: none empty, none above the cap."""
    for rows in list(range(1, 40 * cap, 1 if cap < 64 else 7)) + [97 * cap - 1, 97 * cap, 97 * cap + 1, 1 << 20]:
        n = -(-rows // cap)
        share = rules.share(n, rows)
        assert 1 <= share <= cap, (rows, n, share)
        assert 0 < rows - (n - 1) * share <= share, (rows, n, share)


@pytest.mark.parametrize("cap", [4, 16, 64, 128])
def test_item_bound_holds_for_any_deal(rules, cap):
    """Rows dealt to matrices one each, all to one, evenly, or with rows behind the last."""
    for mats in (1, 2, 7, 64, 1024):
        for rows in (1, 3, 16, 17, 200, 4099):
            for deal in ([rows], [1] * min(mats, rows), [rows // mats + (i < rows % mats) for i in range(mats)],
                         [cap + 1] * min(mats, rows // (cap + 1))):
                if len(deal) > mats or sum(deal) > rows:
                    continue
                n = sum(-(-r // cap) for r in deal) + -(-(rows - sum(deal)) // cap)
                assert 1 + n <= rules.most(rows, mats, cap), (mats, rows, deal[:3])


def test_staged_rows_fit_the_lds(rules):
    for cols in list(range(1, 9000, 13)) + [7168, 8192, 8193, 65536]:
        rows = rules.dec_rows(cols)
        assert 0 <= rows <= 4 and (rows == 0) == (cols > 8192)
        if rows:
            assert rules.dec_lds(cols, rows) <= 64 * 1024 - 256
            assert rules.item(1, 1, 64, cols, 0) == (rows if cols % 8 else 16) and rules.item(8, 8, 64, cols, 0) == rows
            assert rules.layer(1, 1, cols) == rules.layer(rows, 1, cols) == rules.layer(64, 64, cols) == rows
        assert rules.layer(65, 64, cols) == 128 and rules.item(16, 1, 64, cols, 0) == (16 if cols % 8 == 0 or cols <= 1024 else 128)
        assert rules.item(16, 1, 1 << 24, 4096, 0) == 16 and rules.item(17, 1, 1 << 24, 4096, 0) == 128
        assert rules.item(10 ** 8, 1, 64, cols, 0) == 128 and rules.item(10 ** 8, 1, 64, cols, 1) == 64
    for inter in range(1, 2100, 17):
        for k in (1, 2, 8, 9, 15, 16, 17, 64):
            if rules.routes(1, k, 7168, inter, 0):
                assert k <= 16 and inter <= 2048 and rules.sum_lds(inter, k) <= 64 * 1024
            assert not rules.routes(2, k, 7168, inter, 0)
    assert rules.routes(1, 8, 7168, 2048, 1)


def test_stacks_by_their_size(rules):
    """Few rows per matrix: by launches where the codes are few, and without overflow where they are many."""
    assert rules.item(64, 8, 512, 1024, 0) == 16 and rules.item(2000, 8, 512, 1024, 0) == 128
    assert rules.item(1024, 1, 512, 512, 1) == 16 and rules.item(2048, 1, 512, 512, 1) == 64 and rules.item(2048, 1, 512, 512, 0) == 16
    assert rules.item(600, 64, 4096, 7168, 0) == 128 and rules.item(600, 64, 4096, 7168, 1) == 64
    assert rules.item(5000, 1024, 1 << 24, 1 << 24, 0) == 128


def test_ranges_of_the_columns(rules):
    """1 to 16 ranges of at least two column tiles, one where workgroups are plenty."""
    for rt in (1, 16, 256, 448):
        for kt in (1, 2, 16, 56, 64):
            for rows in (17, 64, 300, 4096, 40000):
                s = rules.splits(rt, kt, rows, 1, 128)
                assert s in (1, 2, 4, 8, 16) and (s == 1 or kt // s >= 2)
    assert rules.splits(256, 56, 32768, 64, 128) == 1 and rules.splits(256, 56, 32, 1, 128) > 1
