"""How the products of a program's own experts are cut, by the rules of csrc/cx_shapes.h on the host: items cover the rows
once, launches hold them, and the GPU tests' sizes reach every kernel."""
from __future__ import annotations

import ctypes as C
import subprocess
from pathlib import Path

import pytest

from test_gpu_matmul import GRADS, ONE, STACK
from test_gpu_matmul_large import FORWARD
from test_gpu_matmul_large import GRADS as LARGE_GRADS

CSRC = Path(__file__).resolve().parent.parent / "constellation_amd" / "csrc"

SOURCE = r"""
#include "cx_shapes.h"
using namespace cx;
extern "C" {
int share(int n, int rows) { return mm_share(n, rows); }
int64_t items(int64_t rows, int mats, int stack, int item) { return mm_items(rows, mats, stack, item); }
int64_t form(int64_t rows, int mats, int stack, int64_t out, int64_t depth, int few) {
    const MmForm f = mm_form(rows, mats, stack, out, depth, few);
    return ((int64_t)f.kind << 48) | ((int64_t)f.item_rows << 32) | ((int64_t)f.splits << 16) | f.tiles;
}
int grid_ok(int64_t rows, int mats, int n, int k) { return mm_grid_ok(rows, mats, n, k); }
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.cc").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(d / "rules.cc"), "-o", str(d / "rules.so")],
                   check=True)
    L = C.CDLL(str(d / "rules.so"))
    L.items.restype = L.form.restype = C.c_int64
    L.items.argtypes = [C.c_int64, C.c_int, C.c_int, C.c_int]
    L.form.argtypes = [C.c_int64, C.c_int, C.c_int, C.c_int64, C.c_int64, C.c_int]
    L.grid_ok.argtypes = [C.c_int64, C.c_int, C.c_int, C.c_int]
    return L


def form(rules, P, E, out, depth, few):
    v = rules.form(P, max(1, E), int(E > 0), out, depth, int(few))
    return v >> 48, v >> 32 & 0xFFFF, v >> 16 & 0xFFFF, v & 0xFFFF


@pytest.mark.parametrize("cap", [16, 32, 64, 96, 128, 192, 256])
def test_items_cover_the_rows_once(rules, cap):
    for rows in list(range(1, 12 * cap, 1 if cap < 64 else 5)) + [97 * cap - 1, 97 * cap, 97 * cap + 1, 1 << 20]:
        n = -(-rows // cap)
        share = rules.share(n, rows)
        assert 1 <= share <= cap and 0 < rows - (n - 1) * share <= share, (rows, n, share)


@pytest.mark.parametrize("cap", [16, 64, 256])
def test_item_bound_holds_for_any_deal(rules, cap):
    """Rows dealt to matrices one each, all to one, evenly, or with rows behind the last."""
    for mats in (1, 2, 7, 64, 1024):
        for rows in (1, 3, 16, 17, 200, 4099):
            deals = [[1] * min(mats, rows), [rows], [rows // mats] * mats, [max(1, rows // mats - 1)] * min(mats, rows)]
            for deal in deals:
                if sum(deal) > rows:
                    continue
                rest = rows - sum(deal)
                n = sum(-(-r // cap) for r in deal) + -(-rest // cap)
                assert n <= rules.items(rows, mats, 1, cap), (mats, rows, cap, deal[:4])


def test_forms_are_what_the_kernels_take(rules):
    for P in (1, 2, 15, 16, 17, 40, 64, 65, 100, 333, 1000, 4096, 20000, 1 << 20, 1 << 24):
        for E in (0, 1, 8, 64, 1024):
            for out in (1, 30, 256, 4096, 20000):
                for depth in (2, 100, 4096, 14336):
                    for few in (False, True):
                        kind, rows, splits, tiles = form(rules, P, E, out, depth, few)
                        assert kind in (0, 1, 2) and (few or kind > 0)
                        if kind == 0:
                            assert rows == 16 and tiles in (1, 2) and splits in (1, 2, 4, 8)
                        else:
                            unit = 64 if kind == 2 else 32
                            assert rows % unit == 0 and 1 <= rows // unit <= 4 and 1 <= splits <= 16
                            assert splits == 1 or P * -(-out // 1024) < 1 << 24  # workgroups of the sums
                        assert rules.grid_ok(P, max(1, E), out, max(1, depth // 2)) or P * out > 1 << 30 or P >= 1 << 20 or E == 1024


def test_tests_reach_every_kernel(rules):
    """Of the GPU tests' sizes: each kernel of the forward products, with and without partial sums, at each count of tiles that
    an item may have (by its rows), and both kernels of the gradient at x."""
    seen = set()
    for sizes in (ONE, STACK, FORWARD):
        for s in sizes:
            P, E, N, K = s if len(s) == 4 else (s[0], 0, s[1], s[2])
            kind, rows, splits, _ = form(rules, P, E, N, K * 2, True)
            seen.add((kind, splits > 1))
    assert {(0, False), (0, True), (1, False), (1, True), (2, False), (2, True)} <= seen, seen
    seen = set()
    for P, E, N, K in [*GRADS, *LARGE_GRADS]:
        kind, rows, splits, _ = form(rules, P, E, K, N * 2, False)
        seen.add((kind, splits > 1))
    assert {(1, False), (1, True), (2, False)} <= seen, seen
    # the gradient at the weights: tiles of 128 and 256, and short steps, by cx_mm_grad.hip's rule
    seen = set()
    for P, E, N, K in [*GRADS, *LARGE_GRADS]:
        mats = max(1, E)
        many = mats * -(-K // 256) * -(-N // 256) >= 256
        seen.add("small" if not many else "short" if P < mats * 1024 else "long")
    assert seen == {"small", "short", "long"}
