"""Which calls of a program's own experts' products a launch holds: what is refused is what 2^32 threads do not hold, worked out
here from the kernels' tiles and their threads.  On the host, by the rules of csrc/cx_shapes.h."""
from __future__ import annotations

import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest

from constellation_amd._lib import BF16, CX_EINVAL, lib

CSRC = Path(__file__).resolve().parent.parent / "constellation_amd" / "csrc"

SOURCE = r"""
#include "cx_shapes.h"
using namespace cx;
extern "C" {
void form(int64_t rows, int mats, int stack, int64_t out, int64_t depth, int few, int* f) {
    const MmForm m = mm_form(rows, mats, stack, out, depth, few);
    f[0] = m.kind, f[1] = m.item_rows, f[2] = m.splits, f[3] = m.tiles;
}
int forward_ok(int64_t rows, int mats, int n, int k, int stack) {
    const MmForm f = mm_form(rows, mats, stack, n, (int64_t)k * 2, true);
    return mm_grid_ok(rows, mats, n, k, stack, &f, nullptr, false);
}
int dx_ok(int64_t rows, int mats, int n, int k, int stack) {
    const MmForm f = mm_form(rows, mats, stack, k, (int64_t)n * 2, false);
    return mm_grid_ok(rows, mats, n, k, stack, nullptr, &f, false);
}
int dw_ok(int64_t rows, int mats, int n, int k, int stack) { return mm_grid_ok(rows, mats, n, k, stack, nullptr, nullptr, true); }
int dw_kind(int64_t rows, int mats, int n, int k) { return mm_dw_kind(rows, mats, n, k); }
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("grid")
    (d / "rules.cc").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(d / "rules.cc"), "-o", str(d / "rules.so")],
                   check=True)
    L = C.CDLL(str(d / "rules.so"))
    L.form.argtypes = [C.c_int64, C.c_int, C.c_int, C.c_int64, C.c_int64, C.c_int, C.POINTER(C.c_int)]
    for f in (L.forward_ok, L.dx_ok, L.dw_ok):
        f.argtypes = [C.c_int64, C.c_int, C.c_int, C.c_int, C.c_int]
    L.dw_kind.argtypes = [C.c_int64, C.c_int, C.c_int, C.c_int]
    return L


def cdiv(a, b):
    return -(-a // b)


def threads(rules, P, E, stack, out, depth, few):
    """Of the largest launch of a product."""
    f = (C.c_int * 4)()
    rules.form(P, E, stack, out, depth, few, f)
    kind, rows, splits, tiles = f
    items = min(P, E) + P // rows + 1 if stack else cdiv(P, rows)
    if kind == 0:
        return items * cdiv(cdiv(out, 16), 8 // splits * tiles) * 512
    m = cdiv(out, 128 * kind) * splits
    grid = cdiv(items, 8) * 8 * m if stack else items * cdiv(m, 8) * 8
    return max(grid * 256 * kind, P * cdiv(out, 1024) * 256 if splits > 1 else 0)


def dw_threads(rules, P, E, n, k):
    kind = rules.dw_kind(P, E, n, k)
    bm, bn = {1: (128, 128), 2: (256, 256), 3: (256, 128)}[kind]
    tiles = E * cdiv(k, bm) * cdiv(n, bn)
    return (cdiv(tiles, 512) * 512 if kind == 3 else tiles) * (512 if kind == 2 else 256)


def test_what_is_refused_is_what_a_launch_does_not_hold(rules):
    r = random.Random(0)
    yes = no = 0
    for _ in range(20000):
        P, E, n, k = (int(2 ** r.uniform(0, hi)) for hi in (30, 10, 22, 22))
        stack = r.random() < 0.7
        E = E if stack else 1
        for ok, t in ((rules.forward_ok, threads(rules, P, E, stack, n, k * 2, 1)), (rules.dx_ok, threads(rules, P, E, stack, k, n * 2, 0)),
                      (rules.dw_ok, dw_threads(rules, P, E, n, k))):
            got = bool(ok(P, E, n, k, stack))
            assert got == (t < 2 ** 32), (P, E, n, k, stack, t)
            yes, no = yes + got, no + (not got)
    assert yes > 1000 and no > 1000
    assert not any(ok(2 ** 30 + 1, 1, 8, 8, 0) for ok in (rules.forward_ok, rules.dx_ok, rules.dw_ok))


# 2^28 - 128 rows are 2^21 - 1 items of 128, counted in eights, of 256 threads: the last that stay below 2^32
@pytest.mark.parametrize("P,E,n,k,stack", [(2_300_000, 1, 4096, 7168, 0), (2_300_000, 1, 7168, 2048, 0), (131072, 1, 131072, 7168, 0), (40_000_000, 1, 16, 8, 0),
                                           ((1 << 28) - 128, 1, 1, 1, 0), (4_000_000, 256, 4096, 7168, 1), (1 << 24, 1024, 4096, 2048, 1)])
def test_ordinary_sizes_are_held(rules, P, E, n, k, stack):
    assert rules.forward_ok(P, E, n, k, stack) and rules.dx_ok(P, E, n, k, stack) and rules.dw_ok(P, E, n, k, stack)


def test_the_library_takes_them():
    """The C ABI as far as the scratch, which it asks for after it has found that launches hold the call."""
    raw = C.create_string_buffer(4096)
    at = (C.addressof(raw) + 255) // 256 * 256  # in the place of device buffers, never read
    for P, n, k, text in ((2_300_000, 4096, 7161, b"scratch must be"), (1 << 29, 4096, 7161, b"too many rows or matrices for one launch")):
        assert lib().cx_matmul(at, at, P, at, BF16, 1, n, k, 0, None, 1, None, P, at, BF16, None, None, 0, None) == CX_EINVAL
        assert text in lib().cx_last_error()
        assert lib().cx_i8_matmul(at, at, at, P, at, at, 1, n, k, 0, None, 1, None, P, at, BF16, None, 0, None) == CX_EINVAL
        assert text in lib().cx_last_error()
        assert lib().cx_matmul_grad(at, at, at, at, BF16, None, 1, n, k, None, P, at, at, BF16, None, 0, None) == CX_EINVAL
        assert text in lib().cx_last_error()
