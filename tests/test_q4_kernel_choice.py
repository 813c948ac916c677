"""Which kernel the sizes of the 4-bit tests take, by the rules of csrc/cx_shapes.h on
the host: a changed rule must not move a kernel's tests to another kernel unseen."""
from __future__ import annotations

import pytest

from test_gpu_q4_gemm import DEC_LAYERS, GEMM_LAYERS, ONE, STACKS
from test_q4_shapes import rules  # noqa: F401  (a fixture)


def tiles(N, K, gated):
    return (-(-(N // 2) // 8) if gated else -(-N // 16)), -(-K // 128)


def gemm_splits(rules, rows, mats, N, K, gated, e4m3):
    item = rules.item(rows, mats, N, K, int(e4m3))
    assert item == (64 if e4m3 else 128), (rows, mats, N, K, gated, e4m3, item)
    return rules.splits(*tiles(N, K, gated), rows, mats, item)


@pytest.mark.parametrize("e4m3", [False, True])
def test_products_of_one_matrix_reach_the_gemm(rules, e4m3):
    """Of each epilogue: outputs straight from the accumulators and through partial sums, of
    widths that whole stores divide and that they do not."""
    seen = set()
    for T, N, K in ONE:
        for gated in (False, True):
            s = gemm_splits(rules, T, 1, N, K, gated, e4m3)
            seen.add((s > 1, gated, (N // 2 if gated else N) % 8 == 0))
    assert seen == {(a, b, c) for a in (False, True) for b in (False, True) for c in (False, True)}


@pytest.mark.parametrize("e4m3", [False, True])
def test_stacks_reach_the_gemm(rules, e4m3):
    seen = {(gemm_splits(rules, P, E, N, K, gated, e4m3) > 1, gated) for P, E, N, K in STACKS for gated in (False, True)}
    assert len(seen) == 4


def test_layers(rules):
    for T, K, E, H, I, shared in GEMM_LAYERS:
        assert rules.layer(T * (K + shared), E + shared, max(H, I)) == 128 and not rules.routes(T, K, H, I, shared)
    for T, K, E, H, I, shared, alone in DEC_LAYERS:
        assert rules.layer(T * (K + shared), E + shared, max(H, I)) < 16 and bool(rules.routes(T, K, H, I, shared)) == alone
