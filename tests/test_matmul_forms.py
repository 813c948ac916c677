"""The GPU tests' sizes reach every form of the products of a program's own experts: whatever the rule returns for sizes all over
its range, some test runs, with items of each count of tiles."""
from __future__ import annotations

import random

import test_gpu_matmul as small
import test_gpu_matmul_forms as forms
import test_gpu_matmul_large as large
from test_gpu_q4 import split
from test_matmul_rules import form, rules  # noqa: F401  (rules is a fixture)


def chosen(rules, P, E, out, depth, few):  # noqa: F811
    """A form: ranges and tiles a wave of few rows; otherwise the kernel, whether it has ranges, and an item's most tiles in n."""
    kind, rows, splits, tiles = form(rules, P, E, out, depth, few)
    return (0, splits, tiles) if kind == 0 else (kind, splits > 1, rows // (64 if kind == 2 else 32))


def run(rules, P, E, out, depth, few):  # noqa: F811
    """What a test with these rows, dealt as tests deal them, makes kernels do: the tiles of each of its items."""
    kind, cap, splits, tiles = form(rules, P, E, out, depth, few)
    if kind == 0:
        return {(0, splits, tiles)}
    off = split(P, E, P).tolist() if E else [0, P]
    got = set()
    for rows in (b - a for a, b in zip(off, off[1:]) if b > a):
        n = -(-rows // cap)
        share = rules.share(n, rows)
        got |= {(kind, splits > 1, -(-min(share, rows - i * share) // (64 if kind == 2 else 32))) for i in range(n)}
    return got


def four(sizes):
    return [(s[0], 0, s[1], s[2]) if len(s) == 3 else s for s in sizes]


def all_forms(rules, el, few):  # noqa: F811
    r, out = random.Random(0), set()
    for _ in range(40000):
        P, N, K = (int(2 ** r.uniform(0, hi)) for hi in (17, 15, 14))
        E = r.choice([0, 0, 1, 8, 64, int(2 ** r.uniform(0, 10))])
        out.add(chosen(rules, P, E, N, K * el, few) if few else chosen(rules, P, E, K, N * el, few))
    return out


def test_forward_in_16_bits(rules):  # noqa: F811
    sizes = four(small.ONE) + small.STACK + large.FORWARD + forms.FEW + forms.TILES
    got = set().union(*(run(rules, P, E, N, K * 2, True) for P, E, N, K in sizes))
    assert all_forms(rules, 2, True) <= got, all_forms(rules, 2, True) - got
    for odd in (0, 1):  # rows that are whole pieces of 16 bytes, and others
        few = set().union(*(run(rules, P, E, N, K * 2, True) for P, E, N, K in sizes if (K % 8 != 0) == odd))
        assert {f for f in got if f[0] == 0} <= few, (odd, few)


def test_forward_in_8_bits(rules):  # noqa: F811
    sizes = four(small.ONE) + small.STACK + [(P, E, N, -(-K // 16) * 16) for P, E, N, K in large.FORWARD] + forms.FEW_8 + forms.TILES_8
    got = set().union(*(run(rules, P, E, N, K, True) for P, E, N, K in sizes))
    assert all_forms(rules, 1, True) <= got, all_forms(rules, 1, True) - got
    for odd in (0, 1):
        few = set().union(*(run(rules, P, E, N, K, True) for P, E, N, K in sizes if (K % 16 != 0) == odd))
        assert {f for f in got if f[0] == 0} <= few, (odd, few)


def test_gradient_at_x(rules):  # noqa: F811
    sizes = [s for s in small.GRADS + large.GRADS + forms.GRADS if s[0] > 0]
    got = set().union(*(run(rules, P, E, K, N * 2, False) for P, E, N, K in sizes))
    assert all_forms(rules, 2, False) <= got, all_forms(rules, 2, False) - got
