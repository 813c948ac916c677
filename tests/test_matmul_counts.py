"""Counts that do not fit the C ABI's 32 bits are refused: they would arrive there as what is left of them modulo 2^32, a call
on a few of the rows.  No GPU: tensors without memory, and a library that says that it was called."""
from __future__ import annotations

import pytest
import torch

from constellation_amd.engine import I8Layer
from test_q4_layer_checks import Called, ctx  # noqa: F401  (ctx is a fixture)

BIG = 2 ** 32 + 8
BF, Q, F32, I32 = torch.bfloat16, torch.int8, torch.float32, torch.int32


def m(*s, dtype=BF):
    return torch.empty(s, dtype=dtype, device="meta")


CALLS = {
    "rows of x": lambda c, n: c.matmul(m(n, 8), m(8, 8)),
    "columns": lambda c, n: c.matmul(m(4, n), m(8, n)),
    "weight rows": lambda c, n: c.matmul(m(4, 8), m(n, 8)),
    "matrices": lambda c, n: c.matmul(m(4, 8), m(n, 8, 8), offsets=m(n + 1, dtype=I32)),
    "order": lambda c, n: c.matmul(m(4, 8), m(8, 8), order=m(n, dtype=I32)),
    "top_k": lambda c, n: c.matmul(m(4, 8), m(8, 8), order=m(4, dtype=I32), top_k=n),
    "gradient's rows": lambda c, n: c.matmul_grad(m(n, 8), m(n, 8), m(8, 8)),
    "gradient's columns": lambda c, n: c.matmul_grad(m(4, 8), m(4, n), m(8, n)),
    "gradient's weight rows": lambda c, n: c.matmul_grad(m(4, n), m(4, 8), m(n, 8)),
    "rows to 8 bits": lambda c, n: c.quantize_i8(m(n, 1)),
    "rows to 8 bits, of all leading dimensions": lambda c, n: c.quantize_i8(m(n // 8, 8, 1)),
    "columns to 8 bits": lambda c, n: c.quantize_i8(m(1, n)),
    "rows of 8 bits": lambda c, n: c.i8_matmul(m(n, 8, dtype=Q), m(n, dtype=F32), m(8, 8, dtype=Q), m(8, dtype=F32)),
    "order in 8 bits": lambda c, n: c.i8_matmul(m(4, 8, dtype=Q), m(4, dtype=F32), m(8, 8, dtype=Q), m(8, dtype=F32), order=m(n, dtype=I32)),
    "top_k in 8 bits": lambda c, n: c.i8_matmul(m(4, 8, dtype=Q), m(4, dtype=F32), m(8, 8, dtype=Q), m(8, dtype=F32), order=m(4, dtype=I32), top_k=n),
}


@pytest.mark.parametrize("what", CALLS)
def test_counts_past_32_bits(ctx, what):  # noqa: F811
    with pytest.raises(Called):
        CALLS[what](ctx, 16)
    with pytest.raises(ValueError, match="fit 32 bits"):
        CALLS[what](ctx, BIG)


@pytest.mark.parametrize("E,H,I", [(2, BIG, 4), (2, 4, BIG), (2, 4, BIG // 2), (BIG, 4, 4)])
def test_a_layer_past_32_bits(ctx, E, H, I):  # noqa: F811
    with pytest.raises(ValueError, match="fit 32 bits"):
        I8Layer(ctx, m(E, 2 * I, H, dtype=Q), m(E, 2 * I, dtype=F32), m(E, H, I, dtype=Q), m(E, H, dtype=F32))


def test_tokens_past_32_bits(ctx):  # noqa: F811
    layer = I8Layer(ctx, m(2, 8, 8, dtype=Q), m(2, 8, dtype=F32), m(2, 8, 4, dtype=Q), m(2, 8, dtype=F32))
    for n, k, error in ((4, 2, Called), (BIG, 2, ValueError), (4, BIG, ValueError)):
        with pytest.raises(error):
            ctx.moe(layer, m(n, 8), m(n, k, dtype=I32), m(n, k, dtype=F32))
    for n, error in ((4, Called), (BIG, ValueError)):
        with pytest.raises(error):
            ctx.moe_layer(layer, m(n, 8), m(2, 8), m(2, dtype=F32), n_group=1, topk_group=1, top_k=1)
