"""Products with 4-bit weights through the GEMM, against their formulas in 64 bits on
the CPU.  Tolerances count roundings, as in test_gpu_q4.py: a sum of n exact products
is off by at most n 2^-24 of the sum of their sizes, and the output's rounding adds
half a step.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_q4 import BF, F8, HF, SF, TINY, U, dense, make, make_x, near, product_ref, rand, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,N,K,group", [(18, 40, 1025, 64), (150, 24, 1030, 128)])
def test_top_k_without_an_order(gpu, T, N, K, group, dtype):
    """Without an order row p of y is row p of x, whatever top_k is: a row's power of two belongs to that row."""
    from constellation_amd.engine import Q4Matrix
    codes, scales = make(T, 1, N, K, group)
    w = Q4Matrix.pack(codes.cuda(), scales.cuda(), K, group=group)
    try:
        # rows whose sizes differ by powers of two, so that another row's factor shows
        x = rand(1, T, K, dtype=dtype) * (2.0 ** (torch.arange(T) % 5).to(dtype))[:, None]
        want, e = product_ref(x.double(), dense(codes, scales, K, group)[0], False)
        for top_k in (1, 0, -3, 7, 1 << 30):
            print(f"[q4 gemm] no order, top_k {top_k} {dtype}", flush=True)
            y = gpu.q4_matmul(w, x.cuda(), top_k=top_k)
            torch.cuda.synchronize()
            near(y, want, rounded(want, e, dtype), top_k)
    finally:
        w.free()
