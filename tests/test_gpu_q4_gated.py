"""The gated epilogue of each kernel of the 4-bit products: silu(gate) * up with one
weight of 1 in each row, so that gate and up are values of x and only the epilogue rounds."""
from __future__ import annotations

import pytest
import torch

from test_gpu_q4 import BF, SF, U

pytestmark = pytest.mark.gpu

# an exponential within one unit (2 half steps), a sum, a quotient and a product of a rounding each, and
# what they add up to in the second order
ROUNDINGS = 5.01


@pytest.mark.parametrize("name,T,N,K", [("few rows", 20, 32, 64), ("decode", 3, 32, 1025), ("gemm", 2000, 1024, 1030), ("gemm in ranges", 80, 48, 1025)])
def test_silu_is_as_exact_as_its_exponential(gpu, name, T, N, K):
    from constellation_amd.engine import Q4Matrix
    print(f"[q4 gated] {name}", flush=True)
    codes = torch.zeros(1, N, (K + 1) // 2, dtype=torch.uint8)
    codes[0, :N // 2, 0] = 2        # gate: 1.0 in column 0
    codes[0, N // 2:, 0] = 2 << 4   # up: 1.0 in column 1
    w = Q4Matrix.pack(codes.cuda(), torch.ones(1, N, -(-K // 128), dtype=BF).cuda(), K, gated=True)
    try:
        for start in range(0, 24, T) if T < 24 else (0,):
            gate = torch.linspace(-85, 85, max(T, 24))[start:start + T].to(BF)
            x = torch.zeros(gate.numel(), K, dtype=BF)
            x[:, 0], x[:, 1] = gate, 1.0
            y = gpu.q4_matmul(w, x.cuda(), out_dtype=SF).cpu().double()
            g = gate.double()
            want = (g / (1 + torch.exp(-g)))[:, None].expand(-1, N // 2)
            off = ((y - want).abs() / want.abs().clamp(min=2.0 ** -126)).max()
            assert float(off) <= ROUNDINGS * U, (name, float(off) / U)
    finally:
        w.free()
