"""Products and gradients of more rows than tiles of 16 would let a launch hold: the launched tiles have 128 or 256."""
from __future__ import annotations

import pytest
import torch

from test_gpu_q4 import BF, HALF, SF, TINY, U, rand

pytestmark = pytest.mark.gpu


def test_many_rows_of_a_small_matrix(gpu):
    """40 million rows of 8 columns by 16 x 8: rows of one repeated block, so that every block's results are the same."""
    print("[mm] 40 million rows", flush=True)
    block, n = 40_000, 1000
    x, w = rand(1, block, 8, dtype=BF).cuda(), rand(2, 16, 8, dtype=BF, std=0.1).cuda()
    want = x.double() @ w.double().T
    tol = (x.double().abs() @ w.double().abs().T) * 16 * U
    y = gpu.matmul(x.repeat(n, 1), w, out_dtype=BF).view(n, block, 16)
    assert torch.equal(y, y[:1].expand_as(y))
    e = tol + (want.abs() + tol) * HALF[BF] + TINY[BF]
    assert bool(((y[0].double() - want).abs() <= e).all())
    dy = rand(3, block, 16, dtype=BF).cuda()
    dx, _ = gpu.matmul_grad(dy.repeat(n, 1), x.repeat(n, 1), w, want_dw=False)
    dx = dx.view(n, block, 8)
    assert torch.equal(dx, dx[:1].expand_as(dx))
    want, tol = dy.double() @ w.double(), (dy.double().abs() @ w.double().abs()) * 24 * U
    assert bool(((dx[0].double() - want).abs() <= tol + (want.abs() + tol) * HALF[BF] + TINY[BF]).all())
    gpu.sync()


@pytest.mark.parametrize("dtype", [BF, SF])
def test_many_rows_to_8_bits(gpu, dtype):
    """More rows than one launch holds: 2^25 of a wave each."""
    block, n = 40_003, 839
    assert block * n > (1 << 25) + 3
    print(f"[mm] {block * n} rows to 8 bits {dtype}", flush=True)
    x = rand(4, block, 9, dtype=dtype)
    q, s = gpu.quantize_i8(x.cuda())
    want = (x.float().abs().amax(1) / torch.tensor(127.0)).clamp_min(1e-12)
    assert torch.equal(s.cpu(), want) and torch.equal(q.cpu(), torch.round(x.float() / want[:, None]).to(torch.int8))
    many, scales = gpu.quantize_i8(x.cuda().repeat(n, 1))
    assert torch.equal(many.view(n, block, 9), q.expand(n, block, 9)) and torch.equal(scales.view(n, block), s.expand(n, block))
    gpu.sync()
