"""The rows around the experts at the ends of their ranges of sizes."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("short", [1, 3, 16, 257])
def test_gather_of_the_widest_rows(gpu, short):
    """Rows of just under 2^31 bytes, in pieces of 1 to 16 bytes."""
    n = 2 ** 31 - short
    print(f"[rows] gather of {n} bytes", flush=True)
    x = torch.empty(1, n, dtype=torch.uint8, device="cuda")
    x[0, :1 << 20] = torch.arange(1 << 20, device="cuda") % 251
    x[0, 1 << 20:] = 7
    x[0, -5:] = torch.tensor([1, 2, 3, 4, 5], device="cuda")
    xs = gpu.gather_rows(x, torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    gpu.sync()
    assert xs.shape == x.shape and torch.equal(xs, x)
