"""The products and gradients of test_gpu_matmul.py at sizes that take the larger tiles, ranges of the contraction
and steps of every count, against the formulas in 64 bits on the GPU, with the same tolerances."""
from __future__ import annotations

import pytest
import torch

from test_gpu_matmul import poisoned, rounded
from test_gpu_q4 import BF, HF, SF, TINY, HALF, U, rand, split

pytestmark = pytest.mark.gpu

# rows, matrices (0: one, without offsets), weight rows, columns
FORWARD = [(2500, 0, 4104, 136), (4096, 0, 4096, 136), (2600, 0, 4096, 712), (3001, 0, 1040, 2056), (700, 0, 2064, 4104), (2000, 0, 2048, 7168), (300, 0, 4096, 2048), (65, 0, 1030, 7168),
           (6000, 5, 2056, 200), (9000, 70, 1032, 264), (5000, 40, 2064, 392), (4100, 3, 520, 1032), (900, 30, 4104, 1032)]
GRADS = [(1100, 0, 4104, 4096), (3000, 40, 712, 520), (1200, 300, 40, 24), (700, 0, 2064, 1032), (90, 0, 4104, 1032), (6000, 5, 2056, 1032), (2600, 0, 1032, 4104)]


def close(got, want, tol, out, what):
    got = got.double()
    e = tol + (want.abs() + tol) * HALF[out] + TINY[out]
    over = (got - want).abs() - e
    assert not bool(torch.isnan(over).any()) and float(over.max()) <= 0, (what, float(over.max()))


def product(x, w, off, gated):
    """Sums, outputs and how far each may be off, on x's device; rows behind the last matrix are zeros."""
    P, N, K = x.shape[0], w.shape[1], w.shape[2]
    y, e = (torch.zeros(P, N, dtype=torch.float64, device=x.device) for _ in range(2))
    for m in range(w.shape[0]):
        a, b = off[m], off[m + 1]
        if a < b:
            y[a:b] = x[a:b].double() @ w[m].double().T
            e[a:b] = (x[a:b].double().abs() @ w[m].double().abs().T) * (K + 8) * U
    if not gated:
        return y, e, y, e
    g, u, eg, eu = y[:, :N // 2], y[:, N // 2:], e[:, :N // 2], e[:, N // 2:]
    s = g * torch.sigmoid(g)
    return y, e, s * u, 1.1 * eg * (u.abs() + eu) + s.abs() * eu + (s * u).abs() * (g.abs() + 16) * 2 * U


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("P,E,N,K", FORWARD)
def test_forward(gpu, P, E, N, K, dtype):
    off = split(P, E, P).tolist() if E else [0, P]
    x, w = poisoned(rand(1, P, K, dtype=dtype), off[-1]).cuda(), rand(2, max(1, E), N, K, dtype=dtype, std=0.1).cuda()
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda") if E else None
    for gated, out in ((False, dtype), (True, dtype), (False, SF)):
        print(f"[mm] large {P} over {E} {N}x{K} gated {gated} {dtype} to {out}", flush=True)
        sums, es, want, e = product(x, w, off, gated)
        torch.full((P * N * 2,), float("nan"), device="cuda")  # goes back to the allocator
        y = gpu.matmul(x, w if E else w[0], gated=gated, keep=gated, offsets=offsets, out_dtype=out)
        if gated:
            y, pre = y
            close(pre, sums, es, dtype, "pre")
        close(y, want, e, out, gated)
    gpu.sync()


@pytest.mark.parametrize("P,E,N,K", FORWARD)
def test_forward_int8(gpu, P, E, N, K):
    K = -(-K // 16) * 16
    off = split(P, E, P).tolist() if E else [0, P]
    x, w = (torch.randint(-128, 128, s, generator=torch.Generator().manual_seed(i)).to(torch.int8).cuda() for i, s in enumerate(((P, K), (max(1, E), N, K))))
    xs, ws = torch.rand(P, device="cuda") * 1e-3 + 1e-4, torch.rand(max(1, E), N, device="cuda") * 0.1
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda") if E else None
    for gated in (False, True):
        print(f"[mm] large int8 {P} over {E} {N}x{K} gated {gated}", flush=True)
        y = torch.zeros(P, N, dtype=torch.float64, device="cuda")
        for m in range(w.shape[0]):
            a, b = off[m], off[m + 1]
            if a < b:
                y[a:b] = (x[a:b].double() @ w[m].double().T) * xs[a:b, None].double() * ws[m].double()
        e = y.abs() * 4 * U
        if gated:
            g, u, eg, eu = y[:, :N // 2], y[:, N // 2:], e[:, :N // 2], e[:, N // 2:]
            s = g * torch.sigmoid(g)
            y, e = s * u, 1.1 * eg * (u.abs() + eu) + s.abs() * eu + (s * u).abs() * (g.abs() + 16) * 2 * U
        got = gpu.i8_matmul(x, xs, w if E else w[0], ws if E else ws[0], gated=gated, offsets=offsets, out_dtype=SF)
        close(got, y, e, SF, gated)
    gpu.sync()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("P,E,N,K", GRADS)
def test_gradients(gpu, P, E, N, K, dtype):
    off = split(P, E, P).tolist() if E else [0, P]
    x, dy = poisoned(rand(1, P, K, dtype=dtype), off[-1]).cuda(), poisoned(rand(2, P, N, dtype=dtype, std=0.1), off[-1]).cuda()
    w = rand(3, max(1, E), N, K, dtype=dtype, std=0.1).cuda()
    print(f"[mm] large gradients {P} over {E} {N}x{K} {dtype}", flush=True)
    dx, ex = (torch.zeros(P, K, dtype=torch.float64, device="cuda") for _ in range(2))
    dw, ew = (torch.zeros(w.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for m in range(w.shape[0]):
        a, b = off[m], off[m + 1]
        if a == b:
            continue
        d, xx, ww = dy[a:b].double(), x[a:b].double(), w[m].double()
        dx[a:b], ex[a:b] = d @ ww, (d.abs() @ ww.abs()) * (N + 8) * U
        dw[m], ew[m] = d.T @ xx, (d.abs().T @ xx.abs()) * (b - a + 8) * U
    torch.full((P * K * 2 + w.numel() * 4,), float("nan"), device="cuda")  # goes back to the allocator
    for out in (dtype, SF):
        gx, gw = gpu.matmul_grad(dy, x, w if E else w[0], offsets=torch.tensor(off, dtype=torch.int32, device="cuda") if E else None, dw_dtype=out)
        close(gx, dx, ex, dtype, "dx")
        close(gw.view(w.shape), dw, ew, out, "dw")
        assert not gx[off[-1]:].any()
    gpu.sync()


def test_places_past_32_bits(gpu):
    """Rows of x, dy and outputs, and matrices of a stack, that lie past 4 GB of their buffers: what is far behind
    equals the same rows in a small call."""
    print("[mm] past 4 GB", flush=True)
    N, K = 4096, 4096
    P = 540_000  # rows of 8 KB: 4.4 GB of x, of y and of dy
    x = torch.empty(P, K, dtype=BF, device="cuda")
    tail = 600
    x[:P - tail] = 1.0
    g = torch.Generator(device="cuda").manual_seed(0)
    x[P - tail:] = torch.randn(tail, K, generator=g, device="cuda").to(BF)
    w = (torch.randn(N, K, generator=g, device="cuda") * 0.02).to(BF)
    y = gpu.matmul(x, w)
    near = gpu.matmul(x[P - tail:].contiguous(), w)
    # another cut of the same sums: both are within the fp32 bound and a half step of the exact value
    size = x[P - tail:].float().abs() @ w.float().abs().T
    assert bool(((y[P - tail:].float() - near.float()).abs() <= 2 * (size * (K + 8) * U + near.float().abs() * HALF[BF] * 1.01)).all())
    dx, _ = gpu.matmul_grad(y, x, w, want_dw=False)
    small, _ = gpu.matmul_grad(y[P - tail:].contiguous(), x[P - tail:].contiguous(), w, want_dw=False)
    size = y[P - tail:].float().abs() @ w.float().abs()
    assert bool(((dx[P - tail:].float() - small.float()).abs() <= 2 * (size * (N + 8) * U + small.float().abs() * HALF[BF] * 1.01)).all())
    # the rows of the last matrix of two: sums over places past 4 GB
    off = torch.tensor([0, P - tail, P], dtype=torch.int32, device="cuda")
    _, dw = gpu.matmul_grad(y[:, :64].contiguous(), x, w[:64].expand(2, 64, K).contiguous(), offsets=off, want_dx=False, dw_dtype=SF)
    want = y[P - tail:, :64].double().T @ x[P - tail:].double()
    size = y[P - tail:, :64].double().abs().T @ x[P - tail:].double().abs()
    assert bool(((dw[1].double() - want).abs() <= size * (tail + 8) * U + want.abs() * U).all())
    gpu.sync()
