"""The products and gradients of test_gpu_matmul.py in each form that the rules choose: every number of ranges and tiles of the
kernel for few rows, at aligned rows and others, and tiles of 128 and 256 with items of each length, whole contractions and
ranges of them, for 16 bits, for 8 and for the gradient at x.  test_matmul_forms.py holds that the sizes do so."""
from __future__ import annotations

import pytest
import torch

from test_gpu_matmul import poisoned
from test_gpu_matmul_large import close, product
from test_gpu_q4 import BF, HF, SF, U, rand, split

pytestmark = pytest.mark.gpu

# rows, matrices (0: one, without offsets), weight rows, columns
FEW = [(1, 0, 16594, 8), (1, 0, 16594, 9), (3, 3, 5544, 200), (3, 3, 5544, 201), (3, 3, 5792, 456), (3, 3, 5792, 457), (1648, 350, 34, 1152),
       (1648, 350, 34, 1153), (1, 0, 34, 464), (1, 0, 34, 465), (9, 0, 70, 208), (9, 0, 70, 205), (5, 0, 32, 1024), (5, 0, 32, 1021)]
TILES = [(220, 8, 284, 6160), (966, 12, 176, 8288), (2090, 0, 148, 11216), (193, 0, 4148, 11112), (2453, 8, 300, 10824)]
FEW_8 = [(1, 0, 16594, 16), (1, 0, 16594, 9), (730, 395, 36, 432), (730, 395, 36, 433), (433, 364, 34, 960), (433, 364, 34, 955), (845, 375, 34, 2336),
         (845, 375, 34, 2335), (1, 0, 34, 400), (1, 0, 34, 405), (5, 0, 32, 1024), (5, 0, 32, 1021), (3, 0, 32, 2064), (3, 0, 32, 2063)]
TILES_8 = [(1054, 0, 32, 4320), (941, 8, 34, 4064), (2187, 0, 32, 4120), (1193, 8, 32, 8176), (725, 27, 140, 5080), (247, 3, 2092, 10176), (4439, 0, 140, 11224),
           (193, 0, 4148, 22224)]
GRADS = [(4496, 3, 34, 136), (205, 0, 32, 8328), (210, 0, 32, 11280), (1985, 8, 990, 8), (854, 8, 4080, 8), (1210, 8, 4100, 8), (212, 8, 3052, 648),
         (653, 8, 4538, 664), (1796, 8, 10428, 144), (3382, 0, 18670, 152), (3801, 8, 32, 2656)]


def deal(P, E):
    return split(P, E, P).tolist() if E else [0, P]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("P,E,N,K", FEW + TILES)
def test_forward(gpu, P, E, N, K, dtype):
    off = deal(P, E)
    x, w = poisoned(rand(1, P, K, dtype=dtype), off[-1]).cuda(), rand(2, max(1, E), N, K, dtype=dtype, std=0.1).cuda()
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda") if E else None
    for gated, out in ((False, dtype), (True, dtype), (False, SF)):
        print(f"[mm] form {P} over {E} {N}x{K} gated {gated} {dtype} to {out}", flush=True)
        sums, es, want, e = product(x, w, off, gated)
        torch.full((P * N * 2,), float("nan"), device="cuda")  # goes back to the allocator
        y = gpu.matmul(x, w if E else w[0], gated=gated, keep=gated, offsets=offsets, out_dtype=out)
        if gated:
            y, pre = y
            close(pre, sums, es, dtype, "pre")
        close(y, want, e, out, gated)
        assert not y[off[-1]:].any()
    gpu.sync()


@pytest.mark.parametrize("P,E,N,K", FEW_8 + TILES_8)
def test_forward_int8(gpu, P, E, N, K):
    off = deal(P, E)
    x, w = (torch.randint(-128, 128, s, generator=torch.Generator().manual_seed(i)).to(torch.int8).cuda() for i, s in enumerate(((P, K), (max(1, E), N, K))))
    g = torch.Generator().manual_seed(3)
    xs, ws = (torch.rand(P, generator=g) * 1e-3 + 1e-4).cuda(), (torch.rand(max(1, E), N, generator=g) * 0.1).cuda()
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda") if E else None
    for gated in (False, True):
        print(f"[mm] form int8 {P} over {E} {N}x{K} gated {gated}", flush=True)
        y = torch.zeros(P, N, dtype=torch.float64, device="cuda")
        for m in range(w.shape[0]):
            a, b = off[m], off[m + 1]
            if a < b:
                y[a:b] = (x[a:b].double() @ w[m].double().T) * xs[a:b, None].double() * ws[m].double()
        e = y.abs() * 4 * U  # the sum is exact; its conversion and two scales round
        if gated:
            g, u, eg, eu = y[:, :N // 2], y[:, N // 2:], e[:, :N // 2], e[:, N // 2:]
            s = g * torch.sigmoid(g)
            y, e = s * u, 1.1 * eg * (u.abs() + eu) + s.abs() * eu + (s * u).abs() * (g.abs() + 16) * 2 * U
        got = gpu.i8_matmul(x, xs, w if E else w[0], ws if E else ws[0], gated=gated, offsets=offsets, out_dtype=SF)
        close(got, y, e, SF, gated)
        assert not got[off[-1]:].any()
    gpu.sync()


@pytest.mark.parametrize("P,E,N,K", [(1193, 8, 32, 8176), (2187, 0, 32, 4096), (725, 27, 140, 5120), (193, 0, 4148, 22224)])
def test_partial_sums_of_integers_are_not_numbers(gpu, P, E, N, K):
    """The ranges' sums lie in memory among floats, here as bits that a float has for signaling NaN (-8388607 .. -4194305):
    x 127 and weights -60 .. -100 over ranges of 512 to 640 columns and others."""
    print(f"[mm] form int8 bits {P} over {E} {N}x{K}", flush=True)
    off = deal(P, E)
    x = torch.full((P, K), 127, dtype=torch.int8, device="cuda")
    c = torch.arange(max(1, E) * N, device="cuda").view(max(1, E), N) % 41 - 100
    w = c[:, :, None].expand(-1, -1, K).to(torch.int8).contiguous()
    one, ones = torch.ones(P, device="cuda"), torch.ones(max(1, E), N, device="cuda")
    got = gpu.i8_matmul(x, one, w if E else w[0], ones if E else ones[0], offsets=torch.tensor(off, dtype=torch.int32, device="cuda") if E else None, out_dtype=SF)
    want = torch.zeros(P, N, dtype=torch.float32, device="cuda")
    for m in range(w.shape[0]):
        want[off[m]:off[m + 1]] = (c[m].long() * (127 * K)).float()  # the exact sum, rounded once
    assert torch.equal(got, want)
    gpu.sync()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("P,E,N,K", GRADS)
def test_gradients(gpu, P, E, N, K, dtype):
    off = deal(P, E)
    x, dy = poisoned(rand(1, P, K, dtype=dtype), off[-1]).cuda(), poisoned(rand(2, P, N, dtype=dtype, std=0.1), off[-1]).cuda()
    w = rand(3, max(1, E), N, K, dtype=dtype, std=0.1).cuda()
    print(f"[mm] form gradients {P} over {E} {N}x{K} {dtype}", flush=True)
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
    gx, gw = gpu.matmul_grad(dy, x, w if E else w[0], offsets=torch.tensor(off, dtype=torch.int32, device="cuda") if E else None)
    close(gx, dx, ex, dtype, "dx")
    close(gw.view(w.shape), dw, ew, dtype, "dw")
    assert not gx[off[-1]:].any()
    gpu.sync()
