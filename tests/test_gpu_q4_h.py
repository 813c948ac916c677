"""How much of h a layer of 4-bit experts keeps between its two products.  Every row of
its matrices has one weight of 1, so that gate, up and the down product are values as they
are, and all that rounds is silu, h's way into the second product and the routes' sum."""
from __future__ import annotations

import pytest
import torch

from test_gpu_q4 import BF, HALF, HF, TINY, U, near

pytestmark = pytest.mark.gpu


def picks(n_mats, cols_of_row, cols):
    """codes of matrices whose row r has a 1 in column cols_of_row[r] (another one in each matrix)"""
    codes = torch.zeros(n_mats, len(cols_of_row), (cols + 1) // 2, dtype=torch.uint8)
    at = (torch.tensor(cols_of_row)[None] + 3 * torch.arange(n_mats)[:, None]) % cols
    codes.scatter_(2, (at // 2)[..., None], (2 << (4 * (at % 2))).to(torch.uint8)[..., None])
    return codes, at


# kernel, tokens, routes, experts, hidden, inter: one token's two launches (one and four steps of 512 columns), the decode
# kernel with 1 to 4 rows an item, the GEMM with and without ranges of the columns
CASES = [("one token", 1, 3, 5, 96, 136), ("one token", 1, 8, 12, 64, 2048), ("one token", 1, 16, 20, 40, 1000), ("decode", 2, 2, 5, 72, 40),
         ("decode", 3, 4, 40, 64, 2048), ("decode", 2, 2, 4, 64, 7000), ("gemm", 70, 2, 2, 130, 264), ("gemm", 40, 3, 4, 64, 8200),
         ("gemm", 900, 4, 5, 2048, 130)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kernel,T,K,E,H,I", CASES)
def test_h_keeps_its_bits(gpu, kernel, T, K, E, H, I, dtype):
    from constellation_amd.engine import Q4Layer, Q4Matrix
    group = 32 if I % 64 else 64 if I % 128 else 128
    print(f"[q4 h] {kernel} {T}x{K} of {E} {H}x{I} group {group} {dtype}", flush=True)
    gu_codes, gu_at = picks(E, [(7 * n) % H for n in range(I)] + [(5 * n + 1) % H for n in range(I)], H)
    dn_codes, dn_at = picks(E, [(11 * n) % I for n in range(H)], I)
    ones = [torch.ones(E, n, -(-c // group), dtype=BF).cuda() for n, c in ((2 * I, H), (H, I))]
    mats = [Q4Matrix.pack(gu_codes.cuda(), ones[0], H, group=group, gated=True), Q4Matrix.pack(dn_codes.cuda(), ones[1], I, group=group)]
    try:
        layer = Q4Layer(gpu, *mats)
        g = torch.Generator().manual_seed(T + I)
        x = (torch.randn(T, H, generator=g) * 3).to(dtype)
        ids = torch.rand(T, E, generator=g).topk(K, dim=1).indices.to(torch.int32)
        w = torch.rand(T, K, generator=g) + 0.1
        y, yf = gpu.moe(layer, x.cuda(), ids.cuda(), w.cuda(), want_f32=True)
        torch.cuda.synchronize()
        gpu.sync()
        want, tol = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
        x64 = x.double()
        for k in range(K):
            e = ids[:, k].long()
            gate, up = x64.gather(1, gu_at[e, :I]), x64.gather(1, gu_at[e, I:])
            h = gate * torch.sigmoid(gate) * up
            term = w[:, k:k + 1].double() * h.gather(1, dn_at[e])
            want += term
            # silu and its product 5 roundings, h in two parts 2 (or 2^-39 of its row's largest value), the products with
            # its factor and the route's weight and the sum of routes 2 + K
            tol += term.abs() * (9 + K) * U + w[:, k:k + 1].double() * h.abs().amax(1, keepdim=True) * 2.0 ** -39
        near(yf, want, tol, "fp32")
        near(y, want, tol + (want.abs() + tol) * HALF[dtype] + TINY[dtype], "rounded")
    finally:
        for m in mats:
            m.free()


@pytest.mark.parametrize("T,I", [(1, 136), (3, 136), (70, 136)])
def test_an_infinite_h_stays_in_its_token(gpu, T, I):
    """The token whose h is infinite has no finite output; the others are as without it."""
    from constellation_amd.engine import Q4Layer, Q4Matrix
    print(f"[q4 h] infinite {T}", flush=True)
    E, H = 2, 64
    gu_codes = torch.full((E, 2 * I, H // 2), 0x22, dtype=torch.uint8)  # ones: an infinity times zero would be a NaN
    dn_codes = torch.full((E, H, I // 2), 0x22, dtype=torch.uint8)
    mats = [Q4Matrix.pack(gu_codes.cuda(), torch.ones(E, 2 * I, 1, dtype=BF).cuda(), H, gated=True),
            Q4Matrix.pack(dn_codes.cuda(), torch.ones(E, H, 2, dtype=BF).cuda(), I)]
    try:
        layer = Q4Layer(gpu, *mats)
        x = torch.rand(T, H, generator=torch.Generator().manual_seed(1)).to(BF) + 1
        ids, w = torch.tensor([[0, 1]] * T, dtype=torch.int32).cuda(), torch.ones(T, 2).cuda()
        clean = gpu.moe(layer, x.cuda(), ids, w, want_f32=True)[1]
        x[0, 5] = float("inf")
        got = gpu.moe(layer, x.cuda(), ids, w, want_f32=True)[1]
        torch.cuda.synchronize()
        assert bool(torch.isinf(got[0]).all()) and bool((got[0] > 0).all())  # sums of infinities
        assert torch.equal(got[1:], clean[1:])
    finally:
        for m in mats:
            m.free()


def test_h_of_more_than_4_gb(gpu):
    """Places in h past 32 bits: the last rows of a call whose h in two planes takes 4.4 GB."""
    from constellation_amd.engine import Q4Layer, Q4Matrix
    from test_gpu_q4 import dense, layer_ref, make, rounded
    T, K, E, H, I = 67_000, 8, 9, 64, 2048
    print(f"[q4 h] {T}x{K} of {E} {H}x{I}", flush=True)
    gu, dn = make(1, E, 2 * I, H, 64), make(2, E, H, I, 128)
    mats = [Q4Matrix.pack(gu[0].cuda(), gu[1].cuda(), H, group=64, gated=True), Q4Matrix.pack(dn[0].cuda(), dn[1].cuda(), I)]
    try:
        layer = Q4Layer(gpu, *mats)
        x = torch.randn(T, H, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(BF)
        ids = torch.rand(T, E, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).topk(K, dim=1).indices.to(torch.int32)
        w = torch.rand(T, K, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
        y, yf = gpu.moe(layer, x, ids, w, want_f32=True)
        torch.cuda.synchronize()
        gpu.sync()
        some = torch.cat((torch.arange(8), torch.arange(T - 24, T), torch.randperm(T, generator=torch.Generator().manual_seed(4))[:16]))
        want, tol = layer_ref(x.cpu().double()[some], ids.cpu()[some], w.cpu()[some], dense(*gu, H, 64), dense(*dn, I, 128), 2.0 ** -22)
        near(yf.cpu()[some], want, tol, "fp32")
        near(y.cpu()[some], want, rounded(want, tol, BF), "rounded")
    finally:
        torch.cuda.synchronize()
        for m in mats:
            m.free()
