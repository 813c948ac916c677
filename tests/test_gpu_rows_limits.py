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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K,H,few,many", [(6, 37, 299, 300), (7, 64, 499, 500), (16, 129, 112, 113), (9, 2056, 388, 389)])
def test_combine_gradient_on_both_sides_of_its_rule(gpu, K, H, few, many, dtype):
    """One route a workgroup and eight: a token's gradients have the same bits, and are the formula's."""
    print(f"[rows] gradient of {K} rows of {H} {dtype}", flush=True)
    g = torch.Generator().manual_seed(H)
    E = 24
    ids = torch.rand(many, E, generator=g).topk(K, dim=1).indices.to(torch.int32)
    ids[torch.rand(many, K, generator=g) < 0.1] = -1
    dout, w = torch.randn(many, H, generator=g).to(dtype), torch.rand(many, K, generator=g)
    by_pair = torch.randn(many, K, H, generator=g).to(dtype)
    got = {}
    for T in (few, many):
        place = gpu.sort_tokens(ids[:T].cuda(), E)[2]
        at = torch.where(place < 0, ~place, place).long()
        ys = torch.empty(T * K, H, dtype=dtype, device="cuda")
        ys[at.view(-1)] = by_pair[:T].reshape(-1, H).cuda()
        dys, dw = gpu.combine_rows_grad(dout[:T].cuda(), ys, place, w[:T].cuda())
        got[T] = dys[at].cpu(), dw.cpu()
    assert all(torch.equal(a, b[:few]) for a, b in zip(got[few], got[many]))
    held = (ids >= 0).double()
    want_dw, size = (torch.einsum("th,tkh->tk", a, b) * held for a, b in ((dout.double(), by_pair.double()), (dout.double().abs(), by_pair.double().abs())))
    assert bool(((got[many][1].double() - want_dw).abs() <= (H + 8) * 2.0 ** -24 * size).all())
    want = (w.double() * held)[..., None] * dout.double()[:, None]
    half = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[dtype]
    assert bool(((got[many][0].double() - want).abs() <= want.abs() * (half + 2.0 ** -23) + 2.0 ** -130).all())
