"""A layer of 4-bit experts split over nodes: each holds some of the stacks, and the dispatcher
sends every route to the one that holds its expert."""
from __future__ import annotations

import pytest
import torch

from test_gpu_q4 import BF, dense, layer_ref, make, near, rand, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 3, 90])
def test_two_nodes_equal_one(gpu, T):
    from constellation_amd import moe_dispatch as D
    from constellation_amd._lib import CxError
    from constellation_amd.engine import Q4Layer, Q4Matrix
    print(f"[q4 split] {T} tokens", flush=True)
    E, K, H, I = 12, 4, 256, 128
    gu, dn = make(1, E, 2 * I, H, 32), make(2, E, H, I, 64)
    halves = [[0, 3, 4, 7, 10], [11, 9, 8, 6, 5, 2, 1]]
    mats = []

    def packed(pick):
        g = Q4Matrix.pack(gu[0][pick].cuda(), gu[1][pick].cuda(), H, group=32, gated=True)
        d = Q4Matrix.pack(dn[0][pick].cuda(), dn[1][pick].cuda(), I, group=64)
        mats.extend((g, d))
        return g, d
    try:
        nodes = [D.LocalNode({0: Q4Layer(gpu, *packed(h), experts=h, n_experts=E)}) for h in halves]
        x = rand(3, T, H, dtype=BF)
        g = torch.Generator().manual_seed(T)
        ids = torch.rand(T, E, generator=g).topk(K, dim=1).indices.to(torch.int32)
        ids[0, 0] = -1
        w = torch.rand(T, K, generator=g)
        want, tol = layer_ref(x.double(), ids, w, dense(*gu, H, 32), dense(*dn, I, 64), 2.0 ** -22)
        y = D.run_topk_moe_layer(nodes, x.cuda(), 0, ids.cuda(), w.cuda(), n_experts=E, shared=False)
        torch.cuda.synchronize()
        D.check_routes()
        near(y, want, rounded(want, tol, BF), "two nodes")
        # one node alone: its own routes, the others left out and reported
        only = torch.where(torch.isin(ids, torch.tensor(halves[1])), ids, -1).to(torch.int32)
        lay = nodes[1].layers[0]
        alone = gpu.moe(lay, x.cuda(), only.cuda(), w.cuda())
        gpu.sync()
        assert torch.equal(gpu.moe(lay, x.cuda(), ids.cuda(), w.cuda()), alone)
        with pytest.raises(CxError, match="out of range"):
            gpu.sync()
        # router and experts in one call, with the router's ids
        wr, bias = rand(6, E, H, dtype=BF, std=0.02).cuda(), rand(7, E, std=0.01).cuda()
        opt = dict(n_group=4, topk_group=2, top_k=K, norm_topk_prob=True, routed_scaling_factor=2.5)
        here = torch.zeros(E, dtype=torch.uint8)
        here[halves[1]] = 1
        y1, _, ids1, w1 = gpu.moe_layer(lay, x.cuda(), wr, bias, resident=here.cuda(), **opt)
        assert torch.equal(y1, gpu.moe(lay, x.cuda(), ids1, w1)) and bool(torch.isin(ids1.cpu(), torch.tensor(halves[1] + [-1])).all())
        gpu.sync()
        y2, ids2, w2 = D.run_moe_layer_batched(nodes, x.cuda(), 0, wr, bias, shared=False, **opt)
        assert torch.equal(y2, D.run_topk_moe_layer(nodes, x.cuda(), 0, ids2, w2, n_experts=E, shared=False))
    finally:
        torch.cuda.synchronize()
        for m in mats:
            m.free()
