"""moe_dispatch with remote nodes only needs no GPU, and so no torch that was built for
one: the module and a remote call work where torch lacks its GPU bindings."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

PROGRAM = r"""
import numpy as np, torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
from constellation_amd import moe_dispatch as D, moe_layer_protocol as P

def node(frame):
    hdr = P.decode_header(frame[:P.HEADER_BYTES])
    req = P.decode_moe_layer_request(frame[P.HEADER_BYTES:])
    body = P.encode_moe_layer_response({"status_code": 0, "batch_size": req["batch_size"], "hidden_dim": req["hidden_dim"],
                                        "output_dtype": req["output_dtype"], "output": req["activation"]})
    return P.frame(P.MOE_LAYER_RESPONSE, hdr["request_id"], body)

x = torch.arange(32, dtype=torch.float32).view(2, 16).to(torch.bfloat16)
y = D.run_topk_moe_layer([D.RemoteNode(node, {0: range(4)})], x, 0, torch.tensor([[0, 1], [2, 3]]), torch.ones(2, 2), n_experts=4, shared=False)
assert torch.equal(x, y)
print("ok")
"""


def test_dispatch_to_remote_nodes():
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr[-2000:]
