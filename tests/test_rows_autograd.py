"""gather_rows and combine_rows record no graph: tensors that require grad are refused where
a graph is being recorded, rather than answered with a result that has none.  No GPU:
a context of "device -1", where CPU tensors are at home."""
from __future__ import annotations

import pytest
import torch

from test_q4_layer_checks import Called, ctx  # noqa: F401  (ctx is a fixture)

T, K, H = 3, 2, 8


@pytest.mark.parametrize("which", ["x", "ys", "weights", "add"])
def test_a_recorded_graph_is_not_lost(ctx, which):  # noqa: F811
    place = torch.arange(T * K, dtype=torch.int32).view(T, K)
    t = {"x": torch.zeros(T, H), "ys": torch.zeros(T * K, H), "weights": torch.ones(T, K), "add": torch.zeros(T, H)}

    def call():
        if which == "x":
            return ctx.gather_rows(t["x"], place)
        return ctx.combine_rows(t["ys"], place, t["weights"], add=t["add"])
    with pytest.raises(Called):  # reaches the library
        call()
    t[which].requires_grad_()
    with pytest.raises(ValueError, match="records no graph"):
        call()
    with torch.no_grad(), pytest.raises(Called):
        call()

    class Own(torch.autograd.Function):  # whose forward records nothing
        @staticmethod
        def forward(fn, _):
            with pytest.raises(Called):
                call()
            return torch.zeros(())
    Own.apply(t[which])
