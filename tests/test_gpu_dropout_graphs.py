"""Masks that graphs draw."""

import pytest
import torch

from deepof_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("kind", ["dropout", "group_norm"])
def test_two_captures_draw_masks_of_their_own(kind):
    """Two graphs of the same call, replayed in turn: no mask comes twice."""
    x = torch.randn(2, 64, 16, 16, device=DEV).abs() + 1.0
    x = x.contiguous(memory_format=torch.channels_last)

    def call():
        if kind == "dropout":
            return ops.dropout(x, 0.5)
        return ops.group_norm(x, 8, dropout=0.5)

    call()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    masks = []
    for _ in range(3):
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            masks.append(out != 0)
        masks.append(call() != 0)
    n = x.numel()
    for i, m in enumerate(masks):
        # 6 standard deviations of n draws
        assert abs(float(m.double().mean()) - 0.5) < 3 / n**0.5
        for other in masks[:i]:
            assert abs(float((m == other).double().mean()) - 0.5) < 3 / n**0.5
