"""CPU: what the layer operators' Python side refuses before any device work."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad


def test_tangents_are_refused_not_dropped():
    from ai2bmd_amd.norm import no_graph
    x, p = torch.zeros(3), torch.zeros(3)
    no_graph(x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        no_graph(x, p, None)
        with pytest.raises(RuntimeError, match="tangent"):
            no_graph(p, dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
            no_graph(None, dual)
    no_graph(x, p)
