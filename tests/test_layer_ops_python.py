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


def test_plan_arguments_are_not_rounded_or_wrapped():
    from ai2bmd_amd.attention import FragmentAttention, _whole
    for bad in (dict(start=[0, 2.5], end=[2.5, 6]), dict(start=[0, 2], end=[2, 6.7]), dict(start=[0, float("nan")], end=[float("nan"), 4]),
                dict(query_start=[0, 1], query_end=[1, 2.5]), dict(buckets=[0, 0.5, 1]), dict(buckets=[0, 1 << 32, 1]), dict(buckets=[True]),
                dict(heads=1025), dict(heads=2048), dict(end=[2, (1 << 30) + 1])):
        a = dict(start=[0, 2], end=[2, 6], heads=2, dim=8)
        a.update(bad)
        with pytest.raises(ValueError):
            FragmentAttention(a.pop("start"), a.pop("end"), a.pop("heads"), a.pop("dim"), **a)
    for good in ([0, 5], (0, 5), np.array([0.0, 5.0]), np.array([0, 5], dtype=np.int16), torch.tensor([0, 5])):
        got = _whole(good, "start", np.int64)
        assert got.dtype == np.int64 and got.tolist() == [0, 5]
