"""CPU: the layer operators refuse what they cannot take before any device work, at the C boundary (errno-style codes)
and in Python (ValueError / RuntimeError)."""
import ctypes as C

import pytest
import torch

P = C.c_void_p(1 << 20)  # an address that is never followed: every call below is refused before a launch


def test_layernorm_entry_points_refuse(lib_built):
    from ai2bmd_amd import capi
    L = capi.lib()
    good = [0, 1, 1, P, 64, P, P, 8, 64, 1e-5, P, 64, P, None]

    def call(**change):
        a = list(good)
        for k, v in change.items():
            a[int(k[1:])] = v
        return L.vsn_layernorm(*a)

    assert call(_1=3) == call(_1=-1) == -22                     # type
    assert call(_2=2) == -22                                    # parameters neither the rows' type nor float32
    assert call(_7=-1) == call(_8=0) == call(_8=4097) == -22    # rows, width
    assert call(_9=-1.0) == call(_9=float("nan")) == -22        # eps
    assert call(_3=None) == call(_10=None) == -22               # arrays
    assert call(_4=63) == call(_11=63) == -22                   # rows that overlap
    assert L.vsn_layernorm_workspace(-1, 64) == L.vsn_layernorm_workspace(8, 0) == -22
    size = L.vsn_layernorm_workspace(10 ** 9, 4096)
    assert 0 < size <= 1024 * 2 * 4096 * 4
    back = [0, 0, 0, P, 64, P, 64, P, P, 8, 64, P, 64, P, P, P, 1 << 20, None]
    for k, v in ((15, None), (16, 8), (7, None), (3, None), (5, None), (11, None), (4, 60), (6, 60), (12, 60), (10, 5000)):
        a = list(back)
        a[k] = v
        assert L.vsn_layernorm_backward(*a) == -22, k
    if not torch.cuda.is_available():
        assert L.vsn_layernorm(*good) == -19 and L.vsn_layernorm_backward(*back) == -19


def test_layer_norm_refuses_host_tensors():
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="cuda"):
        layer_norm(x)
    with pytest.raises(ValueError, match="cuda"):
        layer_norm_backward(x, x, torch.zeros(4, 2))
