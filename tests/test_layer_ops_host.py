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


def i64(*v):
    return (C.c_int64 * len(v))(*v)


def test_attention_entry_points_refuse(lib_built):
    from ai2bmd_amd import capi
    L = capi.lib()
    h = C.c_void_p()
    s, e = i64(0, 5), i64(5, 9)
    lut = (C.c_int32 * 5)(0, 1, 2, 1, 0)
    good = [C.byref(h), 0, 2, s, e, None, None, 8, 8, 32, 2, lut, 3]

    def create(**change):
        a = list(good)
        for k, v in change.items():
            a[int(k[1:])] = v
        return L.vsn_attn_create(*a)

    assert create(_0=None) == -22
    assert create(_2=0) == create(_2=-1) == -22                                       # no fragments
    assert create(_3=None) == create(_3=i64(0, 6)) == create(_3=i64(1, 5)) == -22      # gaps, a start that is not 0
    assert create(_4=i64(5, 4)) == create(_4=i64(5, 1 << 40)) == -22                   # backwards, too many rows
    assert create(_5=s) == create(_5=i64(0, 3), _6=i64(2, 4)) == -22                   # half of the query ranges, a gap
    assert create(_7=0) == create(_8=3) == create(_8=0) == -22                         # heads
    assert create(_9=4) == create(_9=36) == create(_9=136) == -22                      # head_dim
    assert create(_10=1024) == create(_10=-1) == create(_11=None) == -22               # reach, map
    assert create(_12=2) == create(_12=4097) == create(_12=-1) == -22                  # a bucket beyond the table
    assert create(_11=(C.c_int32 * 5)(0, 1, -1, 1, 0)) == -22
    assert not h.value
    assert L.vsn_attn_workspace(None, 1, 1, 0) == -22
    io, g = capi.VsnAttnIO(), capi.VsnAttnGrads()
    assert L.vsn_attn_forward(None, C.byref(io), None, 0, None) == -22
    assert L.vsn_attn_backward(None, C.byref(io), C.byref(g), None, 0, None) == -22
    L.vsn_attn_destroy(None)
    if not torch.cuda.is_available():
        assert create() == -19


def test_attention_plan_refuses_in_python():
    from ai2bmd_amd.attention import FragmentAttention
    with pytest.raises(RuntimeError, match="cuda"):
        FragmentAttention([0], [4], 2, 8, device="cpu")
    for bad in (dict(start=[1], end=[4]), dict(start=[0, 5], end=[4, 6]), dict(start=[], end=[]), dict(start=[0], end=[[4]]),
                dict(heads=3, num_kv_heads=2), dict(dim=12), dict(dim=136), dict(dim=0), dict(buckets=[0, 1]), dict(buckets=[0, -1, 0]),
                dict(buckets=[0] * 2049), dict(buckets=[0, 1, 2], num_buckets=2), dict(buckets=[0], num_buckets=5000), dict(query_start=[0]),
                dict(query_start=[0, 1], query_end=[1, 2])):
        a = dict(start=[0], end=[4], heads=2, dim=8)
        a.update(bad)
        with pytest.raises(ValueError):
            FragmentAttention(a.pop("start"), a.pop("end"), a.pop("heads"), a.pop("dim"), **a)


def test_relative_buckets():
    from ai2bmd_amd.attention import relative_buckets
    assert relative_buckets(9, 4).tolist() == list(range(9))
    assert relative_buckets(3, 0).tolist() == [0]
    b = relative_buckets(32, 128)
    assert len(b) == 257 and b[128] == 0 and b.min() == 0 and b.max() == 31
    assert b[128 - 7:128][::-1].tolist() == [1, 2, 3, 4, 5, 6, 7] and b[129:136].tolist() == [17, 18, 19, 20, 21, 22, 23]
    back, ahead = b[:128][::-1], b[129:]
    assert (ahead == back + 16).all() and (back[1:] >= back[:-1]).all()
    # the border of bucket 8 + n lies at 8 * 16^(n / 8): 16 ^ (1 / 2) = 4 gives 32 for n = 4, 8 * 16^(1 / 8) = 11.3 for n = 1
    assert back[31 - 1] == 11 and back[32 - 1] == 12 and back[11 - 1] == 8 and back[12 - 1] == 9 and back[128 - 1] == 15
    for bad in ((31, 128), (2, 128), (0, 4), (32, 1024), (32, -1)):
        with pytest.raises(ValueError):
            relative_buckets(*bad)


def test_plans_that_no_launch_could_count_are_refused(lib_built):
    """2^32 threads along an axis: 2^26 waves of 64.  Fragments of one row with 1024 heads (too many heads for the kernel of
    one-tile fragments): a wave per fragment and head."""
    import numpy as np

    from ai2bmd_amd import capi
    L = capi.lib()

    def create(n, heads, rows=1):
        end = np.arange(1, n + 1, dtype=np.int64) * rows
        h = C.c_void_p()
        rc = L.vsn_attn_create(C.byref(h), 0, n, capi.i64_ptr(end - rows), capi.i64_ptr(end), None, None, heads, heads, 8, 0, None, 0)
        if rc == 0:
            L.vsn_attn_destroy(h)
        return rc

    fits = 0 if torch.cuda.is_available() else -19
    assert create(65535, 1024) == fits and create(65536, 1024) == -22
    # workgroups of four waves that share the tiles of 128 rows: 2^24 of them
    assert create(16383, 1024, 65) == fits and create(16384, 1024, 65) == -22
    # one-tile fragments by the million: one wave walks all heads
    assert create(8_500_000, 8) == fits
