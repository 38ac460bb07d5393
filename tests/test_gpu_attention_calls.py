"""GPU: calls of fragment attention that its header allows or refuses, at the C boundary, and launch shapes of large batches."""
import ctypes as C

import pytest
import torch

from test_gpu_attention import CLIP, COARSE, TYPES, Case

pytestmark = pytest.mark.gpu


def backward(case, plan, flags=1, less=0, **change):
    """vsn_attn_backward with every gradient of the case, `change`d -> (code, gradients, bytes of workspace)"""
    from ai2bmd_amd import capi
    lib = capi.lib()
    out, stats = plan.forward(case.q, case.k, case.v, save=True, **case.terms)
    t = case.terms
    io, held = plan._io(case.q, case.k, case.v, t.get("pos"), t.get("slope"), t.get("residue"), t.get("table"), t.get("query_pos"),
                        t.get("query_residue"), None)
    io.stats = stats.data_ptr()
    f32 = dict(device="cuda")
    made = dict(dq=torch.empty_like(case.q), dk=torch.empty_like(case.k), dv=torch.empty_like(case.v),
                dpos=torch.empty(case.k.shape[0], 3, **f32), dquery_pos=torch.empty(case.q.shape[0], 3, **f32),
                dslope=torch.empty(case.heads, **f32), dtable=torch.empty(case.heads, max(plan.num_buckets, 1), **f32))
    if not case.apart:
        made["dquery_pos"] = None
    for name, value in change.items():
        if name in made:
            made[name] = value
        else:
            setattr(io, name, value)
    g = capi.VsnAttnGrads(case.dout.data_ptr(), case.dout.stride(0), case.dout.stride(1),
                          *(0 if made[n] is None else made[n].data_ptr() for n in ("dq", "dk", "dv", "dpos", "dquery_pos", "dslope", "dtable")))
    size = lib.vsn_attn_workspace(plan._h, case.q.shape[0], case.k.shape[0], flags)
    assert size >= 0
    work = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    rc = lib.vsn_attn_backward(plan._h, C.byref(io), C.byref(g), work.data_ptr(), size - less, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return rc, made, size


def test_one_gradient_for_both_ends_only_where_the_rows_are_the_same():
    # ranges of their own, of the same total: dpos alone is refused, dpos with dquery_pos is not
    for queries, code in (([5, 3], -22), ([3, 5], -22)):
        case = Case([3, 5], torch.float32, heads=2, dim=16, lut=CLIP, queries=queries)
        plan = case.plan()
        assert backward(case, plan, dquery_pos=None)[0] == code
        rc, made, _ = backward(case, plan)
        want = case.results(plan)
        assert rc == 0 and all(torch.equal(made[n], want[n]) for n in ("dq", "dk", "dv", "dpos", "dquery_pos", "dslope", "dtable"))
    # the same ranges and the same positions, given twice
    both = Case([3, 5], torch.float32, heads=2, dim=16, lut=CLIP)
    apart = Case([3, 5], torch.float32, heads=2, dim=16, lut=CLIP, queries=[3, 5])
    apart.q, apart.k, apart.v, apart.dout = both.q, both.k, both.v, both.dout
    apart.terms = {**both.terms, "query_pos": both.terms["pos"], "query_residue": both.terms["residue"]}
    rc, made, _ = backward(apart, apart.plan(), dquery_pos=None)
    assert rc == 0 and torch.equal(made["dpos"], both.results()["dpos"])


def test_a_refused_device_leaves_no_error_behind():
    from ai2bmd_amd.attention import FragmentAttention
    from ai2bmd_amd import capi
    from ai2bmd_amd.norm import layer_norm
    x = torch.randn(4, 64, device="cuda")
    for _ in range(2):
        with pytest.raises(RuntimeError, match="-19"):
            FragmentAttention([0], [4], 2, 8, device="cuda:99")
        layer_norm(x)
        assert capi.lib().vsn_layernorm(99, 0, 0, x.data_ptr(), 64, None, None, 4, 64, 1e-5, x.data_ptr(), 64, None, None) == -19
        assert (x + 1).isfinite().all()


def test_statistics_of_rows_behind_the_last_fragment_are_zeros():
    case = Case([20, 45], torch.float32, extra=5)
    plan = case.plan()
    for _ in range(3):
        torch.full((8, 70, 2), 7.0, device="cuda")  # memory that the next allocation takes over
        _, stats = plan.forward(case.q, case.k, case.v, save=True, **case.terms)
        assert not stats[:, 65:].any() and (stats[:, :65, 1] > 0).all()


def test_workspace_is_for_the_terms_that_a_call_has():
    case = Case([150, 12, 60, 400], torch.float32, heads=4, dim=16, lut=list(range(257)))
    plan = case.plan()
    every = ("dq", "dk", "dv", "dpos", "dslope", "dtable")
    rc, want, full = backward(case, plan)
    assert rc == 0 and backward(case, plan, less=1)[0] == -22
    partial = {2: dict(dpos=None), 4: dict(dtable=None), 6: dict(dpos=None, dtable=None)}
    sizes = {}
    for flags, without in partial.items():
        rc, made, sizes[flags] = backward(case, plan, flags=1 | flags, **without)
        assert rc == 0 and all(torch.equal(made[n], want[n]) for n in every if made[n] is not None)
        assert backward(case, plan, flags=1 | flags, less=1, **without)[0] == -22
    assert sizes[6] < sizes[2] < full and sizes[6] < sizes[4] < full
    assert full - sizes[4] >= 4 * 257 * 4 and full - sizes[2] >= 622 * 4 * 24   # the table's sums; the positions' of both sides
    assert backward(case, plan, flags=3)[0] == backward(case, plan, flags=5)[0] == -22     # too small for what is asked
    assert plan._L.vsn_attn_workspace(plan._h, 622, 622, 8) == plan._L.vsn_attn_workspace(plan._h, 622, 622, -1) == -22


# Launch shapes of large batches: a worker of the backward passes takes a second item (from 4096 one-tile fragments, 4096 / heads
# two-tile ones, 4096 / heads runs of 32 rows, 2048 / heads with a table or of 128 shared rows), and workgroups hold several
# waves with LDS of their own (one-tile fragments from 1024 waves on, the others always).

@pytest.mark.parametrize("T", TYPES, ids=str)
def test_more_one_tile_fragments_than_workers(T):
    Case([1 + (7 * i) % 32 for i in range(4500)], T, heads=2, dim=8, lut=COARSE).check()


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("lut", [None, COARSE], ids=["slope", "table"])
def test_more_two_tile_fragments_than_workers(T, lut):
    Case([33 + i % 12 for i in range(700)], T, dim=16, lut=lut).check()


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("kv,dim", [(8, 72), (2, 24)])
def test_more_runs_of_32_rows_than_workers_and_several_waves_a_workgroup(T, kv, dim):
    Case([33 + (5 * i) % 32 for i in range(1100)], T, kv=kv, dim=dim, lut=COARSE).check()


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("dim", [16, 64])
def test_more_shared_tiles_than_workers(T, dim):
    Case([65 + (11 * i) % 90 for i in range(300)], T, dim=dim, lut=COARSE).check()


@pytest.mark.parametrize("T", TYPES, ids=str)
def test_thousands_of_keys(T):
    Case([9001, 700], T, heads=2, dim=16, lut=COARSE).check()


@pytest.mark.parametrize("sizes,step", [([64], 1 << 25), ([30, 34], 1 << 25), ([4101], 1 << 20), ([300, 3801], 1 << 20)])
def test_offsets_beyond_32_bits(sizes, step):
    """rows up to 2^25 elements apart: a tile's offsets pass 2^31 elements, an array's 2^32"""
    case = Case(sizes, torch.bfloat16, heads=2, dim=16, lut=CLIP)
    plan = case.plan()
    want = case.results(plan)
    for name in ("q", "k", "v", "dout"):
        rows = getattr(case, name)
        wide = torch.empty((rows.shape[0] - 1) * step + 32, dtype=torch.bfloat16, device="cuda").as_strided((rows.shape[0], 2, 16), (step, 16, 1))
        setattr(case, name, wide.copy_(rows))
        assert plan._rows(wide, name, 2, 0, torch.bfloat16) is wide  # read in place
    got = case.results(plan)
    assert all(torch.equal(got[n], want[n]) for n in want)
