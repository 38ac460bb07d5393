"""GPU: calls of the layer norm that its header or docstring allows: in place, many rows, parameters on either side."""
import pytest
import torch

from test_gpu_layer_norm import TYPES, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("rows,width,ld", [(37, 256, 256), (3001, 256, 261), (37, 509, 509), (9001, 67, 70), (5, 4095, 4095), (700, 12, 12)])
def test_the_rows_gradient_may_take_the_place_of_dy(T, rows, width, ld):
    """vsn_layernorm_backward with dx = dy gives the bits of a call with an array of its own, and leaves what lies between
    the rows"""
    from ai2bmd_amd import capi
    from ai2bmd_amd.norm import DTYPE, layer_norm, layer_norm_backward
    x, w, b, dy = make(rows, width, T, rows + width)
    _, stats = layer_norm(x, w, b)
    dx, dw, db = layer_norm_backward(dy, x, stats, w, b)
    wide = torch.full((rows, ld), 7.0, dtype=T, device="cuda")
    wide[:, :width] = dy
    gw, gb = torch.empty_like(w), torch.empty_like(b)
    lib = capi.lib()
    size = lib.vsn_layernorm_workspace(rows, width)
    work = torch.empty(size // 4, device="cuda")
    code = DTYPE[T]
    assert lib.vsn_layernorm_backward(0, code, code, wide.data_ptr(), ld, x.data_ptr(), width, stats.data_ptr(), w.data_ptr(), rows,
                                      width, wide.data_ptr(), ld, gw.data_ptr(), gb.data_ptr(), work.data_ptr(), size,
                                      torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(wide[:, :width], dx) and torch.equal(gw, dw) and torch.equal(gb, db) and (wide[:, width:] == 7).all()


@pytest.mark.parametrize("T", TYPES[1:], ids=str)
@pytest.mark.parametrize("rows,width", [(40_001, 256), (20_011, 509), (70_003, 33), (300_007, 8), (9_001, 4096)])
def test_16_bit_rows_that_are_walked_in_several_turns(T, rows, width):
    """more rows than 2048 (forward) and 1024 (backward) workgroups take in one turn"""
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(rows, width, T, 17)
    y, stats = layer_norm(x, w, b)
    check(x, w, b, dy, y, layer_norm_backward(dy, x, stats, w, b))
    for at in (0, rows // 2, rows - 9):
        assert torch.equal(layer_norm(x[at:at + 9], w, b)[0], y[at:at + 9])


def test_outputs_and_tangents_of_a_graph_are_refused():
    from torch.autograd import forward_ad

    from ai2bmd_amd.attention import FragmentAttention
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(8, 64, torch.float32, 2)
    _, stats = layer_norm(x, w, b)
    leaf = torch.zeros(8, 64, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="autograd"):
        layer_norm(x, w, b, out=leaf)
    with torch.no_grad():
        assert layer_norm(x, w, b, out=leaf)[0] is leaf
    plan = FragmentAttention([0], [8], 2, 32)
    rows = x.view(8, 2, 32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: layer_norm(dual, w, b), lambda: layer_norm(x, forward_ad.make_dual(w, w), b), lambda: layer_norm_backward(dual, x, stats, w, b),
                     lambda: plan.forward(rows, dual.view(8, 2, 32), rows)):
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call()


def test_an_output_that_overlaps_its_rows_is_refused():
    from ai2bmd_amd.norm import layer_norm
    wide = torch.randn(12, 64, device="cuda")
    flat = wide.view(-1)
    part = wide[:10, :32]  # rows 64 apart: an output of rows 32 apart at the same address would meet rows not read yet
    for x, out in ((part, flat[:320].view(10, 32)), (wide[:10], flat[64:704].view(10, 64)), (wide[2:12], flat[64:704].view(10, 64)),
                   (part, flat[5:325].view(10, 32))):
        with pytest.raises(ValueError, match="overlap"):
            layer_norm(x, out=out)
    want = layer_norm(wide[:5])[0]
    assert torch.equal(layer_norm(wide[:5], out=wide[5:10])[0], want)       # side by side
    assert torch.equal(layer_norm(wide[:5], out=flat[:320].view(5, 64))[0], want) and torch.equal(wide[:5], want)
    columns = torch.randn(32, 10, device="cuda")                             # copied first: may be written over
    want = layer_norm(columns.t())[0]
    assert torch.equal(layer_norm(columns.t(), out=columns.view(10, 32))[0], want)


def test_offsets_beyond_32_bits():
    """2^31 elements and more, by many rows and by rows far apart"""
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    for rows, width, step in ((8_400_001, 256, 256), (2_101, 300, 1 << 20)):
        few = 2_000
        x, w, b, dy = make(few, width, torch.bfloat16, 5)
        y, stats = layer_norm(x, w, b)
        dx = layer_norm_backward(dy, x, stats, w, b)[0]
        xs, dys = (torch.empty((rows - 1) * step + width, dtype=torch.bfloat16, device="cuda").as_strided((rows, width), (step, 1)) for _ in range(2))
        for wide, part in ((xs, x), (dys, dy)):
            if step == width:
                wide.zero_()
            else:
                wide[:rows - few] = part[:rows - few]
            wide[-few:] = part
        out, st = layer_norm(xs, w, b)
        grads = layer_norm_backward(dys, xs, st, w, b)
        assert torch.equal(out[-few:], y) and torch.equal(st[-few:], stats) and torch.equal(grads[0][-few:], dx)
        del xs, dys, out, grads


@pytest.mark.parametrize("rows,width", [(180_001, 192), (110_001, 320), (360_001, 96), (270_001, 128), (90_001, 384)])
def test_float32_rows_beyond_the_cache_of_any_width(rows, width):
    """widths on both sides of the launch rule: lanes of a row all full, and not"""
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(rows, width, torch.float32, 11)
    y, stats = layer_norm(x, w, b)
    check(x, w, b, dy, y, layer_norm_backward(dy, x, stats, w, b))
    assert torch.equal(layer_norm(x[-7:], w, b)[0], y[-7:])


def test_lazily_negated_views_are_refused():
    """their memory holds the values before the negation"""
    from ai2bmd_amd.attention import FragmentAttention
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(8, 64, torch.float32, 2)
    _, stats = layer_norm(x, w, b)
    neg = torch._neg_view
    plan = FragmentAttention([0], [8], 2, 32)
    rows, pos, slope = x.view(8, 2, 32), x[:, :3].contiguous(), w[:2].contiguous()
    for call in (lambda: layer_norm(neg(x), w, b), lambda: layer_norm(x, neg(w), b), lambda: layer_norm(x, w, neg(b)), lambda: layer_norm(x, out=neg(dy)),
                 lambda: layer_norm_backward(neg(dy), x, stats, w, b), lambda: layer_norm_backward(dy, x, neg(stats), w, b),
                 lambda: plan.forward(neg(rows), rows, rows), lambda: plan.forward(rows, neg(rows), rows), lambda: plan.forward(rows, rows, neg(rows)),
                 lambda: plan.forward(rows, rows, rows, pos=neg(pos), slope=slope), lambda: plan.forward(rows, rows, rows, pos=pos, slope=neg(slope))):
        with pytest.raises(ValueError, match="negated"):
            call()
    assert torch.equal(layer_norm(neg(x).resolve_neg(), w, b)[0], layer_norm(-x, w, b)[0])
