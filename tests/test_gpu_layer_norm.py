"""GPU: layer norm (ai2bmd_amd/norm.py) against its formula in 64 bits: types, widths, strides, empty and single rows,
gradients against differences, other streams, captured graphs.

Tolerances.  A value rounded to type T is off by at most u = eps(T) / 2 of itself.  Before that everything is float32:
a sum of n terms in s steps is off by at most s 2^-24 sum|terms|; a row's sums take width / lanes + 6 <= 70 steps, so the
mean is off by at most 70 2^-24 A (A = max|x| of the row) and, through rstd, h by K (A rstd + |h| + 1) with K = 100 2^-24
(70 for the mean, the rest for the square sum, the root and five products)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
K = 100 * 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def unit(t):
    return torch.finfo(t).eps / 2


def formula(x, w, b, dy, eps=1e-5):
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    h = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    rows = tuple(range(x.dim() - 1))
    return h * w + b, dx, (dy * h).sum(rows), dy.sum(rows), h, rstd, w, b


def check(x, w, b, dy, y, grads):
    T = x.dtype
    y64, dx64, dw64, db64, h, rstd, w64, b64 = formula(x, w, b, dy)
    spread = x.double().abs().amax(-1, keepdim=True) * rstd + h.abs() + 1
    assert ((y.double() - y64).abs() <= unit(T) * y64.abs() * (1 + K) + K * spread * (w64.abs() + b64.abs()) + 1e-7).all()
    dx, dw, db = grads
    g = (dy.double() * w64).abs()
    # dx: three terms, each with the row's sums (70 steps) and h's error in it
    top = g.amax(-1, keepdim=True) * rstd * spread.amax(-1, keepdim=True) * (h.abs().amax(-1, keepdim=True) + 1)
    assert ((dx.double() - dx64).abs() <= unit(T) * dx64.abs() * (1 + K) + 4 * K * top + 1e-7).all()
    rows = x.numel() // x.shape[-1]
    steps = rows / 1024 + 32 + 1024 / 8 + 8  # rows of a lane, row groups of a workgroup, workgroups of the second launch
    size = (dy.double().abs() * (h.abs() + spread)).sum(tuple(range(x.dim() - 1)))
    for got, want, p in ((dw, dw64, w), (db, db64, b)):
        if p is None:
            assert got is None
        else:
            assert got.dtype == p.dtype and got.shape == p.shape
            limit = unit(p.dtype) * want.abs() * (1 + K) + (steps * 2.0 ** -24 + K) * (size + dy.double().abs().sum(tuple(range(x.dim() - 1))))
            assert ((got.double() - want).abs() <= limit + 1e-7).all()


def normal(*shape, dtype, seed, spread=1.0, shift=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * spread + shift).to(dtype)


def make(rows, width, T, seed, param=None):
    P = param or T
    return (normal(rows, width, dtype=T, seed=seed, spread=2.0, shift=0.5), normal(width, dtype=P, seed=seed + 1, shift=1.0, spread=0.3),
            normal(width, dtype=P, seed=seed + 2, spread=0.3), normal(rows, width, dtype=T, seed=seed + 3))


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 256), (3, 7), (5, 64), (33, 65), (175, 256), (257, 509), (64, 512), (130, 1000),
                                        (9, 1025), (17, 2049), (2, 4095), (3, 4096), (5003, 256), (9001, 67)])
def test_sizes_and_types(T, rows, width):
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(rows, width, T, rows * 7 + width)
    y, stats = layer_norm(x, w, b)
    check(x, w, b, dy, y, layer_norm_backward(dy, x, stats, w, b))


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float16], ids=str)
def test_float32_parameters_and_absent_ones(T):
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(77, 192, T, 5, param=torch.float32)
    for pw, pb in ((w, b), (w, None), (None, b), (None, None)):
        y, stats = layer_norm(x, pw, pb)
        check(x, pw, pb, dy, y, layer_norm_backward(dy, x, stats, pw, pb))


@pytest.mark.parametrize("T", TYPES, ids=str)
def test_strides_and_orders(T):
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(60, 96, T, 9)
    y0, s0 = layer_norm(x, w, b)
    g0 = layer_norm_backward(dy, x, s0, w, b)
    wide = normal(60, 101, dtype=T, seed=1)
    wide[:, 3:99] = x
    layouts = [wide[:, 3:99],                                   # rows 101 elements apart, first element at an odd address
               x.t().contiguous().t(),                          # columns apart
               x.view(4, 15, 96).transpose(0, 1).contiguous().transpose(0, 1)]  # leading axes out of order
    for other in layouts:
        y, stats = layer_norm(other, w, b)
        assert torch.equal(y.reshape(60, 96), y0) and torch.equal(stats, s0)
        grad = dy.view(other.shape)
        dx, dw, db = layer_norm_backward(grad.transpose(-1, -2).contiguous().transpose(-1, -2), other, stats, w, b)
        assert torch.equal(dx.reshape(60, 96), g0[0]) and torch.equal(dw, g0[1]) and torch.equal(db, g0[2])
    one = torch.ones(1, 1, dtype=T, device="cuda").expand(60, 96)  # a broadcast gradient: every stride 0
    check(x, w, b, one, y0, layer_norm_backward(one, x, s0, w, b))


def test_no_rows_and_in_place_output():
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(0, 128, torch.float32, 3)
    y, stats = layer_norm(x, w, b)
    dx, dw, db = layer_norm_backward(dy, x, stats, w, b)
    assert y.shape == dx.shape == (0, 128) and not dw.any() and not db.any()
    x, w, b, _ = make(40, 128, torch.float32, 4)
    y, _ = layer_norm(x, w, b)
    assert layer_norm(x, w, b, out=x)[0] is x and torch.equal(x, y)


def test_a_bad_row_stays_its_own_and_constant_rows_are_finite():
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(70, 64, torch.float32, 6)
    x[3] = float("nan")
    x[4, 5] = float("inf")
    x[5] = 7.0
    y, stats = layer_norm(x, w, b)
    dx, _, _ = layer_norm_backward(dy, x, stats, w, b)
    good = torch.ones(70, dtype=torch.bool, device="cuda")
    good[3:5] = False
    assert torch.isfinite(y[good]).all() and torch.isfinite(dx[good]).all()
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).any()
    assert torch.equal(y[5], b)


def test_gradient_against_differences():
    """central differences of sum(y dy) in the 64-bit formula, step 1e-4: off by h^2 |f'''| / 6 < 1e-6 here; the kernel's
    own error is below 1e-5 for these O(1) values (K times the sizes above)."""
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(6, 48, torch.float32, 8)
    _, stats = layer_norm(x, w, b)
    dx, dw, db = layer_norm_backward(dy, x, stats, w, b)
    value = lambda x_, w_, b_: (formula(x_, w_, b_, dy)[0] * dy.double()).sum()
    for at in ((0, 0), (3, 17), (5, 47)):
        step = torch.zeros(6, 48, dtype=torch.float64, device="cuda")
        step[at] = 1e-4
        assert abs((value(x + step, w, b) - value(x - step, w, b)) / 2e-4 - dx[at]) < 1e-4
    for c in (0, 20, 47):
        step = torch.zeros(48, dtype=torch.float64, device="cuda")
        step[c] = 1e-4
        assert abs((value(x, w + step, b) - value(x, w - step, b)) / 2e-4 - dw[c]) < 1e-4
        assert abs((value(x, w, b + step) - value(x, w, b - step)) / 2e-4 - db[c]) < 1e-4


def test_repeats_streams_and_graph_replays():
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(3001, 256, torch.bfloat16, 12)
    y0, s0 = layer_norm(x, w, b)
    g0 = layer_norm_backward(dy, x, s0, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, stats = layer_norm(x, w, b)
        g = layer_norm_backward(dy, x, stats, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, y0) and all(torch.equal(p, q) for p, q in zip(g, g0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, stats = layer_norm(x, w, b)
        g = layer_norm_backward(dy, x, stats, w, b)
    for seed in (21, 22, 23):
        x.copy_(normal(3001, 256, dtype=torch.bfloat16, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        ye, se = layer_norm(x, w, b)
        ge = layer_norm_backward(dy, x, se, w, b)
        torch.cuda.synchronize()
        assert torch.equal(y, ye) and all(torch.equal(p, q) for p, q in zip(g, ge))


def test_refusals():
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(8, 64, torch.bfloat16, 2)
    _, stats = layer_norm(x, w, b)
    for bad in (lambda: layer_norm(x.double()), lambda: layer_norm(x, w[:32]), lambda: layer_norm(x, w.half()),
                lambda: layer_norm(x, w, b.float()), lambda: layer_norm(x, w.cpu()), lambda: layer_norm(x, eps=-1.0),
                lambda: layer_norm(x, out=torch.empty(8, 64, device="cuda")), lambda: layer_norm(torch.zeros(2, 4097, device="cuda")),
                lambda: layer_norm(torch.zeros(2, 0, device="cuda")), lambda: layer_norm_backward(dy[:4], x, stats, w, b),
                lambda: layer_norm_backward(dy, x, stats[:4], w, b), lambda: layer_norm_backward(dy.float(), x, stats, w, b)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="autograd"):
        layer_norm(x, w.requires_grad_(), b)
    with torch.no_grad():
        layer_norm(x, w, b)


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("width", [5, 8, 9, 15, 17, 31, 63, 129, 255, 511, 1023, 4095])
@pytest.mark.parametrize("own_params", [True, False])
def test_rows_that_end_within_a_vector(T, width, own_params):
    """a row between poisoned columns: what is loaded next to it must not count, and what is next to it stays"""
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(37, width, T, width, param=T if own_params else torch.float32)
    inside = [torch.full((37, width + 5), float("nan"), dtype=T, device="cuda") for _ in range(2)]
    for wide, rows in zip(inside, (x, dy)):
        wide[:, 2:2 + width] = rows
    xs, dys = (wide[:, 2:2 + width] for wide in inside)
    params = torch.full((2, width + 2), float("nan"), dtype=w.dtype, device="cuda")
    params[0, 1:-1], params[1, 1:-1] = w, b
    ws, bs = params[0, 1:-1], params[1, 1:-1]
    out = torch.full((39, width), 7.0, dtype=T, device="cuda")
    y, stats = layer_norm(xs, ws, bs, out=out[1:38])
    check(x, w, b, dy, y, layer_norm_backward(dys, xs, stats, ws, bs))
    assert (out[0] == 7).all() and (out[38] == 7).all()
    again = x.clone()
    assert torch.equal(layer_norm(again, w, b, out=again)[0], y)


@pytest.mark.parametrize("rows,width", [(140_001, 256), (33_001, 1024), (530_001, 64), (33_001, 1025)])
def test_float32_rows_beyond_the_cache(rows, width):
    from ai2bmd_amd.norm import layer_norm, layer_norm_backward
    x, w, b, dy = make(rows, width, torch.float32, 11)
    y, stats = layer_norm(x, w, b)
    check(x, w, b, dy, y, layer_norm_backward(dy, x, stats, w, b))
    assert torch.equal(layer_norm(x[-7:], w, b)[0], y[-7:])
