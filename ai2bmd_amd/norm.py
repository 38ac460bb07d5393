"""Layer norm on the MI355X as an operator, forward and backward with the gradients of weight and bias.

The norm of the reference's ViS-MP layer (torch.nn.LayerNorm, ViSNet/model/visnet_block.py:180,237), for rows of atoms or
edges outside the force engine, which holds the same norm fused and frozen: a layer that is trained needs dx, dw and db.
Like everything here it is differentiated by hand: the two functions are called explicitly and build no autograd graph.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import capi

MAX_WIDTH = 4096
DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # VSN_F32, VSN_BF16, VSN_F16 (include/vsn.h)


def dtype_code(t: torch.Tensor, name: str) -> int:
    code = DTYPE.get(t.dtype)
    if code is None:
        raise ValueError(f"{name}: float32, bfloat16 or float16 expected, not {t.dtype}")
    return code


def on_device(t: torch.Tensor, name: str, device=None) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name}: this package is the MI355X path ('cuda:<k>' tensors only), got one on {t.device}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.is_neg():  # its memory holds the negated values, and the kernels read memory
        raise ValueError(f"{name}: a lazily negated view; call resolve_neg() first")


def no_graph(*tensors) -> None:
    """The operators build no autograd graph and carry no tangent; a result that silently cut one would train nothing."""
    if forward_ad._current_level >= 0:  # (within forward_ad.dual_level: the tensors have to be looked at)
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("no tangent is computed: forward-mode differentiation is not supported")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("no autograd graph is built: call under torch.no_grad() and use the backward function")


def ptr(t):
    return t.data_ptr() if t is not None else None


def stream_of(t: torch.Tensor) -> int:
    """The current stream of the tensor's device, without the Stream object that torch.cuda.current_stream makes (3 us)."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _rows(t: torch.Tensor, width: int):
    """(tensor, rows, elements between rows): the tensor as it is where its rows are evenly spaced, else a copy."""
    rows = t.numel() // width
    if t.is_contiguous() or rows == 0:
        return t, rows, width
    if t.stride(-1) == 1 or width == 1:
        lead = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
        if all(lead[i][1] == lead[i + 1][0] * lead[i + 1][1] for i in range(len(lead) - 1)):
            step = lead[-1][1] if lead else width
            if step >= width:
                return t, rows, step
    return t.contiguous(), rows, width


def _span(t: torch.Tensor):
    """first address of a tensor and the one behind its last element"""
    first = t.data_ptr()
    if not t.numel():
        return first, first
    return first, first + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _param(p, x, name: str) -> None:
    if not p.is_cuda or p.device != x.device or p.is_neg():
        on_device(p, name, x.device)
    if p.shape != x.shape[-1:] or not p.is_contiguous():
        raise ValueError(f"{name}: contiguous [{x.shape[-1]}] expected, got {tuple(p.shape)}")
    if p.dtype != x.dtype and p.dtype != torch.float32:
        raise ValueError(f"{name}: {x.dtype} or float32 expected, not {p.dtype}")


def _check(x, weight, bias):
    """(width, type codes of the rows and of the parameters)"""
    on_device(x, "x")
    code = dtype_code(x, "x")
    width = x.shape[-1] if x.dim() else 0
    if not 1 <= width <= MAX_WIDTH:
        raise ValueError(f"x: a last axis of 1 ... {MAX_WIDTH} expected, got {tuple(x.shape)}")
    if weight is not None:
        _param(weight, x, "weight")
    if bias is not None:
        _param(bias, x, "bias")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias differ in type")
    of = weight if weight is not None else bias
    return width, code, code if of is None else DTYPE[of.dtype]


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, out=None):
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis -> (y, stats).

    `x` [..., width], float32 / bfloat16 / float16; evenly spaced rows are read in place, other layouts are copied.
    `weight`, `bias` [width] of x's type or float32 (None: 1 and 0).  `out`: contiguous, of x's shape and type; x itself,
    or apart from all inputs.
    `stats` float32 [rows, 2] (mean, 1 / sqrt(var + eps)) goes to layer_norm_backward.  On the current stream of x's device."""
    width, code, param_code = _check(x, weight, bias)
    no_graph(x, weight, bias, out)
    if not eps >= 0:
        raise ValueError("eps: a number >= 0 expected")
    if out is not None:
        on_device(out, "out", x.device)
        if out.shape != x.shape or out.dtype != x.dtype or not out.is_contiguous():
            raise ValueError("out: contiguous, with x's shape and type expected")
    y = x.new_empty(x.shape) if out is None else out
    src, rows, ld = _rows(x, width)
    if out is not None:
        (o0, o1), (x0, x1) = _span(out), _span(src)
        if o0 < x1 and x0 < o1 and not (o0 == x0 and ld == width):
            raise ValueError("out: x itself or memory apart from it expected (their rows overlap)")
    stats = torch.empty(rows, 2, dtype=torch.float32, device=x.device)
    rc = capi.lib().vsn_layernorm(x.device.index, code, param_code, src.data_ptr(), ld, ptr(weight), ptr(bias), rows,
                                  width, eps, y.data_ptr(), width, stats.data_ptr(), stream_of(x))
    if rc:
        raise RuntimeError(f"vsn_layernorm failed ({rc})")
    return y, stats


def layer_norm_backward(dy, x, stats, weight=None, bias=None):
    """Gradients (dx, dweight, dbias) of layer_norm at `x`, with the `stats` it returned, from dy = dL/dy.

    dweight / dbias have the parameters' type and are None where the parameter is.  Sums run in a fixed order."""
    width, code, param_code = _check(x, weight, bias)
    no_graph(dy, x, stats, weight, bias)
    on_device(dy, "dy", x.device)
    on_device(stats, "stats", x.device)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("dy: x's shape and type expected")
    src, rows, ld = _rows(x, width)
    if stats.shape != (rows, 2) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError(f"stats: contiguous float32 [{rows}, 2] expected")
    grad, _, ldg = _rows(dy, width)
    dx = x.new_empty(x.shape)
    dw = torch.empty_like(weight) if weight is not None else None
    db = torch.empty_like(bias) if bias is not None else None
    lib = capi.lib()
    size = lib.vsn_layernorm_workspace(rows, width) if weight is not None or bias is not None else 0
    work = torch.empty(size // 4, dtype=torch.float32, device=x.device) if size else None
    rc = lib.vsn_layernorm_backward(x.device.index, code, param_code, grad.data_ptr(), ldg, src.data_ptr(), ld,
                                    stats.data_ptr(), ptr(weight), rows, width, dx.data_ptr(), width, ptr(dw), ptr(db),
                                    ptr(work), size, stream_of(x))
    if rc:
        raise RuntimeError(f"vsn_layernorm_backward failed ({rc})")
    return dx, dw, db
