"""Fragment attention on the MI355X: softmax attention among all atoms of a fragment, forward and backward.

The engine's attention (ViSNet/model/visnet_block.py:276-312) runs over at most 32 neighbours inside the cutoff, without a
softmax and with frozen weights.  A layer that lets every atom of a fragment - or of a whole protein - see every other one
has scores

    s_ij = scale q_i.k_j - slope_h |x_i - x_j| + table[h, bucket(residue_j - residue_i)]

over the rows of one fragment (FragmentData.start / end): a slope per head that lowers a score with the distance, and a
learned bias per head and bucket of the residue offset; both are optional.  Like everything here it is differentiated by
hand: `forward` and `backward` are called explicitly and build no autograd graph.
"""
from __future__ import annotations

import ctypes as C
from collections import namedtuple

import numpy as np
import torch

from . import capi
from .norm import dtype_code, no_graph, on_device, ptr, stream_of

MAX_REACH, MAX_BUCKETS, MAX_ROW_STEP, MAX_ROWS, MAX_HEADS = 1023, 4096, 1 << 25, 1 << 30, 1024
BACKWARD, NO_POS, NO_TABLE = 1, 2, 4  # VSN_ATTN_* (include/vsn.h)
AttentionGrads = namedtuple("AttentionGrads", "dq dk dv dpos dquery_pos dslope dtable")


def relative_buckets(num_buckets: int, reach: int) -> np.ndarray:
    """int32 [2 reach + 1]: the bucket of every residue offset clipped to -reach ... reach.

    With num_buckets >= 2 reach + 1 every offset has its own; else each direction has half of them (an even number), the
    near offsets one each and the others in logarithmically growing steps, the last bucket holding all from there on."""
    if not 0 <= reach <= MAX_REACH or num_buckets < 1:
        raise ValueError(f"relative_buckets: reach 0 ... {MAX_REACH} and at least one bucket expected")
    offset = np.arange(-reach, reach + 1)
    if num_buckets >= 2 * reach + 1:
        return (offset + reach).astype(np.int32)
    half, near = num_buckets // 2, num_buckets // 4
    if num_buckets % 2 or near < 1 or reach <= near:
        raise ValueError("relative_buckets: an even number of buckets, at least 4, expected (or 2 reach + 1 of them)")
    bucket = []
    for far in range(reach + 1):
        # the largest n < half - near with (far / near)^(half - near) >= (reach / near)^n, in whole numbers: an offset that
        # lies on a border must not depend on a logarithm's last bit
        n = 0
        while far >= near and n + 1 < half - near and \
                far ** (half - near) * near ** (n + 1) >= near ** (half - near) * reach ** (n + 1):
            n += 1
        bucket.append(far if far < near else near + n)
    return (np.asarray(bucket)[np.abs(offset)] + np.where(offset > 0, half, 0)).astype(np.int32)


def _whole(a, name: str, dtype) -> np.ndarray:
    """one-dimensional array of whole numbers in `dtype`; a conversion that would change a value is refused"""
    a = np.asarray(a)
    if a.ndim != 1 or a.dtype.kind not in "iuf":
        raise ValueError(f"{name}: one-dimensional array of whole numbers expected")
    with np.errstate(invalid="ignore"):
        to = np.ascontiguousarray(a, dtype=dtype)
    if (to != a).any():
        raise ValueError(f"{name}: whole numbers in the range of {np.dtype(dtype).name} expected")
    return to


class FragmentAttention:
    """The plan of one batch layout: which rows belong together, heads, and the bucket map.

    `start`, `end` [B]: first and one-past-last row of every fragment, contiguous and ascending from 0 (FragmentData's).
    `query_start`, `query_end`: rows of the query array, where queries are not the fragment's own rows (one read-out row
    per fragment: arange(B), arange(B) + 1).  `num_kv_heads` divides `num_heads`: shared key and value heads.
    `buckets` int [2 reach + 1]: see relative_buckets; `num_buckets`: columns of the table (default: as many as used).
    A plan holds no results; several calls may use it at once.  Make it and let go of it outside of a graph capture (both
    allocate or free device memory), and keep it as long as a graph that captured its calls is replayed."""

    def __init__(self, start, end, num_heads: int, head_dim: int, num_kv_heads: int = None, query_start=None,
                 query_end=None, buckets=None, num_buckets: int = None, device="cuda:0") -> None:
        if not str(device).startswith("cuda"):
            raise RuntimeError("FragmentAttention: this package is the MI355X path ('cuda:<k>' devices only)")
        self.device = torch.device("cuda", torch.device(device).index or 0)
        self.num_heads, self.head_dim = int(num_heads), int(head_dim)
        self.num_kv_heads = self.num_heads if num_kv_heads is None else int(num_kv_heads)
        k0, k1 = _whole(start, "start", np.int64), _whole(end, "end", np.int64)
        if (query_start is None) != (query_end is None):
            raise ValueError("query_start and query_end come together")
        self.own_queries = query_start is not None
        q0, q1 = (k0, k1) if not self.own_queries else (_whole(query_start, "query_start", np.int64),
                                                        _whole(query_end, "query_end", np.int64))
        for lo, hi, name in ((k0, k1, "start / end"), (q0, q1, "query_start / query_end")):
            if len(lo) == 0 or len(lo) != len(k0) or len(hi) != len(k0) or lo[0] != 0 or (lo[1:] != hi[:-1]).any() \
                    or (hi < lo).any():
                raise ValueError(f"{name}: contiguous ascending ranges from 0, one per fragment, expected")
            if hi[-1] > MAX_ROWS:
                raise ValueError(f"{name}: at most 2^30 rows expected")
        if self.num_heads < 1 or self.num_kv_heads < 1 or self.num_heads % self.num_kv_heads:
            raise ValueError("num_kv_heads has to divide num_heads")
        if self.num_heads > MAX_HEADS:
            raise ValueError(f"num_heads: at most {MAX_HEADS} expected")
        if not 8 <= self.head_dim <= 128 or self.head_dim % 8:
            raise ValueError("head_dim: a multiple of 8 from 8 to 128 expected")
        self.rows_k, self.rows_q = int(k1[-1]), int(q1[-1])
        self.num_buckets, reach, lut = 0, 0, None
        if buckets is not None:
            lut = _whole(buckets, "buckets", np.int32)
            reach = len(lut) // 2
            if len(lut) % 2 == 0 or reach > MAX_REACH or lut.min() < 0:
                raise ValueError(f"buckets: [2 reach + 1] bucket numbers, reach <= {MAX_REACH}, expected")
            self.num_buckets = int(lut.max()) + 1 if num_buckets is None else int(num_buckets)
            if not lut.max() < self.num_buckets <= MAX_BUCKETS:
                raise ValueError(f"num_buckets: more than the largest bucket number and at most {MAX_BUCKETS} expected")
        self._L = capi.lib()
        self._h = C.c_void_p()
        rc = self._L.vsn_attn_create(
            C.byref(self._h), self.device.index, len(k0), capi.i64_ptr(k0), capi.i64_ptr(k1),
            capi.i64_ptr(q0) if self.own_queries else None, capi.i64_ptr(q1) if self.own_queries else None,
            self.num_heads, self.num_kv_heads, self.head_dim, reach,
            lut.ctypes.data_as(C.POINTER(C.c_int32)) if lut is not None else None, self.num_buckets)
        if rc:
            raise RuntimeError(f"vsn_attn_create failed ({rc})")

    # -- arguments ---------------------------------------------------------------------------------------------------
    def _rows(self, t, name: str, heads: int, least: int, dtype, exact=None):
        """The tensor as it is where the kernels can address it (dense last axis, 16-byte steps), else a copy."""
        if not t.is_cuda or t.device != self.device or t.is_neg():
            on_device(t, name, self.device)
        if t.dtype != dtype:
            raise ValueError(f"{name}: {dtype} expected, not {t.dtype}")
        shape = t.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim or shape[0] < least \
                or exact not in (None, shape[0]):
            raise ValueError(f"{name}: [{'>= %d' % least if exact is None else exact}, {heads}, {self.head_dim}] "
                             f"expected, got {tuple(t.shape)}")
        if t.numel() == 0:
            return t
        step = 16 // t.element_size()
        row, head, last = t.stride()
        if last != 1 or row % step or head % step or row > MAX_ROW_STEP or (heads > 1 and head < self.head_dim) \
                or t.data_ptr() % 16:
            return t.clone(memory_format=torch.contiguous_format)
        return t

    def _small(self, t, name: str, shape, dtype):
        if not t.is_cuda or t.device != self.device or t.is_neg():
            on_device(t, name, self.device)
        if t.dtype != dtype or t.shape != shape:
            raise ValueError(f"{name}: {dtype} {tuple(shape)} expected, got {t.dtype} {tuple(t.shape)}")
        return t if t.is_contiguous() else t.contiguous()

    def _io(self, q, k, v, pos, slope, residue, table, query_pos, query_residue, scale):
        """(arguments of the C call without its outputs, the tensors that have to stay alive until it is queued)"""
        on_device(q, "q", self.device)
        code = dtype_code(q, "q")
        q = self._rows(q, "q", self.num_heads, self.rows_q, q.dtype)
        k = self._rows(k, "k", self.num_kv_heads, self.rows_k, q.dtype)
        v = self._rows(v, "v", self.num_kv_heads, self.rows_k, q.dtype, exact=k.shape[0])
        if not self.own_queries and q.shape[0] != k.shape[0]:
            raise ValueError("q and k: the same rows expected (the plan has no query ranges of its own)")
        if (pos is None) != (slope is None) or (residue is None) != (table is None):
            raise ValueError("pos and slope come together, and so do residue and table")
        if not self.own_queries and (query_pos is not None or query_residue is not None):
            raise ValueError("query_pos / query_residue: only with query ranges of their own")
        if self.own_queries and ((query_pos is None) != (pos is None) or (query_residue is None) != (residue is None)):
            raise ValueError("query_pos / query_residue: expected with pos / residue")
        no_graph(q, k, v, pos, slope, table, query_pos)
        if pos is not None:
            pos = self._small(pos, "pos", (k.shape[0], 3), torch.float32)
            query_pos = self._small(query_pos, "query_pos", (q.shape[0], 3), torch.float32) if self.own_queries else pos
            slope = self._small(slope, "slope", (self.num_heads,), torch.float32)
        if residue is not None:
            if not self.num_buckets:
                raise ValueError("table: the plan was made without buckets")
            residue = self._small(residue, "residue", (k.shape[0],), torch.int32)
            query_residue = self._small(query_residue, "query_residue", (q.shape[0],), torch.int32) \
                if self.own_queries else residue
            table = self._small(table, "table", (self.num_heads, self.num_buckets), torch.float32)
        io = capi.VsnAttnIO(code, self.head_dim ** -0.5 if scale is None else float(scale), q.shape[0], k.shape[0],
                            q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), q.stride(1), k.stride(0),
                            k.stride(1), v.stride(0), v.stride(1))
        if pos is not None:
            io.q_pos, io.k_pos, io.slope = query_pos.data_ptr(), pos.data_ptr(), slope.data_ptr()
        if residue is not None:
            io.q_res, io.k_res, io.table = query_residue.data_ptr(), residue.data_ptr(), table.data_ptr()
        return io, (q, k, v, pos, query_pos, slope, residue, query_residue, table)

    def _rows_out(self, shape, used: int, dtype):
        """rows behind the last fragment are not written by the kernels: zeros where there are any"""
        make = torch.empty if shape[0] == used else torch.zeros
        return make(shape, dtype=dtype, device=self.device)

    def _space(self, rows_q: int, rows_k: int, backward: int):
        size = self._L.vsn_attn_workspace(self._h, rows_q, rows_k, backward)
        return torch.empty(size, dtype=torch.uint8, device=self.device) if size else None, size

    # -- calls -------------------------------------------------------------------------------------------------------
    def forward(self, q, k, v, *, pos=None, slope=None, residue=None, table=None, query_pos=None, query_residue=None,
                scale=None, out=None, save=False):
        """out [rows_q, heads, head_dim], or (out, stats) with save=True for a backward pass.

        q [rows_q, heads, head_dim], k, v [rows_k, kv_heads, head_dim] in float32, bfloat16 or float16; any strides
        (layouts the kernels cannot address are copied first).  pos float32 [rows_k, 3] with slope [heads]; residue
        int32 [rows_k] with table float32 [heads, buckets]; query_pos / query_residue where the queries have rows of
        their own.  `scale` defaults to head_dim ** -0.5.  A row without keys, or whose scores are all -inf, gives 0.
        Rows behind the last fragment give 0; in a given `out` (apart from the inputs) they stay as they were.  Runs on the current stream."""
        io, held = self._io(q, k, v, pos, slope, residue, table, query_pos, query_residue, scale)
        rows = held[0].shape[0]
        shape = (rows, self.num_heads, self.head_dim)
        if out is None:
            out = self._rows_out(shape, self.rows_q, held[0].dtype)
        elif self._rows(out, "out", self.num_heads, self.rows_q, held[0].dtype, exact=rows) is not out:
            raise ValueError("out: a dense last axis, and strides and address of whole 16-byte steps expected")
        no_graph(out)
        io.out, io.out_row, io.out_head = out.data_ptr(), out.stride(0), out.stride(1)
        stats = None
        if save:
            make = torch.empty if rows == self.rows_q else torch.zeros
            stats = make(self.num_heads, rows, 2, dtype=torch.float32, device=self.device)
            io.stats = stats.data_ptr()
        work, size = self._space(rows, held[1].shape[0], 0)
        rc = self._L.vsn_attn_forward(self._h, C.byref(io), ptr(work), size, stream_of(held[0]))
        if rc:
            raise RuntimeError(f"vsn_attn_forward failed ({rc})")
        return (out, stats) if save else out

    def backward(self, dout, q, k, v, stats, *, pos=None, slope=None, residue=None, table=None, query_pos=None,
                 query_residue=None, scale=None) -> AttentionGrads:
        """Gradients of forward(..., save=True) with the same arguments, from dout = dL/dout.

        dq, dk, dv in the rows' type (key heads summed over the queries' heads that share them); dpos float32 [rows_k, 3]
        (both ends of every pair where queries and keys are the same rows, else the keys' with dquery_pos for the queries'),
        dslope [heads], dtable [heads, buckets]; None where the term is absent.  `stats`: what forward returned."""
        io, held = self._io(q, k, v, pos, slope, residue, table, query_pos, query_residue, scale)
        q, k = held[0], held[1]
        no_graph(dout, stats)
        dout = self._rows(dout, "dout", self.num_heads, self.rows_q, q.dtype, exact=q.shape[0])
        stats = self._small(stats, "stats", (self.num_heads, q.shape[0], 2), torch.float32)
        io.stats = stats.data_ptr()
        f32 = dict(dtype=torch.float32, device=self.device)
        dq = self._rows_out(q.shape, self.rows_q, q.dtype)
        dk = self._rows_out(k.shape, self.rows_k, q.dtype)
        dv = self._rows_out(k.shape, self.rows_k, q.dtype)
        dpos = dquery_pos = dslope = dtable = None
        if pos is not None:
            dpos = self._rows_out((k.shape[0], 3), self.rows_k, torch.float32)
            dquery_pos = self._rows_out((q.shape[0], 3), self.rows_q, torch.float32) if self.own_queries else None
            dslope = torch.empty(self.num_heads, **f32)
        if table is not None:
            dtable = torch.empty(self.num_heads, self.num_buckets, **f32)
        address = lambda t: 0 if t is None else t.data_ptr()
        grads = capi.VsnAttnGrads(dout.data_ptr(), dout.stride(0), dout.stride(1), dq.data_ptr(), dk.data_ptr(),
                                  dv.data_ptr(), address(dpos), address(dquery_pos), address(dslope), address(dtable))
        absent = (NO_POS if pos is None else 0) | (NO_TABLE if table is None else 0)
        work, size = self._space(q.shape[0], k.shape[0], BACKWARD | absent)
        rc = self._L.vsn_attn_backward(self._h, C.byref(io), C.byref(grads), ptr(work), size, stream_of(q))
        if rc:
            raise RuntimeError(f"vsn_attn_backward failed ({rc})")
        return AttentionGrads(dq, dk, dv, dpos, dquery_pos, dslope, dtable)

    def __del__(self):
        try:
            if self._h:
                self._L.vsn_attn_destroy(self._h)
                self._h = None
        except Exception:
            pass
