"""Document vectors on the device (include/mdd.h, "Document vectors"): the methods that minhash.Engine has for them.

A document as a row of numbers instead of a set of shingles: ids are looked up in an embedding table and averaged (`embed`,
`embed_backward`), rows are normalised (`rms_norm`, `rms_norm_backward`) and held in 8 bits (`rms_norm_q8`) or in microscaled 4
bits (`mx_quantize`), compared with an index (`mx_matmul`) or among themselves (`mx_pairs`), and candidate pairs are checked on the
8-bit rows (`edge_cosines`).  An extension: the reference compares documents by their shingles only.  torch owns the memory;
every computation is a kernel of libmdd_hip.so on the engine's stream.  A call made under another current stream is ordered
with it on both sides.  Matrices may be row-strided views (unit stride inside a row).  Wrong arguments raise lib.MddError.  No
autograd node is made: the gradients have methods of their own, and a tensor that requires one is refused outside torch.no_grad().
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple, Optional

import torch

from . import lib as _lib

_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_Q8 = {"int8": (3, torch.int8), "e4m3": (4, torch.float8_e4m3fn)}
_Q8_OF = {torch.int8: 3, torch.float8_e4m3fn: 4}
MAX_DIM = 32768
MAX_PAIR_ROWS = 1 << 22          # of one search for near pairs


class TooManyPairs(_lib.MddError):
    """a search for near pairs found `count` of them, more than the caller's `limit`"""

    def __init__(self, count: int, limit: int, min_cosine: float):
        super().__init__(f"{count} pairs reach {min_cosine}: more than max_pairs={limit}")
        self.count, self.limit = count, limit


class MxMatrix(NamedTuple):
    """A matrix in microscaled 4-bit form, packed in the order in which the matrix instruction reads it (include/mdd.h): codes
    uint8 [row tiles, column tiles, 4, 32, 16], scales uint8 [row tiles, column tiles, 2, 32, 2]; tiles of 32 rows x 128 columns."""
    codes: torch.Tensor
    scales: torch.Tensor
    rows: int
    cols: int


def _tensors(x):
    if isinstance(x, torch.Tensor):
        yield x
    elif isinstance(x, (tuple, list)):
        for y in x:
            yield from _tensors(y)


# the current stream as a number: a tenth of a microsecond where torch.cuda.current_stream, which makes an object, takes two
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _ordered(fn):
    """runs fn on the engine's stream; under another current stream that one waits for the results, and they for it"""
    @functools.wraps(fn)
    def call(self, *args, **kw):
        if _raw_stream(self.device_index) == self.stream.cuda_stream:
            return fn(self, *args, **kw)
        cur = torch.cuda.current_stream(self.device)
        self.stream.wait_stream(cur)
        with torch.cuda.stream(self.stream):
            out = fn(self, *args, **kw)
        cur.wait_stream(self.stream)
        for t in _tensors((args, tuple(kw.values()))):
            if t.is_cuda:
                t.record_stream(self.stream)
        for t in _tensors(out):
            t.record_stream(cur)
        return out
    return call


def _need(ok, what):
    if not ok:
        raise _lib.MddError(what)


def _refuse(what):
    raise _lib.MddError(what)


def _no_node(name):
    """a result without a node would cut the tensor's gradient off without a word"""
    if torch.is_grad_enabled():
        _refuse(f"{name} requires a gradient, and no autograd node is made: call under torch.no_grad() or pass {name}.detach(), and the *_backward method yourself")


class VectorOps:
    """mixed into minhash.Engine"""

    # ------------------------------------------------------------------ checks
    # (messages are made only when they are raised: a call is a dozen microseconds, of which these checks would be three)
    def _matrix(self, t, name, dtype=None, rows=None, cols=None):
        """(address, row stride) of a matrix, None for an empty one"""
        if not isinstance(t, torch.Tensor) or t.device != self.device:
            _refuse(f"{name} must be a tensor on {self.device}")
        if t.dim() != 2:
            _refuse(f"{name} must be a matrix, not {t.dim()}-dimensional")
        if t.dtype not in _TYPE if dtype is None else t.dtype != dtype:
            _refuse(f"{name} has type {t.dtype}" + (f", not {dtype}" if dtype else ""))
        if t.requires_grad:
            _no_node(name)
        n, d = t.shape
        if not 1 <= d <= MAX_DIM:
            _refuse(f"{name} has {d} columns: 1 to {MAX_DIM} are supported")
        if rows is not None and n != rows:
            _refuse(f"{name} has {n} rows, not {rows}")
        if cols is not None and d != cols:
            _refuse(f"{name} has {d} columns, not {cols}")
        stride, inner = t.stride()
        if n > 0 and ((inner != 1 and d > 1) or (stride < d and n > 1)):
            _refuse(f"{name} must have unit stride inside its rows")
        return (t.data_ptr() if n else None), (stride if n > 1 else d)

    def _vector(self, t, name, dtypes, size=None):
        if not isinstance(t, torch.Tensor) or t.device != self.device:
            _refuse(f"{name} must be a tensor on {self.device}")
        if t.dim() != 1 or not t.is_contiguous():
            _refuse(f"{name} must be a contiguous vector")
        if t.dtype not in dtypes:
            _refuse(f"{name} has type {t.dtype}")
        if t.requires_grad:
            _no_node(name)
        n = t.numel()
        if size is not None and n != size:
            _refuse(f"{name} has {n} entries, not {size}")
        return t.data_ptr() if n else None

    def _work(self, n_bytes):
        if not n_bytes:
            return None, 0, None
        ws = torch.empty(n_bytes, dtype=torch.uint8, device=self.device)
        return ws.data_ptr(), n_bytes, ws

    def _ids(self, ids, offsets, mode):
        if mode not in ("mean", "sum"):
            _refuse(f"mode {mode!r} is neither 'mean' nor 'sum'")
        p = self._vector(ids, "ids", (torch.int32, torch.int64))
        o, docs = None, 0
        if offsets is not None:
            o = self._vector(offsets, "offsets", (torch.int64,))
            _need(offsets.numel() >= 1, "offsets must have n_docs + 1 entries")
            docs = offsets.numel() - 1
        return p, ids.element_size(), ids.numel(), o, docs

    # ------------------------------------------------------------------ embedding lookup
    @_ordered
    def embed(self, table: torch.Tensor, ids: torch.Tensor, offsets: Optional[torch.Tensor] = None, scale: float = 1.0,
              mode: str = "mean") -> torch.Tensor:
        """scale * table[ids] (a row per id), or with offsets (int64 [n+1], as for the packed text) a row per document: the
        sum or mean of its ids' rows times scale.  Ids outside the table are padding: they contribute nothing and are not
        counted in the mean; a document without other ids gives zeros.  Returns [n, dim] in the table's type."""
        tp, ts = self._matrix(table, "table")
        ip, ib, n_ids, op, docs = self._ids(ids, offsets, mode)
        v, dim = table.shape
        out = torch.empty(docs if op else n_ids, dim, dtype=table.dtype, device=self.device)
        wp, wb, ws = self._work(self.L.mdd_embed_ws_bytes(n_ids, dim) if op else 0)
        _lib.check(self.L.mdd_embed(self.ctx, tp, _TYPE[table.dtype], v, ts, dim, ip, ib, n_ids, op, docs, int(mode == "mean"), float(scale),
                                    out.data_ptr() if out.numel() else None, wp, wb), "mdd_embed")
        return out

    @_ordered
    def embed_backward(self, grad: torch.Tensor, ids: torch.Tensor, n_rows: int, offsets: Optional[torch.Tensor] = None, scale: float = 1.0,
                       mode: str = "mean", dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Gradient of embed(table, ids, offsets, scale, mode) with respect to a table of n_rows rows: [n_rows, dim] in float32 or
        the gradient's type, zeros where no id points.  Summed in the order of the positions: repeats bit for bit."""
        gp, gs = self._matrix(grad, "grad")
        ip, ib, n_ids, op, docs = self._ids(ids, offsets, mode)
        if grad.shape[0] != (docs if op else n_ids):
            _refuse(f"grad has {grad.shape[0]} rows, not {docs if op else n_ids}")
        if dtype not in (torch.float32, grad.dtype):
            _refuse(f"dtype {dtype} is neither float32 nor the gradient's")
        _need(n_rows >= 0, "n_rows is negative")
        dim = grad.shape[1]
        out = torch.empty(n_rows, dim, dtype=dtype, device=self.device)
        wp, wb, ws = self._work(self.L.mdd_embed_backward_ws_bytes(n_ids, docs, n_rows, dim))
        _lib.check(self.L.mdd_embed_backward(self.ctx, gp, _TYPE[grad.dtype], gs, dim, ip, ib, n_ids, op, docs, int(mode == "mean"), float(scale),
                                             out.data_ptr() if out.numel() else None, _TYPE[dtype], n_rows, wp, wb), "mdd_embed_backward")
        return out

    # ------------------------------------------------------------------ root-mean-square norm
    def _norm_args(self, x, weight, residual):
        xp, xs = self._matrix(x, "x")
        n, dim = x.shape
        rp, rs = (None, 0) if residual is None else self._matrix(residual, "residual", x.dtype, n, dim)
        wp = None if weight is None else self._vector(weight, "weight", (x.dtype,), dim)
        return xp, xs, rp, rs, wp, n, dim

    @_ordered
    def rms_norm(self, x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
        """h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight.  Returns (y, h rounded to x's type -- x itself without a
        residual --, 1 / sqrt(...) as float32 [n]): what rms_norm_backward wants."""
        xp, xs, rp, rs, wp, n, dim = self._norm_args(x, weight, residual)
        y = torch.empty(n, dim, dtype=x.dtype, device=self.device)
        total = x if residual is None else torch.empty_like(y)
        rstd = torch.empty(n, dtype=torch.float32, device=self.device)
        if n:
            _lib.check(self.L.mdd_rms_norm(self.ctx, xp, _TYPE[x.dtype], xs, rp, rs, wp, float(eps), n, dim, y.data_ptr(),
                                           None if residual is None else total.data_ptr(), rstd.data_ptr()), "mdd_rms_norm")
        return y, total, rstd

    @_ordered
    def rms_norm_q8(self, x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                    kind: str = "int8"):
        """rms_norm with y in 8 bits and a float32 scale per row (y = codes * scale): kind "int8" or "e4m3".  Returns (codes,
        scales, h, or None without a residual).  Codes are the nearest ones to h * weight, held in 64 bits, over the row's
        largest: decided without a rounding of that quotient."""
        if kind not in _Q8:
            _refuse(f"kind {kind!r} is neither 'int8' nor 'e4m3'")
        xp, xs, rp, rs, wp, n, dim = self._norm_args(x, weight, residual)
        codes = torch.empty(n, dim, dtype=_Q8[kind][1], device=self.device)
        scales = torch.empty(n, dtype=torch.float32, device=self.device)
        total = None if residual is None else torch.empty(n, dim, dtype=x.dtype, device=self.device)
        if n:
            _lib.check(self.L.mdd_rms_norm_q8(self.ctx, xp, _TYPE[x.dtype], xs, rp, rs, wp, float(eps), n, dim, _Q8[kind][0], codes.data_ptr(),
                                              scales.data_ptr(), None if total is None else total.data_ptr()), "mdd_rms_norm_q8")
        return codes, scales, total

    @_ordered
    def rms_norm_backward(self, grad: torch.Tensor, total: torch.Tensor, rstd: torch.Tensor, weight: Optional[torch.Tensor] = None,
                          grad_sum: Optional[torch.Tensor] = None):
        """Gradients of rms_norm from the gradient of y, its second and third result, and the gradient that reaches the sum by
        other ways (grad_sum).  Returns (gradient of x and of residual alike, weight's gradient float32 [dim] or None)."""
        hp, hs = self._matrix(total, "total")
        n, dim = total.shape
        gp, gs = self._matrix(grad, "grad", total.dtype, n, dim)
        sp, ss = (None, 0) if grad_sum is None else self._matrix(grad_sum, "grad_sum", total.dtype, n, dim)
        wp = None if weight is None else self._vector(weight, "weight", (total.dtype,), dim)
        rp = self._vector(rstd, "rstd", (torch.float32,), n)
        dx = torch.empty(n, dim, dtype=total.dtype, device=self.device)
        dw = None if weight is None else torch.empty(dim, dtype=torch.float32, device=self.device)
        kp, kb, ws = self._work(0 if dw is None else self.L.mdd_rms_norm_backward_ws_bytes(n, dim))
        _lib.check(self.L.mdd_rms_norm_backward(self.ctx, gp, _TYPE[total.dtype], gs, hp, hs, sp, ss, wp, rp, n, dim, dx.data_ptr() if n else None,
                                                None if dw is None else dw.data_ptr(), kp, kb), "mdd_rms_norm_backward")
        return dx, dw

    # ------------------------------------------------------------------ candidate edges
    def _edges(self, eu, ev):
        up = self._vector(eu, "edge_u", (torch.int32,))
        return up, self._vector(ev, "edge_v", (torch.int32,), eu.numel()), eu.numel()

    @_ordered
    def edge_cosines(self, codes: torch.Tensor, eu: torch.Tensor, ev: torch.Tensor) -> torch.Tensor:
        """float32 [n_edges]: cosine of the rows eu[e] and ev[e] of 8-bit rows (int8 or float8_e4m3fn); 0 where a row is all zeros
        or the edge names a row that is not there.  Scales of the rows cancel and are not needed."""
        _need(isinstance(codes, torch.Tensor) and codes.dtype in _Q8_OF, "codes must be int8 or float8_e4m3fn")
        cp, cs = self._matrix(codes, "codes", codes.dtype)
        up, vp, n = self._edges(eu, ev)
        out = torch.empty(n, dtype=torch.float32, device=self.device)
        if n:
            _lib.check(self.L.mdd_edge_cosines(self.ctx, cp, _Q8_OF[codes.dtype], cs, codes.shape[0], codes.shape[1], up, vp, n, out.data_ptr()),
                       "mdd_edge_cosines")
        return out

    @_ordered
    def sort_edges(self, eu: torch.Tensor, ev: torch.Tensor, n_docs: int):
        """orders an edge list (entries < n_docs) by (eu, ev), in place; returns it"""
        up, vp, n = self._edges(eu, ev)
        wp, wb, ws = self._work(self.L.mdd_sort_edges_ws_bytes(n))
        _lib.check(self.L.mdd_sort_edges(self.ctx, up, vp, n, int(n_docs), wp, wb), "mdd_sort_edges")
        return eu, ev

    # ------------------------------------------------------------------ microscaled 4-bit matrices
    def _packed(self, m, name):
        if not isinstance(m, MxMatrix):
            _refuse(f"{name} must be an MxMatrix")
        rt, ct = (m.rows + 31) // 32, (m.cols + 127) // 128
        if m.rows < 0 or not 1 <= m.cols <= MAX_DIM:
            _refuse(f"{name} is {m.rows} x {m.cols}: 1 to {MAX_DIM} columns are supported")
        for t, size in ((m.codes, rt * ct * 2048), (m.scales, rt * ct * 128)):
            if not isinstance(t, torch.Tensor) or t.device != self.device or t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() != size:
                _refuse(f"{name}: codes and scales must be contiguous uint8 tensors on {self.device} of {rt * ct * 2048} and {rt * ct * 128} bytes")
        return (m.codes.data_ptr(), m.scales.data_ptr()) if m.rows else (None, None)

    @_ordered
    def mx_quantize(self, x: torch.Tensor) -> MxMatrix:
        """x in microscaled 4 bits: e2m1 elements, a power of two per 32 columns (0.53 bytes per element)."""
        xp, xs = self._matrix(x, "x")
        n, dim = x.shape
        rt, ct = (n + 31) // 32, (dim + 127) // 128
        m = MxMatrix(torch.empty(rt, ct, 4, 32, 16, dtype=torch.uint8, device=self.device),
                     torch.empty(rt, ct, 2, 32, 2, dtype=torch.uint8, device=self.device), n, dim)
        if n:
            _lib.check(self.L.mdd_mx_quantize(self.ctx, xp, _TYPE[x.dtype], xs, n, dim, m.codes.data_ptr(), m.scales.data_ptr()), "mdd_mx_quantize")
        return m

    @_ordered
    def mx_matmul(self, a: MxMatrix, b: MxMatrix, dtype: torch.dtype = torch.float32, alpha: float = 1.0) -> torch.Tensor:
        """alpha * A B^T [a.rows, b.rows] in float32 or bfloat16: every row of A against every row of B."""
        ac, as_ = self._packed(a, "a")
        bc, bs = self._packed(b, "b")
        if a.cols != b.cols:
            _refuse(f"a has {a.cols} columns and b {b.cols}")
        if dtype not in (torch.float32, torch.bfloat16):
            _refuse(f"dtype {dtype} is neither float32 nor bfloat16")
        out = torch.empty(a.rows, b.rows, dtype=dtype, device=self.device)
        if out.numel():
            _lib.check(self.L.mdd_mx_matmul(self.ctx, ac, as_, a.rows, bc, bs, b.rows, a.cols, float(alpha), out.data_ptr(), _TYPE[dtype], b.rows),
                       "mdd_mx_matmul")
        return out

    @_ordered
    def mx_pairs(self, m: MxMatrix, min_cosine: float, max_pairs: int = 1 << 28):
        """Every pair of rows u > v whose 4-bit values have a cosine >= min_cosine, ordered by (u, v): int32 tensors (u, v).  The
        n x n matrix is never stored.  Rows of zeros, with a NaN, or of a length outside [2^-60, 2^60] have no pairs.  One synchronisation, for the number of pairs; a second pass when there are more than eight
        per row.  More than max_pairs raise TooManyPairs, an MddError."""
        mc, ms = self._packed(m, "m")
        _need(max_pairs >= 0, "max_pairs is negative")
        cnt = torch.empty(1, dtype=torch.int64, device=self.device)
        wp, wb, ws = self._work(self.L.mdd_mx_pairs_ws_bytes(m.rows))
        cap = min(int(max_pairs), max(4096, 8 * m.rows))
        while True:
            edges = torch.empty(2 * cap, dtype=torch.int32, device=self.device)
            at = edges.data_ptr()
            _lib.check(self.L.mdd_mx_pairs(self.ctx, mc, ms, m.rows, m.cols, float(min_cosine), at, at + 4 * cap, cap, cnt.data_ptr(), wp, wb),
                       "mdd_mx_pairs")
            n = int(cnt.item())
            if n > max_pairs:
                raise TooManyPairs(n, max_pairs, min_cosine)
            if n <= cap:
                break
            cap = n
        return self.sort_edges(edges[:n], edges[cap: cap + n], m.rows)
