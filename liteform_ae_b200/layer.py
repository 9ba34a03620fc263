"""Operators of a layer around the CSR product: the norm that makes the rows it gathers, the product with
bias, activation and residual in its epilogue, and the gradients of both.

    n = rms_norm(x, w, residual=r, out_dtype=torch.float8_e4m3fn)       # n.h = x + r, n.y and n.scale its norm
    y = spmm_csr_act(csr, n.y, scale=n.scale, bias=b, activation="silu", residual=n.h)

and for training, with 16- or 32-bit rows and the transposed pattern that the program keeps beside A:

    z = torch.empty_like(dy);  y = spmm_csr_act(csr, f, bias=b, activation="silu", residual=h, preact=z)
    g = spmm_csr_act_backward(csr, csr_t, f, dy, preact=z, activation="silu")      # g.dB, g.dvalues, g.dbias
    dx, dw = rms_norm_backward(g.dB, h, w, n.rstd, dh=dy)                          # dy also reaches h directly

The reference has no counterpart: its product ends with C = A * B (playground_pipline/format_algos.py:1660-1755).

All computation is done by ``liblf_b200.so`` on torch's current stream of the tensors' device; nothing is
synchronised (except for a ``row_range``, see ``spmm_csr_act``).  The same call on the same inputs gives the same
bits.  Matrices are dense in their last dimension and may have any row stride of at least their width; a row stride
and address on 16-byte boundaries is faster.  Outputs may not share memory with each other or with inputs, but for the
matrices that a call names as allowed.  Nothing is recorded for autograd: tensors that require a gradient are refused while
gradients are enabled, the ``..._backward`` functions give them.  ``ValueError`` for arguments that do not fit together.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import NamedTuple, Optional, Tuple

import numpy as np

from . import _cabi
from ._cabi import LfEpilogue, check, cuda_torch as _torch, on_device, stream_of
from .hyb import DeviceCsr, Workspace

ACTIVATIONS = {None: _cabi.LF_ACT_NONE, "none": _cabi.LF_ACT_NONE, "relu": _cabi.LF_ACT_RELU, "silu": _cabi.LF_ACT_SILU,
               "gelu": _cabi.LF_ACT_GELU, "gelu_tanh": _cabi.LF_ACT_GELU_TANH}

_wide, _any = {}, {}     # LF_DTYPE_* of torch's types: 16 and 32 bits, and with e4m3


def _code(dtype, codes=_wide):
    """``LF_DTYPE_*`` of a torch type."""
    code = codes.get(dtype)
    if code is None:
        if not _wide:     # filled last, whole, so that another thread that finds it filled finds both
            torch = _torch()
            wide = {torch.float32: _cabi.LF_DTYPE_F32, torch.bfloat16: _cabi.LF_DTYPE_BF16, torch.float16: _cabi.LF_DTYPE_F16}
            _any.update({**wide, torch.float8_e4m3fn: _cabi.LF_DTYPE_E4M3})
            _wide.update(wide)
            return _code(dtype, codes)
        raise ValueError(f"type {dtype} is not supported here")
    return code


def _need(cond, message):
    if not cond:
        raise ValueError(message)


def _matrix(t, name, rows, N, dev):
    """Row stride of ``t``, which has to be ``[rows, N]`` on device ``dev`` and dense in a row."""
    if t.shape != (rows, N):
        raise ValueError(f"{name} must have shape ({rows}, {N})")
    if t.get_device() != dev:
        raise ValueError(f"{name} must be on the device of the other operands")
    ld, inner = t.stride()
    if inner != 1 and N != 1:
        raise ValueError(f"{name} must be dense in its last dimension")
    if ld < N:
        if rows > 1:
            raise ValueError(f"rows of {name} overlap")
        return N
    return ld


def _vector(t, name, n, dev, dtype=None):
    if t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a dense vector of {n}")
    if t.get_device() != dev:
        raise ValueError(f"{name} must be on the device of the other operands")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}")
    return t.data_ptr()


def _first(t, name):
    """``(rows, N, device)`` of the operand that the others have to fit."""
    if not t.is_cuda or t.dim() != 2 or t.shape[1] < 1:
        raise ValueError(f"{name} must be a matrix on a CUDA device")
    return t.shape[0], t.shape[1], t.get_device()


def _extent(t):
    """``(address, end, bytes of a row, bytes from a row to the next)``; dense tensors count as one row, at distance 0."""
    p, e, n = t.data_ptr(), t.element_size(), t.numel()
    if not n or t.is_contiguous() or t.dim() != 2 or t.shape[0] < 2:
        return p, p + n * e, n * e, 0
    step, wide = t.stride(0) * e, t.shape[1] * e
    return p, p + (t.shape[0] - 1) * step + wide, wide, step


def _extents_share(a, b) -> bool:
    p, end_a, wide_a, step_a = a
    q, end_b, wide_b, step_b = b
    if end_a <= q or end_b <= p or p == end_a or q == end_b:
        return False
    step = step_a or step_b
    if not step or (step_a and step_b and step_a != step_b):
        return True
    gap = (q - p) % step       # from a row of a to the next of b
    return gap < wide_a or gap + wide_b > step


def _share_memory(a, b) -> bool:
    """Whether two matrices or vectors have bytes in common.  Rows at one distance may lie beside each other, as column slices of a
    buffer do; at two distances, one reaching into the other counts as sharing."""
    return _extents_share(_extent(a), _extent(b))


def _outputs_apart(given, inputs, may_be=()):
    """Refuses outputs that the caller gave in memory that the call reads or writes elsewhere: ``given`` and ``inputs`` are
    ``(tensor, name)``, tensors may be None; ``may_be``: pairs of names that may be one and the same matrix."""
    seen = [(t, name, _extent(t)) for t, name in inputs if t is not None]
    for t, name in given:
        if t is None:
            continue
        at = _extent(t)
        for other, of, there in seen:
            if at[0] < there[1] and there[0] < at[1] and _extents_share(at, there) and not (
                    (name, of) in may_be and at[0] == there[0] and t.dtype == other.dtype and t.shape == other.shape and t.stride() == other.stride()):
                raise ValueError(f"{name} lies in the memory of {of}")
        seen.append((t, name, at))


def _no_graph(*tensors):
    """Refuses what autograd would lose without a word."""
    if _torch().is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("autograd does not see this call: make it under torch.no_grad(), or with detached tensors, and take "
                                 "gradients from the ..._backward functions")


def _act_code(activation):
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"unknown activation {activation!r}")
    return code


def _run(fn, call, dev):
    """``fn(*call)`` with ``dev`` current (a guard costs more than the rest of a small call)."""
    if _torch()._C._cuda_getDevice() == dev:
        status = fn(*call)
    else:
        with on_device(dev):
            status = fn(*call)
    if status:
        check(status)


def _scratch(nbytes, workspace, like):
    """``(buffer, address, size)`` of ``nbytes`` on the device of ``like``; the buffer has to outlive the call.  A call that is
    captured takes memory of its graph's own: a workspace may grow, and its old buffer be another tensor's by the replay."""
    if nbytes == 0:
        return None, 0, 0
    torch = _torch()
    if workspace is None or torch.cuda.is_current_stream_capturing():
        buf = torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    else:
        buf = workspace.get(nbytes)
        _need(buf.get_device() == like.get_device(), "the workspace must be on the device of the operands")
    return buf, buf.data_ptr(), buf.numel()


def empty_rows(rows: int, N: int, dtype, device):
    """``[rows, N]`` uninitialised with every row on a 16-byte boundary (the view of a wider buffer where N does
    not give that by itself): how the operators allocate 8-bit rows."""
    torch = _torch()
    per = 16 // dtype.itemsize
    wide = -(-N // per) * per
    t = torch.empty((rows, wide), dtype=dtype, device=device)
    return t if wide == N else t[:, :N]


def _rows_like(t, dtype):
    """New rows of ``t``'s shape, dense; the shorter way where there is one (half the host time of a small call is this)."""
    torch = _torch()
    if t.is_contiguous():
        return torch.empty_like(t) if t.dtype == dtype else torch.empty_like(t, dtype=dtype)
    return torch.empty(t.shape, dtype=dtype, device=t.device)


# ---- norm -------------------------------------------------------------------------------------------
class NormOutput(NamedTuple):
    y: "object"                 # normed rows
    scale: Optional["object"]   # float32, one per row: what e4m3 rows are multiples of (None for other types)
    h: "object"                 # what was normed: x + residual, or x itself
    rstd: "object"              # float32, one per row, for the backward pass


def rms_norm(x, weight, residual=None, eps: float = 1e-6, out_dtype=None, out=None, scale=None, sum_out=None,
             rstd=None) -> NormOutput:
    """``lf_rms_norm``: ``h = x + residual`` in x's type, ``y = h * rstd * weight`` with ``rstd = (mean(h^2) +
    eps)^(-1/2)``, row by row.  ``out_dtype`` (default: x's): float32, bfloat16, float16, or float8_e4m3fn with one
    scale per row (``y * scale`` is the row).  ``out``, ``scale``, ``sum_out`` and ``rstd`` take the outputs in place of new
    tensors; ``out`` and ``sum_out`` may each be ``x`` or ``residual`` itself."""
    torch = _torch()
    _no_graph(x, weight, residual)
    if out is not None or sum_out is not None or scale is not None or rstd is not None:
        _outputs_apart(((out, "out"), (sum_out, "sum_out"), (scale, "scale"), (rstd, "rstd")),
                       ((x, "x"), (residual, "residual"), (weight, "weight")),
                       (("out", "x"), ("out", "residual"), ("sum_out", "x"), ("sum_out", "residual")))
    M, N, dev = _first(x, "x")
    code = _code(x.dtype)
    ld_x = _matrix(x, "x", M, N, dev)
    w = _vector(weight, "weight", N, dev)
    w_code = _code(weight.dtype)
    if out_dtype is None:
        out_dtype = x.dtype if out is None else out.dtype
    y_code = _code(out_dtype, _any)
    e4m3 = y_code == _cabi.LF_DTYPE_E4M3
    if out is None:
        out = empty_rows(M, N, out_dtype, x.device) if e4m3 and N % 16 else _rows_like(x, out_dtype)
    _need(out.dtype == out_dtype, "out must have out_dtype")
    ld_y = _matrix(out, "out", M, N, dev)
    h, res_ptr, ld_res, sum_ptr, ld_sum = x, 0, 0, 0, 0
    if residual is not None:
        _need(residual.dtype == x.dtype, "the residual must have x's type")
        res_ptr, ld_res = residual.data_ptr(), _matrix(residual, "residual", M, N, dev)
        h = _rows_like(x, x.dtype) if sum_out is None else sum_out
        _need(h.dtype == x.dtype, "sum_out must have x's type")
        sum_ptr, ld_sum = h.data_ptr(), _matrix(h, "sum_out", M, N, dev)
    else:
        _need(sum_out is None, "sum_out goes with a residual")
    if not e4m3:
        _need(scale is None, "a scale goes with 8-bit rows")
    elif scale is None:
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
    if rstd is None:
        rstd = torch.empty(M, dtype=torch.float32, device=x.device)
    s_ptr = _vector(scale, "scale", M, dev, torch.float32) if e4m3 else 0
    r_ptr = _vector(rstd, "rstd", M, dev, torch.float32)
    call = (x.data_ptr(), code, ld_x, res_ptr, ld_res, sum_ptr, ld_sum, w, w_code, eps, out.data_ptr(), y_code, ld_y, s_ptr,
            r_ptr, M, N, stream_of(dev))
    _run(_cabi.load().lf_rms_norm, call, dev)
    return NormOutput(out, scale, h, rstd)


def rms_norm_backward(dy, h, weight, rstd, dh=None, dx=None, dweight=None, workspace: Optional[Workspace] = None):
    """``lf_rms_norm_backward``: ``(dx, dweight)`` for ``y = h * rstd * weight``; ``dx`` (in dy's type) is the gradient
    of x and of the residual alike, with ``dh``, the gradient that reaches h by other ways, added; ``dweight`` is
    float32.  For 8-bit rows pass the gradient of the rows they stand for (the rounding's own is taken as 1).
    ``dx`` may be ``dy``, ``h`` or ``dh``."""
    torch = _torch()
    _no_graph(dy, h, weight, dh)
    if dx is not None or dweight is not None:
        _outputs_apart(((dx, "dx"), (dweight, "dweight")), ((dy, "dy"), (h, "h"), (dh, "dh"), (weight, "weight"), (rstd, "rstd")),
                       (("dx", "dy"), ("dx", "h"), ("dx", "dh"), ("dweight", "weight")))
    lib = _cabi.load()
    M, N, dev = _first(dy, "dy")
    code = _code(dy.dtype)
    _need(h.dtype == dy.dtype and (dh is None or dh.dtype == dy.dtype), "dy, h and dh must have one type")
    ld_dy, ld_h = _matrix(dy, "dy", M, N, dev), _matrix(h, "h", M, N, dev)
    ld_dh = 0 if dh is None else _matrix(dh, "dh", M, N, dev)
    if dx is None:
        dx = _rows_like(dy, dy.dtype)
    if dweight is None:
        dweight = torch.empty(N, dtype=torch.float32, device=dy.device)
    _need(dx.dtype == dy.dtype, "dx must have dy's type")
    ld_dx = _matrix(dx, "dx", M, N, dev)
    w, w_code, r = _vector(weight, "weight", N, dev), _code(weight.dtype), _vector(rstd, "rstd", M, dev, torch.float32)
    dw = _vector(dweight, "dweight", N, dev, torch.float32)
    nbytes = lib.lf_rms_norm_backward_workspace_bytes(M, N)
    keep, ws, nws = _scratch(nbytes, workspace, dy)
    call = (dy.data_ptr(), ld_dy, h.data_ptr(), ld_h, code, w, w_code, r, 0 if dh is None else dh.data_ptr(), ld_dh,
            dx.data_ptr(), ld_dx, dw, M, N, ws, nws, stream_of(dev))
    _run(lib.lf_rms_norm_backward, call, dev)
    return dx, dweight


# ---- product ----------------------------------------------------------------------------------------
@dataclass
class CsrTranspose:
    """The pattern of a matrix by columns: what the product with A transposed takes beside A's values.
    ``order[i]`` is the place of entry i among A's entries, so the values are kept once, with A."""
    indptr: "object"            # torch int64 [K + 1]
    indices: "object"           # torch int32 [nnz]: rows of A, ascending inside a column
    order: "object"             # torch int32 [nnz]
    shape: Tuple[int, int]      # (K, M)

    @property
    def nnz(self) -> int:
        return int(self.indices.numel())

    @staticmethod
    def from_host(indptr, indices, shape, device="cuda") -> "CsrTranspose":
        """From A's own (host) arrays and shape."""
        import torch
        M, K = int(shape[0]), int(shape[1])
        indptr, indices = np.asarray(indptr, dtype=np.int64), np.asarray(indices)
        _need(len(indices) < 2 ** 31 and M < 2 ** 31, "at most 2^31 - 1 entries and rows")
        _need(len(indptr) == M + 1 and indptr[0] == 0 and indptr[-1] == len(indices) and bool((np.diff(indptr) >= 0).all()),
              "indptr must ascend from 0 to the number of entries")
        _need(len(indices) == 0 or (indices.min() >= 0 and indices.max() < K), "columns must lie in the matrix")
        order = np.argsort(indices, kind="stable")
        rows = np.repeat(np.arange(M, dtype=np.int32), np.diff(indptr))[order]
        ptr = np.zeros(K + 1, dtype=np.int64)
        np.cumsum(np.bincount(indices, minlength=K), out=ptr[1:])
        up = lambda a: torch.from_numpy(a).to(device)
        return CsrTranspose(up(ptr), up(rows), up(order.astype(np.int32)), (K, M))

    @staticmethod
    def of(csr: DeviceCsr) -> "CsrTranspose":
        """From a matrix in device memory (sorted on the host: done once per matrix)."""
        return CsrTranspose.from_host(csr.indptr.cpu().numpy(), csr.indices.cpu().numpy(), csr.shape, csr.indptr.device)

    def validate(self, a: Optional[DeviceCsr] = None) -> None:
        """``ValueError`` unless this is a pattern as ``DeviceCsr.validate`` wants it, with an ``order`` that names each entry once;
        with ``a``, unless it is that matrix's.  ``from_host`` and ``of`` make such ones; arrays from elsewhere are not checked
        by the products, which would read beside the values with a wrong ``order``.  Waits for the device."""
        import torch
        nnz, order = self.nnz, self.order
        _need(order.dtype == torch.int32 and order.dim() == 1 and order.numel() == nnz, "order must be an int32 vector, one per entry")
        if nnz:
            _need(int(order.min()) >= 0 and int(order.max()) < nnz, "order must lie among the entries")
            _need(int(torch.bincount(order, minlength=nnz).max()) == 1, "order must name each entry once")
        if a is not None:
            _need(a.shape == (self.shape[1], self.shape[0]) and a.nnz == nnz, "the pattern has another shape than the matrix transposed")
        for t, dtype, name in ((self.indptr, torch.int64, "indptr"), (self.indices, torch.int32, "indices")):
            _need(t.dtype == dtype and t.dim() == 1 and t.is_contiguous() and t.device == order.device, f"{name} must be a dense {dtype} vector beside order")
        _need(self.indptr.numel() == self.shape[0] + 1, "indptr must have one more than the rows")
        if 0 in self.shape:
            _need(nnz == 0 and self.indptr.numel() == self.shape[0] + 1 and not bool(self.indptr.any()), "a matrix without rows or columns has no entries")
            return
        DeviceCsr(self.indptr, self.indices, None, self.shape).validate()
        if a is not None:
            rows = lambda ptr: torch.repeat_interleave(torch.arange(ptr.numel() - 1, device=ptr.device, dtype=torch.int32), torch.diff(ptr))
            _need(bool((a.indices[order.long()] == rows(self.indptr)).all()) and bool((rows(a.indptr)[order.long()] == self.indices).all()),
                  "the pattern is not that of the matrix transposed")


def _csr_arrays(a, values, dev):
    """Addresses of the values and of their order."""
    transposed = isinstance(a, CsrTranspose)
    _need(transposed or values is None, "values go with a CsrTranspose; a DeviceCsr has its own")
    data = values if transposed else a.data
    torch = _torch()
    indptr, indices = a.indptr, a.indices
    _need(indptr.get_device() == dev and indptr.is_contiguous() and indptr.numel() == a.shape[0] + 1 and indptr.dtype == torch.int64,
          "indptr must be a dense int64 vector of one more than the rows, beside B")
    _need(indices.get_device() == dev and indices.is_contiguous() and indices.dtype == torch.int32,
          "indices must be a dense int32 vector beside B")
    if data is None:
        return 0, 0
    _need(data.numel() == a.nnz and data.is_contiguous() and data.get_device() == dev and data.dtype == torch.float32,
          "the values must be a dense float32 vector, one per entry, beside B")
    if not transposed:
        return data.data_ptr(), 0
    order = a.order
    _need(order.get_device() == dev and order.is_contiguous() and order.dtype == torch.int32 and order.numel() == a.nnz,
          "order must be a dense int32 vector, one per entry, beside B")
    return data.data_ptr(), order.data_ptr()


def spmm_csr_act(a, B, scale=None, bias=None, activation: Optional[str] = None, residual=None, out_dtype=None, out=None,
                 preact=None, row_range=None, values=None, workspace: Optional[Workspace] = None):
    """``lf_spmm_csr_act``: ``activation(A @ B + bias) + residual`` for a ``DeviceCsr`` (or a ``CsrTranspose`` with A's
    ``values``, None: all ones).  B: float32, bfloat16, float16, or float8_e4m3fn with ``scale`` (float32, one per row);
    ``activation``: None, "relu", "silu", "gelu" or "gelu_tanh"; ``out_dtype``: float32, bfloat16 or float16 (default:
    B's, bfloat16 for 8-bit rows); ``residual`` may be ``out``; ``preact`` (out's type) is filled with ``A @ B + bias`` for
    the backward pass.  ``row_range=(r0, r1)``: those rows of A only -- their number of entries is read back, which
    waits for the stream; a ``DeviceCsr`` of a slice of ``indptr`` does not.  Entries are not checked against B's rows:
    ``DeviceCsr.validate`` does that, once per matrix (``CsrTranspose.validate`` also for ``order``)."""
    torch = _torch()
    _no_graph(B, bias, residual, scale, values, None if isinstance(a, CsrTranspose) else a.data)
    if out is not None or preact is not None:
        _outputs_apart(((out, "out"), (preact, "preact")), ((B, "B"), (residual, "residual"), (bias, "bias"), (scale, "scale")),
                       (("out", "residual"), ("preact", "residual")))
    lib = _cabi.load()
    K, N, dev = _first(B, "B")
    _need(K == a.shape[1], "B must have one row per matrix column")
    b_code = _code(B.dtype, _any)
    ldb = _matrix(B, "B", K, N, dev)
    act = _act_code(activation)
    _need(b_code != _cabi.LF_DTYPE_E4M3 or scale is not None, "8-bit rows need their scales")
    data, order = _csr_arrays(a, values, dev)
    r0, r1 = (0, a.shape[0]) if row_range is None else (int(row_range[0]), int(row_range[1]))
    _need(0 <= r0 <= r1 <= a.shape[0], "bad row range")
    nnz = a.nnz
    if row_range is not None and (r0, r1) != (0, a.shape[0]):
        ends = a.indptr[[r0, r1]].cpu()
        nnz = int(ends[1]) - int(ends[0])
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else torch.bfloat16 if b_code == _cabi.LF_DTYPE_E4M3 else B.dtype
    if out is None:
        out = torch.empty((r1 - r0, N), dtype=out_dtype, device=B.device)
    _need(out.dtype == out_dtype, "out must have out_dtype")
    ldc = _matrix(out, "out", r1 - r0, N, dev)
    c_ptr = out.data_ptr()
    b_ptr = b_type = r_ptr = r_type = ld_res = z_ptr = ld_z = 0
    if bias is not None:
        b_ptr, b_type = _vector(bias, "bias", N, dev), _code(bias.dtype)
    if residual is not None:
        r_ptr, r_type, ld_res = residual.data_ptr(), _code(residual.dtype), _matrix(residual, "residual", r1 - r0, N, dev)
    if preact is not None:
        _need(preact.dtype == out_dtype, "preact must have the result's type")
        z_ptr, ld_z = preact.data_ptr(), _matrix(preact, "preact", r1 - r0, N, dev)
    ep = LfEpilogue(b_ptr, r_ptr, z_ptr, ld_res, ld_z, b_type, r_type, act)
    s_ptr = 0 if scale is None else _vector(scale, "scale", K, dev, torch.float32)
    nbytes = lib.lf_spmm_csr_act_workspace_bytes(nnz, N, b_code)
    keep, ws, nws = _scratch(nbytes, workspace, B)
    call = (a.indptr.data_ptr(), a.indices.data_ptr(), data, order, r0, r1, nnz, B.data_ptr(), b_code, ldb, s_ptr, c_ptr,
            _code(out_dtype), ldc, N, C.byref(ep), ws, nws, stream_of(dev))
    _run(lib.lf_spmm_csr_act, call, dev)
    return out


def act_backward(dy, preact=None, activation: Optional[str] = None, dz=None, need_dz: bool = True, need_dbias: bool = True,
                 dbias=None, workspace: Optional[Workspace] = None, dz_dtype=None):
    """``lf_act_backward_as``: ``(dz, dbias)`` with ``dz = dy * activation'(preact)`` in ``dz_dtype`` (dy's, the default, or
    float32) and ``dbias`` the float32 sum of its rows before they are rounded; what is not needed is None.  ``dz`` may be
    ``dy`` or ``preact``."""
    torch = _torch()
    _no_graph(dy, preact)
    if dz is not None or dbias is not None:
        _outputs_apart(((dz, "dz"), (dbias, "dbias")), ((dy, "dy"), (preact, "preact")), (("dz", "dy"), ("dz", "preact")))
    lib = _cabi.load()
    M, N, dev = _first(dy, "dy")
    act = _act_code(activation)
    code, ld_dy, ld_z = _code(dy.dtype), _matrix(dy, "dy", M, N, dev), 0
    if act != _cabi.LF_ACT_NONE:
        _need(preact is not None and preact.dtype == dy.dtype, "preact must be given, in dy's type")
        ld_z = _matrix(preact, "preact", M, N, dev)
    if dz_dtype is None:
        dz_dtype = dy.dtype if dz is None else dz.dtype
    if dz is None and need_dz:
        dz = _rows_like(dy, dz_dtype)
    if dbias is None and need_dbias:
        dbias = torch.empty(N, dtype=torch.float32, device=dy.device)
    _need(dz is not None or dbias is not None, "nothing to compute")
    _need(dz is None or (dz.dtype == dz_dtype and dz_dtype in (dy.dtype, torch.float32)), "dz must have dz_dtype: dy's type or float32")
    ld_dz = 0 if dz is None else _matrix(dz, "dz", M, N, dev)
    b_ptr = 0 if dbias is None else _vector(dbias, "dbias", N, dev, torch.float32)
    nbytes = 0 if dbias is None else lib.lf_act_backward_workspace_bytes(M, N)
    keep, ws, nws = _scratch(nbytes, workspace, dy)
    call = (dy.data_ptr(), ld_dy, 0 if act == _cabi.LF_ACT_NONE else preact.data_ptr(), ld_z, code, act,
            0 if dz is None else dz.data_ptr(), code if dz is None else _code(dz_dtype), ld_dz, b_ptr, M, N, ws, nws, stream_of(dev))
    _run(lib.lf_act_backward_as, call, dev)
    return dz, dbias


def spmm_csr_grad_values(a: DeviceCsr, B, dy, preact=None, activation: Optional[str] = None, out=None):
    """``lf_spmm_csr_grad_values``: the gradient of A's values, ``dvalues[e] = <dz[row of e], B[column of e]>`` with
    ``dz = dy * activation'(preact)`` not rounded in between; float32, one per entry.  For a ``DeviceCsr`` of a slice of
    ``indptr`` the entries count from the slice's first, and what is behind its last is left as it is."""
    torch = _torch()
    _no_graph(B, dy, preact)
    if out is not None:
        _outputs_apart(((out, "out"),), ((B, "B"), (dy, "dy"), (preact, "preact")))
    K, N, dev = _first(B, "B")
    M = a.shape[0]
    _need(K == a.shape[1], "B must have one row per matrix column")
    act = _act_code(activation)
    _csr_arrays(a, None, dev)
    ldb, ld_dy, ld_z = _matrix(B, "B", K, N, dev), _matrix(dy, "dy", M, N, dev), 0
    if act != _cabi.LF_ACT_NONE:
        _need(preact is not None and preact.dtype == dy.dtype, "preact must be given, in dy's type")
        ld_z = _matrix(preact, "preact", M, N, dev)
    if out is None:
        out = torch.empty(a.nnz, dtype=torch.float32, device=B.device)
    o_ptr = _vector(out, "out", a.nnz, dev, torch.float32)
    call = (a.indptr.data_ptr(), a.indices.data_ptr(), 0, M, a.nnz, dy.data_ptr(), ld_dy,
            0 if act == _cabi.LF_ACT_NONE else preact.data_ptr(), ld_z, _code(dy.dtype), act, B.data_ptr(), _code(B.dtype), ldb,
            N, o_ptr, stream_of(dev))
    _run(_cabi.load().lf_spmm_csr_grad_values, call, dev)
    return out


class ActGradients(NamedTuple):
    dB: Optional["object"]        # in B's type
    dvalues: Optional["object"]   # float32, one per entry of A
    dbias: Optional["object"]     # float32


def spmm_csr_act_backward(a: DeviceCsr, a_t: Optional[CsrTranspose], B, dy, preact=None, activation: Optional[str] = None,
                          need=("dB", "dvalues", "dbias"), workspace: Optional[Workspace] = None, dz_dtype=None) -> ActGradients:
    """Gradients of ``spmm_csr_act(a, B, bias=..., activation=..., preact=...)`` from ``dy``, the gradient of its result
    (which is also that of the residual): ``act_backward``, ``A^T @ dz`` and ``spmm_csr_grad_values``.  ``preact`` and dy
    have one type, 16 or 32 bits like B (8-bit rows have no gradient here); ``need`` names the ones wanted, ``a_t`` is
    used for dB only.  dB is made of dz rounded to ``dz_dtype``, dy's type or float32; dvalues and dbias take it unrounded.
    The default is dy's type, except for float16 and an activation with slopes beside 0 and 1: there dz may pass 65504 or
    vanish where dB would not, so it is float32 (twice the bytes gathered)."""
    unknown = set(need) - {"dB", "dvalues", "dbias"}
    _need(not unknown, "need names dB, dvalues and dbias")
    _code(B.dtype)
    dB = dvalues = dbias = None
    dz = dy
    plain = _act_code(activation) == _cabi.LF_ACT_NONE
    _need("dB" not in need or (a_t is not None and a_t.shape == (a.shape[1], a.shape[0]) and a_t.nnz == a.nnz),
          "dB needs the transposed pattern of a")
    want_dz = "dB" in need and not plain
    if dz_dtype is None and dy.dtype == _torch().float16 and activation != "relu":
        dz_dtype = _torch().float32
    if want_dz or "dbias" in need:
        got, dbias = act_backward(dy, preact, activation, need_dz=want_dz, need_dbias="dbias" in need, workspace=workspace,
                                  dz_dtype=dz_dtype if want_dz else None)
        dz = got if want_dz else dy
    if "dB" in need:
        dB = spmm_csr_act(a_t, dz, values=a.data, out_dtype=B.dtype, workspace=workspace)
    if "dvalues" in need:
        dvalues = spmm_csr_grad_values(a, B, dy, preact, activation)
    return ActGradients(dB, dvalues, dbias)
