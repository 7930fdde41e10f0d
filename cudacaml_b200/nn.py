"""Operators of residual blocks with experts, on device memory: ``dropout`` from
the counter-based generator of ``rng`` with a mask that is never stored,
``block_norm`` (the norms around a block fused with its gate, dropout and
residual scale) and ``grouped_matmul`` (products grouped by expert with ragged
sizes), each with its gradient. No counterpart in the reference.

Each function issues its kernels on ``stream`` (a ``runtime.Stream``, a raw
handle, or None for the legacy default stream) on the current device and does
not synchronise; outputs are given by the caller. A matrix argument is an
``Array``, a ``backend_cuda.Resident``, or any object in device memory with
``data_ptr()``, ``dtype``, ``shape`` and ``stride()``. Matrices have unit
stride along a row and any stride between rows; a tensor of rank 1 is one row,
one of rank above 2 has to be dense and counts as rows of its last axis.
Element types are f32, bf16 and f16; arithmetic is in 32 bits. Caller mistakes
raise ValueError before anything is issued.
"""
from __future__ import annotations

import ctypes
import struct
from dataclasses import dataclass
from typing import Optional

from . import runtime as R
from .backend_cuda import Resident

F32, BF16, F16, I32 = "f32", "bf16", "f16", "i32"

_CODES = {F32: 0, I32: 2, BF16: 4, F16: 5}
_NAMES = {v: k for k, v in _CODES.items()}
_BY_TEXT = {"torch.float32": 0, "torch.int32": 2, "torch.bfloat16": 4, "torch.float16": 5, "float32": 0, "int32": 2,
            "bfloat16": 4, "float16": 5, "f32": 0, "i32": 2, "bf16": 4, "f16": 5}
_BY_TYPE: dict = {}  # dtype object -> code, filled from _BY_TEXT

KINDS = {"rms": 0, "layer": 1}
ACTS = {"none": 0, "sigmoid": 1, "tanh": 2}


@dataclass
class Array:
    """A view of device memory: pointer, element type ("f32", "bf16", "f16",
    "i32"), shape, and strides in elements (None: dense)."""

    ptr: int
    dtype: str
    shape: tuple
    strides: Optional[tuple] = None


def _code(dtype, what):
    try:
        return _BY_TYPE[dtype]
    except KeyError:
        text = getattr(dtype, "value", None) or str(dtype)
        if text not in _BY_TEXT:
            raise ValueError(f"{what} has element type {text}: f32, bf16, f16 (or i32 for offsets) are supported") from None
        _BY_TYPE[dtype] = _BY_TEXT[text]
        return _BY_TEXT[text]


def _dense(shape):
    out, n = [], 1
    for d in reversed(shape):
        out.append(n)
        n *= max(d, 1)
    return tuple(reversed(out))


def _see(x, what):
    """(pointer, type code, shape, strides) of an argument in device memory."""
    try:
        ptr, dtype, shape, strides, here = x.data_ptr, x.dtype, x.shape, x.stride, x.is_cuda
    except AttributeError:
        if isinstance(x, Array):
            shape = tuple(x.shape)
            return x.ptr or 0, _code(x.dtype, what), shape, tuple(x.strides) if x.strides is not None else _dense(shape)
        if isinstance(x, Resident):
            return x.buf.ptr or 0, _code(x.dtype, what), tuple(x.shape), _dense(x.shape)
        raise ValueError(f"{what} is a {type(x).__name__}: an array in device memory is needed") from None
    if not here:
        raise ValueError(f"{what} is not in device memory")
    code = _BY_TYPE.get(dtype)
    return ptr(), _code(dtype, what) if code is None else code, shape, strides()


def _mat(x, what):
    """(pointer, type code, rows, cols, row stride)."""
    try:  # the common case in few steps: a dense matrix of another library
        if x.is_contiguous() and x.is_cuda:
            rows, cols = x.shape
            return x.data_ptr(), _BY_TYPE[x.dtype], rows, cols, cols
    except (AttributeError, ValueError, KeyError):
        pass
    ptr, code, shape, strides = _see(x, what)
    rank = len(shape)
    if rank == 2:
        rows, cols = shape
        stride, along = strides
        if along != 1 and cols > 1:
            raise ValueError(f"{what} has stride {along} along its rows: 1 is needed")
        return ptr, code, rows, cols, stride if rows > 1 else cols
    if rank == 0:
        return ptr, code, 1, 1, 1
    cols = shape[-1]
    if rank == 1:
        if cols > 1 and strides[0] != 1:
            raise ValueError(f"{what} has stride {strides[0]}: 1 is needed")
        return ptr, code, 1, cols, cols
    rows = 1
    for d in shape[:-1]:
        rows *= d
    want = _dense(shape)
    if rows * cols and any(s != w for s, w, d in zip(strides, want, shape) if d > 1):
        raise ValueError(f"{what} has rank {rank} and is not dense")
    return ptr, code, rows, cols, cols


def _stack(x, what):
    """(pointer, type code, count, rows, cols, stride, row stride) of a rank-3 array."""
    ptr, code, shape, strides = _see(x, what)
    if len(shape) != 3:
        raise ValueError(f"{what} has rank {len(shape)}: [experts, rows, cols] is needed")
    count, rows, cols = shape
    if cols > 1 and strides[2] != 1:
        raise ValueError(f"{what} has stride {strides[2]} along its rows: 1 is needed")
    return ptr, code, count, rows, cols, strides[0] if count > 1 else rows * cols, strides[1] if rows > 1 else cols


def _vector(x, cols, what):
    """(pointer, type code) of a dense vector of `cols`, or (0, None)."""
    if x is None:
        return 0, None
    try:
        if x.is_contiguous() and x.is_cuda and x.shape == (cols,):
            return x.data_ptr(), _BY_TYPE[x.dtype]
    except (AttributeError, KeyError):
        pass
    ptr, code, rows, n, _ = _mat(x, what)
    if rows != 1 or n != cols:
        raise ValueError(f"{what} has {rows * n} elements, expected {cols}")
    return ptr, code


def _same(got, want, what):
    if got != want:
        raise ValueError(f"{what} has shape {list(got)}, expected {list(want)}")


def _typed(code, want, what):
    if code != want:
        raise ValueError(f"{what} has element type {_NAMES.get(code, code)}, expected {_NAMES.get(want, want)}")


def _floats(code, what):
    if code == 2:
        raise ValueError(f"{what} has element type i32: f32, bf16 or f16 is needed")


def _word(v, what):
    if not 0 <= v <= 0xFFFFFFFFFFFFFFFF:
        raise ValueError(f"{what} = {v} is outside [0, 2^64)")
    return v


def _space(ws):
    """(pointer, bytes) of a workspace: a runtime.Buffer, an array, or None."""
    if ws is None:
        return 0, 0
    if isinstance(ws, R.Buffer):
        return ws.ptr or 0, ws.nbytes
    if isinstance(ws, (Array, Resident)):
        ptr, code, shape, _ = _see(ws, "workspace")
        n = 2 if code >= 4 else 4
        for d in shape:
            n *= d
        return ptr, n
    if not getattr(ws, "is_cuda", True):
        raise ValueError("workspace is not in device memory")
    return ws.data_ptr(), ws.numel() * ws.element_size()


def _call(name, args, stream):
    rc = getattr(R._LIB or R.lib(), name)(args, stream.h if isinstance(stream, R.Stream) else stream)
    if rc:
        R.check(rc)


def _bytes_of(name, *args):
    n = ctypes.c_size_t()
    rc = getattr(R._LIB or R.lib(), name)(*args, ctypes.byref(n))
    if rc:
        R.check(rc)
    return n.value


# ------------------------------------------------------------------ dropout
_DROPOUT = struct.Struct("@3P5q3Qdi0P")


def dropout(x, p, seed, out, *, offset=0, base=0, residual=None, stream=None) -> None:
    """out = residual + keep * x / (1 - p).

    Element ``e = base + row * cols + col`` is kept unless word ``e % 4`` of
    Philox-4x32-10 at counter ``(e // 4, offset)`` (64 bits each) under key
    ``seed`` is below ``round(p * 2**32)``. The mask is a function of the
    seed, the offset and the index alone: give each call of a step its own
    offset, and each rank that holds a slice of rows its first index as base.
    ``out`` may be ``x`` or ``residual``."""
    xp, code, rows, cols, xs = _mat(x, "nn.dropout: x")
    _floats(code, "nn.dropout: x")
    op, oc, orows, ocols, os_ = _mat(out, "nn.dropout: out")
    _same((orows, ocols), (rows, cols), "nn.dropout: out")
    _typed(oc, code, "nn.dropout: out")
    rp, rs = 0, 0
    if residual is not None:
        rp, rc, rrows, rcols, rs = _mat(residual, "nn.dropout: residual")
        _same((rrows, rcols), (rows, cols), "nn.dropout: residual")
        _typed(rc, code, "nn.dropout: residual")
    _call("ccb_nn_dropout", _DROPOUT.pack(xp, rp, op, rows, cols, xs, rs, os_, _word(seed, "nn.dropout: seed"), _word(offset, "nn.dropout: offset"),
                                          _word(base, "nn.dropout: base"), p, code), stream)


def dropout_backward(dy, p, seed, out, *, offset=0, base=0, stream=None) -> None:
    """out = the gradient of ``dropout``'s x: keep * dy / (1 - p), with the
    mask of the same seed, offset and base. (The residual's gradient is dy.)"""
    dropout(dy, p, seed, out, offset=offset, base=base, stream=stream)


# --------------------------------------------------------------- block norms
_NORM = struct.Struct("@9P7q3Q3d7i0P")
_NORM_BACK = struct.Struct("@8P8P10q4Q3d7i0P")


def _like(x, rows, cols, code, what):
    """(pointer, row stride) of an optional matrix of the given size and type."""
    if x is None:
        return 0, 0
    ptr, c, r, n, s = _mat(x, what)
    if r != rows or n != cols:
        _same((r, n), (rows, cols), what)
    if c != code:
        _typed(c, code, what)
    return ptr, s


def _gate(gate, rows, cols, code):
    """(pointer, row stride, type code): rank 1 is one row for all, stride 0."""
    if gate is None:
        return 0, 0, 0
    if len(gate.shape) == 1:
        ptr, c = _vector(gate, cols, "nn.block_norm: gate")
        stride = 0
    else:
        ptr, c, r, n, stride = _mat(gate, "nn.block_norm: gate")
        _same((r, n), (rows, cols), "nn.block_norm: gate")
        if rows > 1 and stride < cols:
            raise ValueError("nn.block_norm: the gate's rows overlap (a gate for each channel has rank 1)")
    if c != 0 and c != code:
        raise ValueError("nn.block_norm: the gate has neither the branch's element type nor f32")
    return ptr, stride, c


def _pick(table, name, what):
    if name not in table:
        raise ValueError(f"nn.block_norm: {what} {name!r} (one of {', '.join(table)})")
    return table[name]


def _weights(cols, *named):
    """The pointers of the optional vectors, and their common type code."""
    code, out = None, []
    for name, v in named:
        if v is None:
            out.append(0)
            continue
        ptr, c = _vector(v, cols, name)
        if c == 2:
            _floats(c, name)
        if code is not None and c != code:
            raise ValueError("nn.block_norm: weights and biases have different element types")
        code = c
        out.append(ptr)
    return out, code or 0


def block_norm(x, y=None, h=None, *, kind="rms", eps=1e-6, branch=None, post_norm=True, post_weight=None, post_bias=None, gate=None,
               gate_act="none", scale=1.0, p=0.0, seed=0, offset=0, base=0, pre_weight=None, pre_bias=None, stream=None) -> None:
    """The join of a residual block and the next block's norm, in one pass::

        u = norm(branch) * post_weight + post_bias     (u = branch without post_norm)
        y = x + scale * drop(act(gate) * u)
        h = norm(y) * pre_weight + pre_bias            (from y before its rounding)

    ``kind`` "rms" is v / sqrt(mean(v^2) + eps) along a row, "layer" the same
    of v - mean(v). Without a branch y is x and only h is written. ``gate``
    has x's shape, or rank 1 for one gate a channel; ``gate_act`` is "none",
    "sigmoid" or "tanh". drop is ``dropout`` with p, seed, offset and base. x
    and y may be f32 beside 16-bit branch and h. Either output may be None;
    y may be x."""
    xp, xc, rows, cols, xs = _mat(x, "nn.block_norm: x")
    _floats(xc, "nn.block_norm: x")
    code = xc
    if branch is not None:
        bp, code, brows, bcols, bs = _mat(branch, "nn.block_norm: branch")
        _same((brows, bcols), (rows, cols), "nn.block_norm: branch")
    else:
        bp, bs = 0, 0
        if h is not None:
            code = _mat(h, "nn.block_norm: h")[1]
    if xc != code and xc != 0:
        raise ValueError("nn.block_norm: x has neither the branch's (or h's) element type nor f32")
    yp, ys = _like(y, rows, cols, xc, "nn.block_norm: y")
    hp, hs = _like(h, rows, cols, code, "nn.block_norm: h")
    gp, gs, gc = _gate(gate, rows, cols, code)
    (w1, c1, w2, c2), wc = _weights(cols, ("nn.block_norm: pre_weight", pre_weight), ("nn.block_norm: pre_bias", pre_bias), ("nn.block_norm: post_weight", post_weight), ("nn.block_norm: post_bias", post_bias))
    _call("ccb_nn_block_norm", _NORM.pack(xp, bp, gp, w1, c1, w2, c2, yp, hp, rows, cols, xs, bs, gs, ys, hs, _word(seed, "nn.block_norm: seed"),
                                          _word(offset, "nn.block_norm: offset"), _word(base, "nn.block_norm: base"), p, eps, scale, code, xc, gc, wc,
                                          _pick(KINDS, kind, "kind"), _pick(ACTS, gate_act, "gate_act"), 1 if post_norm else 0), stream)


def block_norm_backward_workspace(rows: int, cols: int) -> int:
    """Bytes of workspace that ``block_norm_backward`` needs at these sizes."""
    return _bytes_of("ccb_nn_block_norm_backward_workspace", rows, cols)


def block_norm_backward(y, *, dy=None, dh=None, dx=None, dbranch=None, dgate=None, dpre_weight=None, dpre_bias=None, dpost_weight=None,
                        dpost_bias=None, workspace=None, kind="rms", eps=1e-6, branch=None, post_norm=True, post_weight=None, post_bias=None,
                        gate=None, gate_act="none", scale=1.0, p=0.0, seed=0, offset=0, base=0, pre_weight=None, pre_bias=None, stream=None) -> None:
    """The gradient of ``block_norm``, from its stored y (x itself where it had
    no branch) and its other inputs. ``dy`` and ``dh`` are the gradients of y
    and h (either may be None: zero). ``dx`` is the whole gradient of x,
    ``dbranch`` and ``dgate`` have their inputs' types (the gradient of a gate
    for each channel is f32), those of weights and biases are f32. Gradients
    that are None are not computed. ``workspace`` (needed for any gradient
    that is summed over rows): ``block_norm_backward_workspace`` bytes.
    dx may be dy, dbranch may be dh."""
    yp, xc, rows, cols, ys = _mat(y, "nn.block_norm: y")
    _floats(xc, "nn.block_norm: y")
    code = xc
    if branch is not None:
        code = _mat(branch, "nn.block_norm: branch")[1]
    elif dh is not None:
        code = _mat(dh, "nn.block_norm: dh")[1]
    if xc != code and xc != 0:
        raise ValueError("nn.block_norm: y has neither the branch's (or dh's) element type nor f32")
    bp, bs = _like(branch, rows, cols, code, "nn.block_norm: branch")
    dyp, dys = _like(dy, rows, cols, xc, "nn.block_norm: dy")
    dhp, dhs = _like(dh, rows, cols, code, "nn.block_norm: dh")
    dxp, dxs = _like(dx, rows, cols, xc, "nn.block_norm: dx")
    dbp, dbs = _like(dbranch, rows, cols, code, "nn.block_norm: dbranch")
    gp, gs, gc = _gate(gate, rows, cols, code)
    dgp, dgs = 0, 0
    if dgate is not None:
        if gate is None:
            raise ValueError("nn.block_norm: dgate without a gate")
        if len(gate.shape) == 1:
            dgp, c = _vector(dgate, cols, "nn.block_norm: dgate")
            _typed(c, 0, "nn.block_norm: dgate")
        else:
            dgp, dgs = _like(dgate, rows, cols, gc, "nn.block_norm: dgate")
    # biases have no part in the gradient but for the gate's, through u
    (w1, w2, c2), wc = _weights(cols, ("nn.block_norm: pre_weight", pre_weight), ("nn.block_norm: post_weight", post_weight), ("nn.block_norm: post_bias", post_bias))
    sums = []
    for name, v in (("nn.block_norm: dpre_weight", dpre_weight), ("nn.block_norm: dpre_bias", dpre_bias), ("nn.block_norm: dpost_weight", dpost_weight), ("nn.block_norm: dpost_bias", dpost_bias)):
        ptr, c = _vector(v, cols, name)
        if c:
            _typed(c, 0, name)
        sums.append(ptr)
    wp, wn = _space(workspace)
    _call("ccb_nn_block_norm_backward",
          _NORM_BACK.pack(yp, dyp, dhp, bp, gp, w1, w2, c2, dxp, dbp, dgp, *sums, wp, rows, cols, ys, dys, dhs, bs, gs, dxs, dbs, dgs, wn,
                          _word(seed, "nn.block_norm: seed"), _word(offset, "nn.block_norm: offset"), _word(base, "nn.block_norm: base"), p, eps,
                          scale, code, xc, gc, wc, _pick(KINDS, kind, "kind"), _pick(ACTS, gate_act, "gate_act"), 1 if post_norm else 0), stream)


# ---------------------------------------------------------- grouped products
_GROUPED = struct.Struct("@6P8qQ2i0P")
_GROUPED_DW = struct.Struct("@6P8qQ2i0P")


def _offsets(offsets, experts, what):
    ptr, code, shape, strides = _see(offsets, f"{what}: offsets")
    _typed(code, 2, f"{what}: offsets")
    if len(shape) != 1 or shape[0] != experts + 1 or (shape[0] > 1 and strides[0] != 1):
        raise ValueError(f"{what}: offsets has shape {list(shape)}, expected [{experts + 1}], dense")
    return ptr


def _err(err, what):
    """The pointer of an optional 32-bit error word: an i32 array, a Buffer, or a raw pointer."""
    if err is None or isinstance(err, int):
        return err or 0
    if isinstance(err, R.Buffer):
        if err.nbytes < 4:
            raise ValueError(f"{what}: err is {err.nbytes} bytes: 4 are needed")
        return err.ptr or 0
    ptr, code, _, _ = _see(err, f"{what}: err")
    _typed(code, 2, f"{what}: err")
    return ptr


def _grouped_args(x, w, offsets, out, transpose_w, workspace, err):
    me = "nn.grouped_matmul"
    xp, code, rows, k, xs = _mat(x, f"{me}: x")
    _floats(code, f"{me}: x")
    wp, wc, experts, a, b, we, ws = _stack(w, f"{me}: w")
    _typed(wc, code, f"{me}: w")
    wk, n = (b, a) if transpose_w else (a, b)
    if wk != k:
        raise ValueError(f"{me}: x has {k} columns and each matrix of w {wk} rows" + (" (transposed)" if transpose_w else ""))
    op, oc, orows, on, os_ = _mat(out, f"{me}: out")
    _same((orows, on), (rows, n), f"{me}: out")
    _typed(oc, code, f"{me}: out")
    fp = _offsets(offsets, experts, me) if offsets is not None else 0
    sp, sn = _space(workspace)
    return _GROUPED.pack(xp, wp, fp, op, sp, _err(err, me), rows, experts, k, n, xs, we, ws, os_, sn, code, 1 if transpose_w else 0)


def grouped_matmul_workspace(x, w, out, *, transpose_w=False) -> int:
    """Bytes of workspace that ``grouped_matmul`` needs for these arrays (0: none)."""
    return _bytes_of("ccb_nn_grouped_matmul_workspace", _grouped_args(x, w, None, out, transpose_w, None, None))


def grouped_matmul(x, w, offsets, out, *, transpose_w=False, workspace=None, err=None, stream=None) -> None:
    """out[r] = x[r] @ w[e] for the rows ``offsets[e] <= r < offsets[e + 1]`` of
    each expert e; rows of no expert give 0. x is [rows, k], w [experts, k, n]
    (or [experts, n, k] with ``transpose_w``), out [rows, n], all of one type;
    ``offsets`` is experts + 1 ascending i32 words in device memory that the
    host does not read. Words out of order or range are clamped and raise bit
    64 of the 32-bit word ``err``; bit 16 says that a wait inside the kernel ran
    out and ``out`` is undefined. The gradient of x is the same call on dy
    with ``transpose_w`` flipped, that of w is ``grouped_matmul_dw``. f32 operands
    are multiplied as three 16-bit planes each, as exact as f32 arithmetic for
    numbers of 2**-110 and more; the planes lie in the workspace, 6 bytes for every
    number of x and of w, also of experts without rows."""
    _call("ccb_nn_grouped_matmul", _grouped_args(x, w, offsets, out, transpose_w, workspace, err), stream)


def _dw_args(x, dy, offsets, out, workspace, err):
    me = "nn.grouped_matmul_dw"
    xp, code, rows, k, xs = _mat(x, f"{me}: x")
    _floats(code, f"{me}: x")
    yp, yc, yrows, n, ys = _mat(dy, f"{me}: dy")
    _typed(yc, code, f"{me}: dy")
    if yrows != rows:
        raise ValueError(f"{me}: x has {rows} rows and dy {yrows}")
    op, oc, experts, ok, on, oe, os_ = _stack(out, f"{me}: out")
    _same((ok, on), (k, n), f"{me}: a matrix of out")
    if oc != 0 and oc != code:
        raise ValueError(f"{me}: out has neither x's element type nor f32")
    fp = _offsets(offsets, experts, me) if offsets is not None else 0
    sp, sn = _space(workspace)
    return _GROUPED_DW.pack(xp, yp, fp, op, sp, _err(err, me), rows, experts, k, n, xs, ys, oe, os_, sn, code, oc)


def grouped_matmul_dw_workspace(x, dy, out) -> int:
    """Bytes of workspace that ``grouped_matmul_dw`` needs for these arrays (0: none)."""
    return _bytes_of("ccb_nn_grouped_matmul_dw_workspace", _dw_args(x, dy, None, out, None, None))


def grouped_matmul_dw(x, dy, offsets, out, *, workspace=None, err=None, stream=None) -> None:
    """out[e] = x[rows of e].T @ dy[rows of e], 0 for an expert without rows: the
    gradient of ``grouped_matmul``'s w ([experts, k, n]; for a transposed w
    swap x and dy). out has x's type or f32."""
    _call("ccb_nn_grouped_matmul_dw", _dw_args(x, dy, offsets, out, workspace, err), stream)


def wait_polls(polls: int = 0) -> None:
    """How often a wait inside the grouped products polls before it gives up
    (bit 16 of ``err``, the output undefined, the stream usable), for the calls
    that follow; 0 is the default, 2**22 (4 us each: 16 s)."""
    if not 0 <= polls < 1 << 32:
        raise ValueError(f"nn.wait_polls: {polls} is outside [0, 2^32)")
    R.check((R._LIB or R.lib()).ccb_nn_wait_polls(polls))
