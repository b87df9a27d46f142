"""Matrix operators of few bits: 8-bit rows and their products, and orthogonalisation by Newton-Schulz products.

They stand next to the 64-bit matrix calls of ``hotpath`` (``gram``, ``rotate``, ``eigh``, ``cholesky``) and take float32, float16 and bfloat16
matrices.  (The reference computes in 64 bits throughout: it has no counterpart.)  Three kinds of arrays go in, and the same kind comes out:

* tensors of a tensor library that the caller has imported (torch on the GPU): the call is put on the tensor's device's current stream and does not
  wait; it can be captured into a graph, but for the first call on a device.  Nothing is imported here for it.  The operators are not differentiated: a
  tensor that asks for gradients is refused while gradients are recorded, one with a tangent of forward mode always.
* ``DeviceArray``: the context's own stream; the call returns when the result is there.
* NumPy arrays: copied to the GPU and back.

Wrong shapes, types and devices raise ``ValueError`` before anything is launched.
"""

from __future__ import annotations

import ctypes as C
import math
import sys

import numpy as np

from ._lib import Context, DeviceArray, _default_ctx, default_context

__all__ = ["NEWTON_SCHULZ", "quantize_rows", "int8_matmul", "int8_linear", "orthogonalize"]

#: (a, b, c) of X <- a X + (b A + c A A) X, as published by K. Jordan et al. (2024): odd polynomial of degree five that takes singular values in (0, 1] to about 0.7 .. 1.2 in five steps
#: (slope 3.44 at zero).  A step with (1.5, -0.5, 0) or (1.875, -1.25, 0.375) afterwards takes them on towards 1.
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)

MAX_K = 131071  # NLS_INT8_MAX_K
_MAX_LD = (2**32 - 1) // 512  # the longest way from an 8-bit row to the next that the kernels take
_A_PADDED, _B_PADDED = 1, 2
_NAMES = ("float32", "float16", "bfloat16")  # the position is the type's number in the C ABI
_NAMED = {name: i for i, name in enumerate(_NAMES)}


def _kind_of(dtype, what) -> int:
    """The number of a float type given as text, as NumPy's or as a tensor library's."""
    text = str(dtype)
    if text.startswith("torch."):
        text = text[6:]
    elif text not in _NAMES:
        try:
            text = np.dtype(dtype).name
        except TypeError:
            pass
    if text not in _NAMES:
        raise ValueError(f"{what} is {text}; the operators of few bits take {', '.join(_NAMES)}")
    return _NAMES.index(text)


def _up16(k: int) -> int:
    return (k + 15) & -16


class _Tensors:
    """Tensors of an imported tensor library on one device, worked on in that device's current stream."""

    host = False

    def __init__(self, lib, index, ctx):
        self.lib, self.index, self.ctx = lib, index, ctx
        self.device = lib.device("cuda", index)
        self.kinds = {getattr(lib, name): i for i, name in enumerate(_NAMES)}
        self.named = {**self.kinds, **_NAMED}
        self.ptr, self.strides, self.dense = lib.Tensor.data_ptr, lib.Tensor.stride, lib.Tensor.contiguous
        self.types = tuple(getattr(lib, name) for name in _NAMES)
        self.int8, self.float32, self.uint8, self.strided, self.Tensor = lib.int8, lib.float32, lib.uint8, lib.strided, lib.Tensor
        self._empty, self._forward = lib.empty, lib.autograd.forward_ad
        self._raw_stream = getattr(lib._C, "_cuda_getCurrentRawStream", None)

    def begin(self):
        if self._raw_stream is not None:
            return self._raw_stream(self.index)
        return self.lib.cuda.current_stream(self.device).cuda_stream

    def take(self, x, what):
        if not isinstance(x, self.Tensor):
            raise ValueError(f"{what} must be a tensor like the other arguments, not {type(x).__name__}")
        if x.get_device() != self.index:
            raise ValueError(f"{what} is on {x.device}, the other arguments on {self.device}")
        if x.layout is not self.strided:
            raise ValueError(f"{what} must be a dense tensor")
        if x.requires_grad and self.lib.is_grad_enabled():
            raise ValueError(f"{what} asks for gradients, which this operator does not give: detach it, or call under no_grad")
        if self._forward.unpack_dual(x).tangent is not None:
            raise ValueError(f"{what} has a tangent, and this operator gives no gradients in forward mode either: hand over its primal")
        return x.resolve_neg() if x.is_neg() else x

    @staticmethod
    def room(x):
        """Bytes of the tensor's memory from its first element on."""
        return x.untyped_storage().nbytes() - x.storage_offset() * x.element_size()

    def empty(self, shape, dtype):
        return self._empty(*shape, dtype=dtype, device=self.device) if shape else self._empty((), dtype=dtype, device=self.device)

    def rows(self, rows, k, ld, lead):
        held = self._empty(*lead, ld, dtype=self.int8, device=self.device)
        return held, held if ld == k else held[..., :k]

    def derived(self):
        """Whether tensors may have tangents: a level of forward mode is open (or not to be seen from here)."""
        return getattr(self._forward, "_current_level", 0) >= 0

    # The usual arguments - dense matrices - in the few checks they need; all others, wrong ones among them, the long way.
    def float_rows(self, x, what):
        if not self.derived() and isinstance(x, self.Tensor) and x.get_device() == self.index and x.layout is self.strided and x.is_contiguous() and not x.requires_grad and not x.is_neg():
            shape, kind = x.shape, self.kinds.get(x.dtype)
            if kind is not None and len(shape) == 2 and shape[1] > 0:
                return x, shape[:1], shape[0], shape[1], shape[1], 1, kind
        return _float_rows(self, x, what)

    def int8_rows(self, x, what, scale, scale_what):
        T, strided = self.Tensor, self.strided
        if (
            isinstance(x, T) and isinstance(scale, T) and x.dtype is self.int8 and scale.dtype is self.float32
            and x.get_device() == self.index == scale.get_device() and x.layout is strided is scale.layout
            and scale.is_contiguous() and not scale.requires_grad and not scale.is_neg() and not self.derived()
        ):  # fmt: skip
            shape = x.shape
            if len(shape) == 2 and scale.shape == shape[:1] and 0 < shape[1] <= MAX_K:
                rows, k = shape
                ld, dense = x.stride()
                if dense == 1 and rows > 1 and k <= ld <= _MAX_LD:
                    if not k & 15:
                        return x, scale, shape[:1], rows, k, ld, True
                    up = (k + 15) & -16
                    return x, scale, shape[:1], rows, k, ld, ld >= up and self.room(x) >= (rows - 1) * ld + up
                if dense == 1 and rows == 1 and not k & 15:
                    return x, scale, shape[:1], rows, k, k, True
        return _int8_rows(self, x, what, scale, scale_what)

    def scratch(self, nbytes):
        return self.lib.empty(nbytes, dtype=self.uint8, device=self.device)

    @staticmethod
    def done(result):
        return result


class _Arrays:
    """NumPy arrays and DeviceArrays, on the context's own stream; results come back as what went in."""

    kinds = {np.dtype("float32"): 0, np.dtype("float16"): 1}
    named = _NAMED
    types = (np.dtype("float32"), np.dtype("float16"))
    int8, float32 = np.dtype("int8"), np.dtype("float32")

    def __init__(self, first, ctx):
        self.host = isinstance(first, np.ndarray)
        self.ctx = first.ctx if ctx is None and not self.host else ctx
        self._keep = []  # device copies and scratch live until the stream has been waited for

    def begin(self):
        if self.ctx is None:
            self.ctx = default_context()
        stream = C.c_void_p()
        self.ctx._check(self.ctx.lib.nls_ctx_stream(self.ctx.handle, C.byref(stream)))
        return stream.value

    def take(self, x, what):
        if self.host != isinstance(x, np.ndarray) or not isinstance(x, (np.ndarray, DeviceArray)):
            raise ValueError(f"{what} must be an array like the other arguments, not {type(x).__name__}")
        if not self.host and x.ctx.device != self.ctx.device:
            raise ValueError(f"{what} is on GPU {x.ctx.device}, the context on GPU {self.ctx.device}")
        return x.astype(x.dtype.newbyteorder("=")) if self.host and not x.dtype.isnative else x

    def ptr(self, x):
        if isinstance(x, DeviceArray):
            return x.ptr
        d = self.ctx.to_device(x, dtype=x.dtype)
        self._keep.append(d)
        return d.ptr

    @staticmethod
    def strides(x):  # (what ptr() uploads has no gaps)
        out, step = [], 1
        for s in reversed(x.shape):
            out.append(step)
            step *= s
        return tuple(reversed(out))

    @staticmethod
    def dense(x):
        return x

    @staticmethod
    def room(x):
        return x.nbytes

    def float_rows(self, x, what):
        return _float_rows(self, x, what)

    def int8_rows(self, x, what, scale, scale_what):
        return _int8_rows(self, x, what, scale, scale_what)

    def empty(self, shape, dtype):
        return DeviceArray(self.ctx, shape, dtype=dtype)

    def rows(self, rows, k, ld, lead):
        held = DeviceArray(self.ctx, (rows, ld), dtype="int8")
        return held, _Rows(held, k, lead)

    def scratch(self, nbytes):
        d = DeviceArray(self.ctx, (nbytes,), dtype="int8")
        self._keep.append(d)
        return d

    def done(self, result):
        self.ctx.synchronize()
        for d in self._keep:
            d.free()
        many = isinstance(result, tuple)
        out = []
        for r in result if many else (result,):
            if isinstance(r, _Rows):
                r = r.host() if self.host else r.device(self.ctx)
            elif self.host:
                d, r = r, r.to_host()
                d.free()
            out.append(r)
        return tuple(out) if many else out[0]


class _Rows:
    """8-bit rows as the kernel writes them (padded to 16 bytes), on their way to the caller's shape."""

    def __init__(self, held, k, lead):
        self.held, self.k, self.shape = held, k, (*lead, k)

    def host(self):
        a = self.held.to_host()[:, : self.k].reshape(self.shape)
        self.held.free()
        return np.ascontiguousarray(a)

    def device(self, ctx):
        if self.held.shape[1] == self.k:
            self.held.shape = self.shape
            return self.held
        return ctx.to_device(self.host(), dtype="int8")


_on_device: dict[int, _Tensors] = {}  # a device's default context and what the tensor library calls its types


def _space(first, ctx):
    lib = sys.modules.get("torch")
    if lib is not None and isinstance(first, lib.Tensor):
        index = first.get_device()
        if index < 0 or not first.is_cuda:
            raise ValueError("tensors must be on the GPU (host data: NumPy arrays)")
        if ctx is not None:
            if ctx.device != index:
                raise ValueError(f"tensors are on GPU {index}, the context on GPU {ctx.device}")
            return _Tensors(lib, index, ctx)
        sp = _on_device.get(index)
        if sp is None or sp.ctx is not _default_ctx.get(index):
            if index not in _default_ctx and lib.cuda.is_current_stream_capturing():
                raise RuntimeError("a device's first call creates its context, which cannot be done in a graph: call once before the capture")
            with lib.cuda.device(index):  # (the first use of a device creates its context, which makes that device the current one)
                sp = _on_device[index] = _Tensors(lib, index, default_context(index))
        return sp
    if isinstance(first, (np.ndarray, DeviceArray)):
        return _Arrays(first, ctx)
    raise ValueError(f"expected a tensor on the GPU, a DeviceArray or a NumPy array, not {type(first).__name__}")


def _call(ctx: Context, fn, *args):
    with ctx.lock:  # the message of a failure belongs to the call that failed
        rc = fn(ctx.handle, *args)
        if rc:
            ctx._check(rc)


def _kind(sp, x, what) -> int:
    kind = sp.kinds.get(x.dtype)
    return _kind_of(x.dtype, what) if kind is None else kind  # (which refuses it)


def _float_rows(sp, x, what):
    """(x as a matrix, leading shape, rows, k, row stride, column stride, type)"""
    x = sp.take(x, what)
    shape = tuple(x.shape)
    kind = _kind(sp, x, what)
    if len(shape) < 1:
        raise ValueError(f"{what} must have at least one axis")
    k, lead = shape[-1], shape[:-1]
    if k < 1:
        raise ValueError(f"{what} has rows of no elements")
    rows = math.prod(lead)
    if len(shape) == 2:
        rs, cs = sp.strides(x)
    elif isinstance(x, DeviceArray):
        rs, cs = k, 1
    else:
        x = x.reshape(rows, k)
        rs, cs = sp.strides(x)
    return x, lead, rows, k, rs, cs, kind


def _int8_rows(sp, x, what, scale, scale_what):
    """(matrix, its scales, leading shape, rows, k, row stride, whether the rows can be read where they are)

    They can when each starts at a multiple of 16 bytes and the bytes up to the next multiple behind its end exist."""
    x, scale = sp.take(x, what), sp.take(scale, scale_what)
    shape = tuple(x.shape)
    if len(shape) < 1 or x.dtype != sp.int8:
        raise ValueError(f"{what} must be a matrix of int8")
    k, lead = shape[-1], shape[:-1]
    if not 1 <= k <= MAX_K:
        raise ValueError(f"{what} has rows of {k} elements; 1 to {MAX_K} products are summed in 32 bits without overflow")
    if tuple(scale.shape) != lead or scale.dtype != sp.float32:
        raise ValueError(f"{scale_what} must be float32 of shape {lead}, not {scale.dtype} of shape {tuple(scale.shape)}")
    rows = math.prod(lead)
    flat = isinstance(x, DeviceArray)
    if not flat and len(shape) != 2:
        x = x.reshape(rows, k)
    st = (k, 1) if flat else sp.strides(x)
    if (k > 1 and st[1] != 1) or (rows > 1 and not k <= st[0] <= _MAX_LD):  # columns apart, rows that share memory, or further apart than the kernels count
        x = sp.dense(x)
        st = sp.strides(x)
    if k & 15:
        up = _up16(k)
        room = sp.room(x)
        ld = max(st[0], k) if rows > 1 else up if room >= up else k
        ready = ld >= up and room >= (rows - 1) * ld + up
    else:
        ld, ready = max(st[0], k) if rows > 1 else k, True
    return x, sp.dense(scale), lead, rows, k, ld, ready


def _bias(sp, bias, n, kind):
    if bias is None:
        return None, 0
    bias = sp.take(bias, "bias")
    code = _kind(sp, bias, "bias")
    if bias.shape != (n,) or code not in (0, kind):
        raise ValueError(f"bias must have shape ({n},) and be float32 or of the result's type, not {bias.dtype} of shape {tuple(bias.shape)}")
    return sp.dense(bias), code


def quantize_rows(x, ctx: Context | None = None):
    """(q, scale): the rows of ``x`` (its last axis) as 8-bit integers with one scale a row, ``x ~ scale[..., None] * q``.

    ``scale = max|x| / 127`` and ``q = 127 x / max|x|`` to the nearest integer, ties to even, decided as in exact arithmetic.  A row of zeros has
    scale 0; a row with a NaN or an infinity has that for its scale and zeros in ``q``.  The rows of a ``q`` that is a tensor start at
    multiples of 16 bytes (its last axis is dense, its rows may have gaps): that is how ``int8_matmul`` and ``int8_linear`` read them without a copy.  A
    ``DeviceArray`` has no gaps: where k is not a multiple of 16 its rows are put together by way of the host, and laid out again by each product."""
    sp = _space(x, ctx)
    x, lead, rows, k, rs, cs, kind = sp.float_rows(x, "x")
    stream = sp.begin()
    ld = _up16(k)
    held, q = sp.rows(rows, k, ld, lead)
    scale = sp.empty(lead, sp.float32)
    if rows:
        _call(sp.ctx, sp.ctx.lib.nls_quantize_rows, sp.ptr(x), kind, rows, k, rs, cs, sp.ptr(held), ld, sp.ptr(scale), stream)
    return sp.done((q, scale))


def int8_matmul(a, a_scale, b, b_scale, bias=None, dtype="float32", ctx: Context | None = None):
    """``y[..., j] = a_scale[...] * b_scale[j] * sum_k a[..., k] b[j, k] (+ bias[j])`` of ``dtype``.

    ``a`` (..., k) and ``b`` (n, k) int8, ``a_scale`` (...) and ``b_scale`` (n) float32, ``bias`` (n) float32 or of ``dtype``.  The sum is exact
    (k <= 131071), the rest is float32, rounded once.  Rows that do not start at multiples of 16 bytes are copied first (but for up to 16 rows of
    ``a``); ``quantize_rows`` lays them out so that they do."""
    sp = _space(a, ctx)
    kind = sp.named.get(dtype) if dtype.__hash__ is not None else None
    if kind is None:
        kind = _kind_of(dtype, "dtype")
    if kind >= len(sp.types):
        raise ValueError("dtype: NumPy arrays and DeviceArrays have no bfloat16")
    a, a_scale, lead, m, k, lda, a_ready = sp.int8_rows(a, "a", a_scale, "a_scale")
    b, b_scale, b_lead, n, kb, ldb, b_ready = sp.int8_rows(b, "b", b_scale, "b_scale")
    if len(b_lead) != 1 or kb != k:
        raise ValueError(f"b must be a matrix with rows of {k} elements, not of shape {(*b_lead, kb)}")
    bias, bias_kind = _bias(sp, bias, n, kind)
    stream = sp.begin()
    y = sp.empty((*lead, n), sp.types[kind])
    if m and n:
        lib = sp.ctx.lib
        pa, pb = sp.ptr(a), sp.ptr(b)
        flags = (_A_PADDED if a_ready else 0) | (_B_PADDED if b_ready else 0)
        nbytes, ws = 0, None
        if not (a_ready and b_ready) or (pa | pb | lda | ldb) & 15:  # rows that have to be laid out again
            need = C.c_size_t()
            lib.nls_int8_matmul_workspace(pa, lda, pb, ldb, m, n, k, flags, need)
            nbytes = need.value
            ws = sp.scratch(nbytes) if nbytes else None
        _call(
            sp.ctx, lib.nls_int8_matmul, pa, lda, sp.ptr(a_scale), pb, ldb, sp.ptr(b_scale), None if bias is None else sp.ptr(bias), bias_kind,
            m, n, k, sp.ptr(y), kind, flags, None if ws is None else sp.ptr(ws), nbytes, stream,
        )  # fmt: skip
    return sp.done(y)


def int8_linear(x, b, b_scale, bias=None, ctx: Context | None = None):
    """``int8_matmul(*quantize_rows(x), b, b_scale, bias, dtype=x.dtype)`` in one call: ``x`` (..., k) in 16 or 32 bits against rows held in 8."""
    sp = _space(x, ctx)
    x, lead, m, k, rs, cs, kind = sp.float_rows(x, "x")
    b, b_scale, b_lead, n, kb, ldb, b_ready = sp.int8_rows(b, "b", b_scale, "b_scale")
    if len(b_lead) != 1 or kb != k:
        raise ValueError(f"b must be a matrix with rows of {k} elements, not of shape {(*b_lead, kb)}")
    bias, bias_kind = _bias(sp, bias, n, kind)
    stream = sp.begin()
    y = sp.empty((*lead, n), sp.types[kind])
    if m and n:
        lib = sp.ctx.lib
        pb = sp.ptr(b)
        flags = _B_PADDED if b_ready else 0
        if m > 4 and b_ready and not (pb | ldb) & 15:  # b is read where it is: room for the rows of x in 8 bits and their scales
            nbytes = (m * _up16(k) + 255 & -256) + (4 * m + 255 & -256)
        else:
            need = C.c_size_t()
            lib.nls_int8_linear_workspace(pb, ldb, m, n, k, flags, need)
            nbytes = need.value
        ws = sp.scratch(nbytes) if nbytes else None
        _call(
            sp.ctx, lib.nls_int8_linear, sp.ptr(x), kind, rs, cs, pb, ldb, sp.ptr(b_scale), None if bias is None else sp.ptr(bias), bias_kind, m, n, k,
            sp.ptr(y), flags, None if ws is None else sp.ptr(ws), nbytes, stream,
        )  # fmt: skip
    return sp.done(y)


def orthogonalize(g, steps: int = 5, coefficients=NEWTON_SCHULZ, eps: float = 1e-7, ctx: Context | None = None):
    """Newton-Schulz orthogonalisation of a matrix, or of every matrix of a batch (the last two axes), in the type it comes in.

    ``X = G / (|G|_F + eps)``, then ``steps`` times ``X <- a X + (b A + c A A) X`` with ``A = X X^T`` taken on the shorter side.  ``coefficients``: one
    (a, b, c) for all steps or one for each.  Every singular value s of X goes through the polynomials a s + b s^3 + c s^5 while the singular vectors
    stay: with coefficients that lead to 1 the result is the orthogonal factor of the polar decomposition (what a QR of a Gaussian matrix gives
    ``orf_frequencies`` up to rotation of the draw), with the default ones the near-orthogonal update of a training step.

    Products and sums carry 22 bits or more, whatever the type of ``g``: the error before the result's own rounding is that of float32 products
    (16-bit matrices of up to 128 rows: and less than a quarter of that rounding).  At most 32 steps, 2^20 rows and columns, and 65535 matrices."""
    sp = _space(g, ctx)
    g = sp.take(g, "g")
    shape = tuple(g.shape)
    if len(shape) < 2:
        raise ValueError("g must be a matrix or a batch of matrices")
    kind = _kind(sp, g, "g")
    if isinstance(steps, bool) or int(steps) != steps or not 1 <= steps <= 32:
        raise ValueError("steps must be a whole number from 1 to 32")
    steps = int(steps)
    try:
        flat = [float(v) for v in coefficients] if len(coefficients) == 3 and not hasattr(coefficients[0], "__len__") else None
        if flat is None:
            flat = [float(v) for row in coefficients for v in row] if len(coefficients) == steps and all(len(row) == 3 for row in coefficients) else []
        else:
            flat *= steps
    except TypeError:
        flat = []
    if len(flat) != 3 * steps or not all(map(math.isfinite, flat)):
        raise ValueError(f"coefficients must be three finite numbers, or three for each of the {steps} steps")
    eps = float(eps)
    if not 0.0 <= eps < 1e30:
        raise ValueError("eps must be a number >= 0")
    table = (C.c_double * (3 * steps))(*flat)
    m, n = shape[-2:]
    batch = math.prod(shape[:-2])
    if max(m, n) > 1 << 20 or batch > 65535:  # (before room is made for the result and its workspace)
        raise ValueError(f"g of shape {shape}: at most 2^20 rows and columns and 65535 matrices")
    if isinstance(g, DeviceArray):
        st = (m * n, n, 1)
    elif len(shape) == 2:
        st = (0, *sp.strides(g))
    else:
        if len(shape) != 3:
            g = g.reshape(batch, m, n)
        st = sp.strides(g)
    stream = sp.begin()
    lib = sp.ctx.lib
    out = sp.empty(shape, sp.types[kind])
    need = C.c_size_t()
    empty = not (batch and m and n)
    lib.nls_orthogonalize_workspace(batch, m, n, st[1], st[2], need)
    ws = None if empty or not need.value else sp.scratch(need.value)
    _call(
        sp.ctx, lib.nls_orthogonalize, None if empty else sp.ptr(g), kind, batch, m, n, *st, table, steps, eps, sp.ptr(out),
        None if ws is None else sp.ptr(ws), need.value, stream,
    )  # fmt: skip
    return sp.done(out)
