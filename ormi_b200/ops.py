"""Transformer-block operators on device buffers (the C ABI's ormi_b200_rmsnorm, ormi_b200_attention, ormi_b200_adamw).

They stand beside the graph's matmuls, softmax and layernorm: RMS norm with the residual's addition, attention with capped
scores, distance bias, document and prefix masks, and AdamW over many tensors, each with what training and serving need
(backward passes, 8-bit outputs and states, few queries over a long cache).

Every function queues its work on the device's compute stream, writes into buffers the caller provides and returns at once.
A buffer is any of

* an :class:`Array` (``empty``, ``upload``), :class:`ormi_b200.graph.Buffer` or a realized :class:`ormi_b200.graph.Node`;
* an object with ``data_ptr()``, ``shape``, ``stride()`` and ``dtype``, such as a torch tensor on the device's GPU.  Other
  libraries' streams are not known here: order them against ``Device.stream`` with events (or a synchronize);
* a view made by :func:`view` from a plain address.

What is asked of shapes, types and strides, and the formulas, stand in include/ormi_b200.h; a call that does not meet them
raises ``BackendError`` before anything is queued.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Sequence

import numpy as np

from . import graph as G
from ._lib import lib, check

F32, BF16, E4M3, I32 = 0, 1, 2, 3
_SIZES = {F32: 4, BF16: 2, E4M3: 1, I32: 4}
_NAMES = {"f32": F32, "bf16": BF16, "e4m3": E4M3, "i32": I32}
_TYPES = {"float32": F32, "bfloat16": BF16, "float8_e4m3fn": E4M3, "int32": I32}
_TYPES.update({"torch." + k: v for k, v in list(_TYPES.items())})
_by_dtype: dict = {}                       # dtype object -> code, filled as types are met

_VIEW = struct.Struct("=Qii8q")            # ormi_b200_view
_VIEW_PACK = _VIEW.pack
_tensor_types: set = set()                 # types with the tensor protocol, filled as they are met
_ABSENT = bytes(_VIEW.size)
_ZEROS = (0, 0, 0, 0)


class View:
    """An address with a type, a shape and strides in elements."""
    __slots__ = ("ptr", "dtype", "shape", "strides")

    def __init__(self, ptr: int, shape: Sequence[int], dtype: str = "f32", strides: Sequence[int] | None = None):
        if dtype not in _NAMES:
            raise ValueError(f"unknown type {dtype!r}: f32, bf16, e4m3 or i32")
        self.ptr, self.dtype, self.shape = ptr, _NAMES[dtype], tuple(int(s) for s in shape)
        self.strides = tuple(G.calc_contiguous_strides(self.shape)) if strides is None else tuple(int(s) for s in strides)
        if len(self.strides) != len(self.shape):
            raise ValueError("one stride for each dimension is wanted")


def view(ptr: int, shape, dtype: str = "f32", strides=None) -> View:
    return View(ptr, shape, dtype, strides)


class Array(View):
    """A contiguous device array of one of the operators' types, from the device's pool; it goes back with the object."""
    __slots__ = ("dev", "nbytes", "__weakref__")

    def __init__(self, dev, shape, dtype: str = "f32"):
        super().__init__(0, shape, dtype)
        self.dev, self.nbytes = dev, max(4, G.numel(self.shape) * _SIZES[self.dtype])
        self.ptr = dev.alloc(self.nbytes)

    def __del__(self):
        ptr, self.ptr = getattr(self, "ptr", 0), 0
        if ptr:
            try:
                self.dev.free(ptr, self.nbytes)
            except Exception:
                pass

    def numpy(self) -> np.ndarray:
        """The values on the host, as float32 (int32 for i32); waits for the work queued so far."""
        raw = np.empty(self.shape, dtype={F32: np.float32, I32: np.int32, BF16: np.uint16, E4M3: np.uint8}[self.dtype])
        if raw.nbytes:
            self.dev.d2h(raw, self.ptr)
        if self.dtype == BF16:
            return (raw.astype(np.uint32) << 16).view(np.float32)
        return _E4M3_VALUES[raw] if self.dtype == E4M3 else raw


def _e4m3_values() -> np.ndarray:
    code = np.arange(256)
    e, m = code >> 3 & 15, code & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))
    v[(code & 127) == 127] = np.nan
    return np.where(code & 128, -v, v).astype(np.float32)


_E4M3_VALUES = _e4m3_values()


def empty(dev, shape, dtype: str = "f32") -> Array:
    return Array(dev, shape, dtype)


def zeros(dev, shape, dtype: str = "f32") -> Array:
    a = Array(dev, shape, dtype)
    check(lib.ormi_b200_memset(dev.handle, ctypes.c_void_p(a.ptr), 0, a.nbytes))
    return a


def upload(dev, array, dtype: str = "f32") -> Array:
    """A device array holding ``array``: f32, i32, or rounded to the nearest bf16."""
    a = np.asarray(array, dtype=np.int32 if dtype == "i32" else np.float32)
    out = Array(dev, a.shape, dtype)
    if dtype == "bf16":
        u = np.ascontiguousarray(a).view(np.uint32).astype(np.uint64)
        u = np.where(np.isnan(a), 0x7fc00000, u + 0x7fff + (u >> 16 & 1)).astype(np.uint64)
        a = (u >> 16).astype(np.uint16)
    elif dtype == "e4m3":
        raise ValueError("upload takes f32, bf16 or i32")
    a = np.ascontiguousarray(a)
    if a.nbytes:
        dev.h2d(out.ptr, a)
    return out


def _same_gpu(owner, dev_index: int):
    index = getattr(owner, "index", None)
    if isinstance(index, int) and index != dev_index:
        raise ValueError(f"a buffer on cuda:{index} where the device is cuda:{dev_index}")


def _pack(x, dev_index: int) -> bytes:
    """``x`` as an ormi_b200_view."""
    if x is None:
        return _ABSENT
    kind = type(x)
    if kind in _tensor_types:                  # the common case first: a call's arguments cost more time than its launch
        code = _by_dtype.get(x.dtype)
        if code is not None and x.get_device() == dev_index:
            shape, strides = x.shape, x.stride()
            n = len(shape)
            if n == 2:
                return _VIEW_PACK(x.data_ptr(), code, 2, shape[0], shape[1], 0, 0, strides[0], strides[1], 0, 0)
            if n == 4:
                return _VIEW_PACK(x.data_ptr(), code, 4, *shape, *strides)
            if n == 1:
                return _VIEW_PACK(x.data_ptr(), code, 1, shape[0], 0, 0, 0, strides[0], 0, 0, 0)
    if isinstance(x, View):
        ptr, code, shape, strides = x.ptr, x.dtype, x.shape, x.strides
        _same_gpu(x.dev if isinstance(x, Array) else None, dev_index)
    elif hasattr(x, "data_ptr"):
        dt = x.dtype
        code = _by_dtype.get(dt)
        if code is None:
            code = _TYPES.get(str(dt))
            if code is None:
                raise TypeError(f"{dt} is not a type of these operators (float32, bfloat16, float8_e4m3fn, int32)")
            _by_dtype[dt] = code
        _tensor_types.add(kind)
        if x.get_device() != dev_index:
            raise ValueError(f"a tensor on {x.device} where the device is cuda:{dev_index}")
        ptr, shape, strides = x.data_ptr(), x.shape, x.stride()
    elif isinstance(x, (G.Node, G.Buffer)):
        data = x.data if isinstance(x, G.Node) else x
        if data is None or data.dev_ptr is None:
            raise ValueError("a graph node that is not realized on the device")
        _same_gpu(getattr(data._release, "__self__", None), dev_index)      # the device whose pool the block goes back to
        ptr, shape = data.dev_ptr, tuple(x.shape)
        strides = tuple(x.strides) if isinstance(x, G.Node) else G.calc_contiguous_strides(shape)
        code = BF16 if isinstance(x, G.Node) and x.bf16 else F32
        if isinstance(x, G.Node) and x.bf16:
            strides = G.calc_contiguous_strides(shape)
    else:
        raise TypeError(f"{type(x).__name__} is not a device buffer")
    n = len(shape)
    if n > 4:
        raise ValueError(f"{n} dimensions: at most 4 are taken")
    if n == 0:
        return _VIEW.pack(ptr, code, 1, 1, 0, 0, 0, 1, 0, 0, 0)
    pad = _ZEROS[n:]
    return _VIEW.pack(ptr, code, n, *shape, *pad, *strides, *pad)


# ------------------------------------------------------------------------------------------------ RMS norm

_NORM_TAIL = struct.Struct("=if")


def rmsnorm(dev, x, weight, out, *, residual=None, residual_out=None, rstd=None, scales=None, group: int = 0, eps: float = 1e-6):
    """``s = x + residual; out = s / sqrt(mean(s^2) + eps) * weight`` over the last dimension.

    ``residual_out`` receives s (the residual stream), ``rstd`` one value per row for the backward pass.  With an e4m3
    ``out``, ``scales`` receives one scale per row (``group=0``) or per 128 columns (``group=128``)."""
    i = dev.index
    check(lib.ormi_b200_rmsnorm(dev.handle, _pack(x, i) + _pack(residual, i) + _pack(weight, i) + _pack(out, i) + _pack(residual_out, i) +
                                _pack(rstd, i) + _pack(scales, i) + _NORM_TAIL.pack(group, eps)))


def rmsnorm_backward(dev, dout, s, weight, rstd, dx, dweight=None, *, dresidual=None):
    """Gradients of :func:`rmsnorm`: ``dx`` (of x and of residual alike, with ``dresidual`` added) and ``dweight``."""
    i = dev.index
    check(lib.ormi_b200_rmsnorm_backward(dev.handle, _pack(dout, i) + _pack(s, i) + _pack(weight, i) + _pack(rstd, i) + _pack(dresidual, i) +
                                         _pack(dx, i) + _pack(dweight, i)))


# ------------------------------------------------------------------------------------------------ attention

_ATTN_TAIL = struct.Struct("=ffii")


def _attention_args(dev, q, k, v, out, lse, scale, causal, cap, slopes, q_docs, k_docs, prefix, key_len, q_start) -> bytes:
    i = dev.index
    if scale is None:
        scale = float(q.shape[-1]) ** -0.5 if q.shape[-1] else 1.0
    return (_pack(q, i) + _pack(k, i) + _pack(v, i) + _pack(out, i) + _pack(lse, i) + _pack(slopes, i) + _pack(q_docs, i) + _pack(k_docs, i) +
            _pack(prefix, i) + _pack(key_len, i) + _pack(q_start, i) + _ATTN_TAIL.pack(scale, cap, 1 if causal else 0, 0))


def attention(dev, q, k, v, out, lse=None, *, scale: float | None = None, causal: bool = False, cap: float = 0.0, slopes=None,
              q_docs=None, k_docs=None, prefix=None, key_len=None, q_start=None):
    """Softmax attention over ``[batch, length, heads, head_dim]`` buffers; ``scale`` defaults to ``head_dim ** -0.5``.

    ``cap``: scores become ``cap * tanh(score / cap)``.  ``slopes[head] * distance`` is taken off a score.  ``q_docs`` /
    ``k_docs``: a query sees the keys of its own document.  ``causal``: a query sees the keys up to its own position and
    the first ``prefix[batch]`` ones.  ``key_len``: valid keys of each batch row.  ``q_start``: position of the first query
    of each batch row (the default puts the queries at the end of the keys).  ``lse`` is what the backward pass needs."""
    check(lib.ormi_b200_attention(dev.handle, _attention_args(dev, q, k, v, out, lse, scale, causal, cap, slopes, q_docs, k_docs, prefix, key_len, q_start)))


def attention_backward(dev, dout, q, k, v, out, lse, dq, dk, dv, *, scale: float | None = None, causal: bool = False, cap: float = 0.0,
                       slopes=None, q_docs=None, k_docs=None, prefix=None, key_len=None, q_start=None):
    """Gradients of :func:`attention` from its own arguments and results."""
    i = dev.index
    check(lib.ormi_b200_attention_backward(dev.handle, _attention_args(dev, q, k, v, out, lse, scale, causal, cap, slopes, q_docs, k_docs, prefix, key_len, q_start) +
                                           _pack(dout, i) + _pack(dq, i) + _pack(dk, i) + _pack(dv, i)))


# ------------------------------------------------------------------------------------------------ AdamW

_ADAM_TENSOR = struct.Struct("=7Qqif")
_ADAM_CONFIG = struct.Struct("=4dqQQQIi")
_FLAT = struct.Struct("=Qii8q")


class AdamW:
    """AdamW over a list of tensors, updated in place by one launch (``ormi_b200_adamw``).

    ``params``: f32.  ``grads``: f32 or bf16.  ``m`` and ``v``: f32 states, or e4m3 codes with ``m_scales`` / ``v_scales``
    (one f32 per 128 elements).  ``copies``: bf16 buffers that receive the rounded parameters.  ``weight_decay``: one number
    or one per tensor.  The buffers are looked at once, here; the object keeps them alive.  Tensors have to be contiguous.
    """

    def __init__(self, dev, params, grads, m, v, *, m_scales=None, v_scales=None, copies=None, weight_decay=0.0,
                 betas=(0.9, 0.999), eps: float = 1e-8, seed: int = 0):
        n = len(params)
        lists = [list(params), list(grads), list(m), list(v)] + [list(x) if x is not None else [None] * n for x in (m_scales, v_scales, copies)]
        decay = [float(weight_decay)] * n if not hasattr(weight_decay, "__len__") else [float(w) for w in weight_decay]
        if any(len(x) != n for x in lists) or len(decay) != n:
            raise ValueError("every list names one buffer for each parameter")
        self.state_bits = 32 if m_scales is None and v_scales is None else 8
        state = F32 if self.state_bits == 32 else E4M3
        wanted = [("param", (F32,)), ("grad", (F32, BF16)), ("m", (state,)), ("v", (state,)), ("m_scales", (F32,)), ("v_scales", (F32,)), ("copy", (BF16,))]
        blob = []
        for i in range(n):
            ptrs, codes, count = [], [], None
            for (name, types), x in zip(wanted, (column[i] for column in lists)):
                ptr, code, ndim, *dims = _FLAT.unpack(_pack(x, dev.index))
                shape, strides = dims[:ndim], dims[4:4 + ndim]
                if x is not None:
                    size = G.numel(shape)
                    if code not in types:
                        raise ValueError(f"tensor {i}: {name} has another type than is wanted")
                    if any(a != 1 and b != c for a, b, c in zip(shape, strides, G.calc_contiguous_strides(shape))) and size:
                        raise ValueError(f"tensor {i}: {name} is not contiguous")
                    if count is None:
                        count = size
                    if size != (-(-count // 128) if name.endswith("scales") else count):
                        raise ValueError(f"tensor {i}: {name} has {size} elements")
                ptrs.append(ptr)
                codes.append(code)
            blob.append(_ADAM_TENSOR.pack(*ptrs, count, codes[1], decay[i]))
        self.dev, self.n, self.blob = dev, n, b"".join(blob)
        self._grads = [(_FLAT.unpack(_pack(g, dev.index))[1], G.numel(g.shape)) for g in lists[1]]
        self.betas, self.eps, self.seed = betas, float(eps), int(seed)
        self.steps_done = 0
        self._keepalive = lists

    def step(self, lr: float = 0.0, *, step: int | None = None, grads=None, grad_scale=None, device_lr=None, device_step=None):
        """One update.  ``step`` counts from 1 and defaults to one more than the last one.  ``grads``: this step's gradients
        where they are not the buffers of the constructor (same types and sizes).  ``grad_scale`` and ``device_lr`` (replaces
        ``lr``): f32 device scalars.  ``device_step``: address of a 64-bit device counter of the steps done,
        which the call reads and increments, for steps that are captured and replayed."""
        blob = self.blob
        if grads is not None:
            if len(grads) != self.n:
                raise ValueError("every list names one buffer for each parameter")
            blob = bytearray(blob)
            for i, g in enumerate(grads):
                ptr, code, ndim, *dims = _FLAT.unpack(_pack(g, self.dev.index))
                shape = dims[:ndim]
                if (code, G.numel(shape)) != self._grads[i] or any(a != 1 and b != c for a, b, c in zip(shape, dims[4:4 + ndim], G.calc_contiguous_strides(shape))):
                    raise ValueError(f"tensor {i}: the gradient has another type or size, or is not contiguous")
                struct.pack_into("=Q", blob, i * _ADAM_TENSOR.size + 8, ptr)
            blob = bytes(blob)
        count = self.steps_done
        if device_step is None:
            count = count + 1 if step is None else int(step)
        config = _ADAM_CONFIG.pack(lr, self.betas[0], self.betas[1], self.eps, count, _scalar(device_step, 8, self.dev), _scalar(device_lr, 4, self.dev),
                                   _scalar(grad_scale, 4, self.dev), self.seed & 0xffffffff, self.state_bits)
        check(lib.ormi_b200_adamw(self.dev.handle, blob, self.n, config))
        self.steps_done = count                    # a refused call has not counted


def _scalar(x, size: int, dev) -> int:
    """Address of a device scalar: an int, or a buffer of one element (two 32-bit ones for a 64-bit counter)."""
    if x is None or isinstance(x, int):
        return x or 0
    if hasattr(x, "data_ptr"):
        if x.get_device() != dev.index or x.numel() * x.element_size() != size:
            raise ValueError(f"a {size}-byte scalar on cuda:{dev.index} is wanted")
        if size == 4 and str(x.dtype) != "torch.float32" or size == 8 and str(x.dtype) != "torch.int64":
            raise ValueError("the scalar has another type than is wanted (float32, or int64 for the step counter)")
        return x.data_ptr()
    ptr, code, ndim, *dims = _FLAT.unpack(_pack(x, dev.index))
    if G.numel(dims[:ndim]) * _SIZES[code] != size or (size == 4 and code != F32):
        raise ValueError(f"a {size}-byte scalar is wanted")
    return ptr
