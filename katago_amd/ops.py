"""Operators of the device library on the caller's tensors (include/katago_hip.h):
a matrix product with bias, activation and residual (``linear``), rotary
positions with several axes (``rope_axes``), attention to an encoder's states
(``cross_attention``), rows in 8 bits (``quantize_rows``) and the matrix product of
such rows (``linear_int8``), group norm with an activation, channels last
(``group_norm``), and its gradient (``group_norm_backward``).

Tensors are torch tensors, or ``DeviceTensor`` views of device memory: anything
with ``data_ptr()``, ``stride()``, ``shape``, ``dtype`` and ``get_device()``. Calls are
asynchronous on ``stream``: a hipStream_t as an int, 0 for the null stream; None for
the stream that torch is on for torch tensors, and the null stream for others. The
caller keeps the tensors alive until they have run. Nothing here records gradients:
tensors that require them are taken under ``torch.no_grad()`` only, as in the methods
of a torch.autograd.Function that calls ``group_norm`` and ``group_norm_backward``, and
tensors with tangents of forward mode are refused. Every call returns its output tensor. Arguments that do not fit raise ``StringError``.
"""
from __future__ import annotations

import ctypes
import sys

from .nn import StringError, hip_check, hip_library

FP32, FP16, BF16 = 0, 1, 2
ACTIVATIONS = {"identity": 0, "relu": 1, "mish": 2, "silu": 3, "gelu": 20}
ROPE_LAYOUTS = {"interleaved": 0, "halves": 1}
_INVALID = 1  # KGH_ERR_INVALID_ARGUMENT
_MOST = 1 << 30  # of an axis; the library counts some in 32 bits

_i32, _i64, _ptr = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


class _LinearParams(ctypes.Structure):
    """kgh_linear_params."""
    _fields_ = [("dtype", _i32), ("activation", _i32), ("rows", _i64), ("in_channels", _i32), ("out_channels", _i32),
                ("x", _ptr), ("x_stride", _i64), ("weights", _ptr), ("weights_stride", _i64), ("bias", _ptr),
                ("residual", _ptr), ("residual_stride", _i64), ("out", _ptr), ("out_stride", _i64),
                ("workspace", _ptr), ("workspace_bytes", ctypes.c_uint64)]


class _RopeParams(ctypes.Structure):
    """kgh_rope_params."""
    _fields_ = [("dtype", _i32), ("layout", _i32), ("inverse", _i32), ("axes", _i32), ("tokens", _i64), ("heads", _i32),
                ("head_dim", _i32), ("pairs", _i32), ("tables", _i32), ("x", _ptr), ("x_token_stride", _i64),
                ("x_head_stride", _i64), ("positions", _ptr), ("positions_stride", _i64), ("freqs", _ptr), ("out", _ptr),
                ("out_token_stride", _i64), ("out_head_stride", _i64)]


class _AttentionParams(ctypes.Structure):
    """kgh_attention_params."""
    _fields_ = [("dtype", _i32), ("batch", _i32), ("q_len", _i32), ("k_len", _i32), ("heads", _i32), ("kv_heads", _i32),
                ("q_head_dim", _i32), ("v_head_dim", _i32), ("scale", ctypes.c_float), ("precise", _i32),
                ("q", _ptr), ("q_strides", _i64 * 3), ("k", _ptr), ("k_strides", _i64 * 3), ("v", _ptr), ("v_strides", _i64 * 3),
                ("out", _ptr), ("out_strides", _i64 * 3), ("key_lengths", _ptr), ("key_mask", _ptr), ("key_mask_stride", _i64),
                ("workspace", _ptr), ("workspace_bytes", ctypes.c_uint64)]


class _QuantizeParams(ctypes.Structure):
    """kgh_quantize_params."""
    _fields_ = [("dtype", _i32), ("channels", _i32), ("rows", _i64), ("x", _ptr), ("x_stride", _i64), ("out", _ptr), ("out_stride", _i64),
                ("scales", _ptr)]


class _LinearInt8Params(ctypes.Structure):
    """kgh_linear_int8_params."""
    _fields_ = [("dtype", _i32), ("activation", _i32), ("rows", _i64), ("in_channels", _i32), ("out_channels", _i32),
                ("x", _ptr), ("x_stride", _i64), ("x_scales", _ptr), ("weights", _ptr), ("weights_stride", _i64), ("weight_scales", _ptr),
                ("bias", _ptr), ("residual", _ptr), ("residual_stride", _i64), ("out", _ptr), ("out_stride", _i64),
                ("workspace", _ptr), ("workspace_bytes", ctypes.c_uint64)]


class _GroupNormParams(ctypes.Structure):
    """kgh_group_norm_params."""
    _fields_ = [("dtype", _i32), ("activation", _i32), ("batch", _i32), ("positions", _i32), ("channels", _i32), ("groups", _i32),
                ("eps", ctypes.c_float), ("x", _ptr), ("x_batch_stride", _i64), ("x_position_stride", _i64), ("weight", _ptr), ("bias", _ptr), ("lengths", _ptr), ("mask", _ptr),
                ("mask_stride", _i64), ("out", _ptr), ("out_batch_stride", _i64), ("out_position_stride", _i64), ("out_scales", _ptr), ("statistics", _ptr),
                ("workspace", _ptr), ("workspace_bytes", ctypes.c_uint64)]


class _GroupNormBackwardParams(ctypes.Structure):
    """kgh_group_norm_backward_params."""
    _fields_ = [("dtype", _i32), ("activation", _i32), ("batch", _i32), ("positions", _i32), ("channels", _i32), ("groups", _i32),
                ("x", _ptr), ("x_batch_stride", _i64), ("x_position_stride", _i64), ("grad_out", _ptr), ("grad_out_batch_stride", _i64),
                ("grad_out_position_stride", _i64), ("statistics", _ptr), ("weight", _ptr), ("bias", _ptr), ("lengths", _ptr), ("mask", _ptr),
                ("mask_stride", _i64), ("grad_x", _ptr), ("grad_x_batch_stride", _i64), ("grad_x_position_stride", _i64), ("grad_weight", _ptr), ("grad_bias", _ptr), ("workspace", _ptr), ("workspace_bytes", ctypes.c_uint64)]


_CALLS = {"kgh_linear": _LinearParams, "kgh_rope_axes": _RopeParams, "kgh_cross_attention": _AttentionParams, "kgh_quantize_rows": _QuantizeParams,
          "kgh_linear_int8": _LinearInt8Params, "kgh_group_norm": _GroupNormParams, "kgh_group_norm_backward": _GroupNormBackwardParams}
_lib = None


def _library() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        lib = hip_library()
        for name, params in _CALLS.items():
            getattr(lib, name).argtypes = [_i32, ctypes.POINTER(params), _ptr]
            if hasattr(lib, name + "_workspace"):
                getattr(lib, name + "_workspace").argtypes = [_i32, ctypes.POINTER(params), ctypes.POINTER(ctypes.c_uint64)]
        _lib = lib
    return _lib


class DeviceTensor:
    """A view of device memory for callers without torch: a pointer (an int or
    ctypes.c_void_p, for instance ``DeviceBuffer.ptr``), a shape, the name of a
    type ("float32", "float16", "bfloat16", "int32", "int8", "uint8", "bool") and
    strides in elements (None: contiguous)."""

    def __init__(self, ptr, shape, dtype: str, strides=None, device: int = 0):
        self._ptr = ptr.value or 0 if isinstance(ptr, _ptr) else int(ptr)
        self.shape = tuple(shape)
        if strides is None:
            strides, n = [], 1
            for s in reversed(self.shape):
                strides.insert(0, n)
                n *= max(s, 1)
        self._strides = tuple(strides)
        self.dtype = dtype
        self._device = device

    def data_ptr(self) -> int:
        return self._ptr

    def stride(self):
        return self._strides

    def get_device(self) -> int:
        return self._device


def _invalid(message: str):
    raise StringError(message, _INVALID)


_CODES = {"float32": FP32, "float16": FP16, "bfloat16": BF16, "int32": "int32", "int8": "int8", "uint8": "uint8", "bool": "bool"}
_BYTES = {"bool": 1, "uint8": 1, "int8": 1, "float16": 2, "bfloat16": 2, "int16": 2, "uint16": 2, "int32": 4, "uint32": 4, "float32": 4,
          "int64": 8, "uint64": 8, "float64": 8}  # of a workspace's elements
_codes = dict(_CODES)  # the same by the tensors' own type objects
_bytes = {}
_types = {code: name for name, code in _CODES.items()}  # the type object met last of each


def _code(op, name, t):
    """A tensor's type: FP32, FP16, BF16 or the name of another one."""
    try:
        return _codes[t.dtype]
    except KeyError:
        pass
    code = _CODES.get(str(t.dtype).rsplit(".", 1)[-1])
    if code is None:
        _invalid(f"{op}: {name} is of type {t.dtype}")
    _codes[t.dtype] = code
    _types[code] = t.dtype
    return code


def _look(op, name, t, ndim, dtype, device):
    """Checks a tensor's axes, type (by a type object) and device; returns its
    strides."""
    strides = t.stride()
    if len(strides) != ndim or t.dtype != dtype or t.get_device() != device or strides[-1] != 1:
        _look_again(op, name, t, strides, ndim, dtype, device)
    return strides


def _look_again(op, name, t, strides, ndim, dtype, device):
    """What does not fit, if anything does not."""
    if len(strides) != ndim:
        _invalid(f"{op}: {name} has {len(strides)} axes, not {ndim}")
    if strides[-1] != 1 and t.shape[-1] > 1:
        _invalid(f"{op}: the last axis of {name} is not contiguous")
    if _code(op, name, t) != _codes[dtype]:
        _invalid(f"{op}: {name} is of type {t.dtype}")
    if t.get_device() != device:
        _invalid(f"{op}: {name} is not on the same device as the first tensor")


def _first(op, name, t):
    """The type and device index that the call goes by."""
    device = t.get_device()
    if device < 0:
        _invalid(f"{op}: {name} is not on a GPU")
    code = _codes.get(t.dtype)
    if code is None:
        code = _code(op, name, t)
    if code not in (FP32, FP16, BF16):
        _invalid(f"{op}: {name} is of type {t.dtype}")
    return code, device


def _stream(t, device):
    """The stream of a call that names none: torch's for its tensors, which the null
    stream does not wait for, nor it for the null stream."""
    torch = sys.modules.get("torch")
    if torch is not None and isinstance(t, torch.Tensor):
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the same without an object around it
        return raw(device) if raw is not None else torch.cuda.current_stream(device).cuda_stream
    return None


def _no_gradients(op, *tensors):
    """Refuses tensors that a result's gradients would be wanted of."""
    torch = sys.modules.get("torch")
    for t in tensors:
        if t is not None and getattr(t, "requires_grad", False) and torch.is_grad_enabled():
            _invalid(f"{op}: a tensor requires gradients, and the result would have none (torch.no_grad() takes it)")
    if torch is not None and getattr(torch.autograd.forward_ad, "_current_level", 0) >= 0:
        _no_tangents(op, torch, tensors)


def _no_tangents(op, torch, tensors):
    """The same of gradients that go forward, within a dual level (but not in a
    torch.autograd.Function's forward, whose jvp is what counts)."""
    if torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
                _invalid(f"{op}: a tensor has a tangent, and the result would have none")


def _sizes(op, *sizes):
    if max(sizes) > _MOST:
        _invalid(f"{op}: an axis is longer than {_MOST}")


def _shape(op, name, t, *want):
    if t.shape != want and tuple(t.shape) != want:
        _invalid(f"{op}: {name} has shape {tuple(t.shape)}, not {want}")


def _workspace(op, workspace, device):
    """Pointer and bytes of a workspace: a contiguous tensor of integers or numbers."""
    if workspace is None:
        return None, 0
    if workspace.get_device() != device:
        _invalid(f"{op}: the workspace is not on the same device as the first tensor")
    strides = workspace.stride()
    if strides == (1,):
        n = workspace.shape[0]
    else:
        n = 1
        for size, stride in zip(reversed(workspace.shape), reversed(strides)):
            if stride != n and size > 1:
                _invalid(f"{op}: the workspace is not contiguous")
            n *= size
    size = _bytes.get(workspace.dtype)
    if size is None:
        size = _bytes[workspace.dtype] = _BYTES.get(str(workspace.dtype).rsplit(".", 1)[-1], 0)
    if size == 0:
        _invalid(f"{op}: the workspace is of type {workspace.dtype}")
    return workspace.data_ptr(), n * size


def _linear_params(x, weights, out, bias, activation, residual, workspace):
    code, device = _first("linear", "x", x)
    dtype = x.dtype
    xs = _look("linear", "x", x, 2, dtype, device)
    ws = _look("linear", "weights", weights, 2, dtype, device)
    rows, in_c = x.shape
    out_c, w_in = weights.shape
    if w_in != in_c:
        _invalid(f"linear: weights have {w_in} input channels, x has {in_c}")
    _sizes("linear", rows, in_c, out_c)
    act = ACTIVATIONS.get(activation or "identity")
    if act is None:
        _invalid(f"linear: unknown activation {activation!r}")
    op = os = bp = None
    rs = space = (None, 0)
    if out is not None:
        os = _look("linear", "out", out, 2, dtype, device)[0]
        _shape("linear", "out", out, rows, out_c)
        op = out.data_ptr()
    if bias is not None:
        _look("linear", "bias", bias, 1, _types[FP32], device)
        _shape("linear", "bias", bias, out_c)
        bp = bias.data_ptr()
    if residual is not None:
        rs = (residual.data_ptr(), _look("linear", "residual", residual, 2, dtype, device)[0])
        _shape("linear", "residual", residual, rows, out_c)
    if workspace is not None:
        space = _workspace("linear", workspace, device)
    return _LinearParams(code, act, rows, in_c, out_c, x.data_ptr(), xs[0], weights.data_ptr(), ws[0], bp, *rs, op, os or 0, *space), device


def linear_workspace(x, weights) -> int:
    """kgh_linear_workspace: bytes of workspace that ``linear`` makes use of for
    tensors of these shapes and types (0: none). A larger one serves too."""
    p, device = _linear_params(x, weights, None, None, None, None, None)
    p.out_stride = p.out_channels
    n = ctypes.c_uint64()
    hip_check(_library().kgh_linear_workspace(device, p, n))
    return n.value


def linear(x, weights, out, bias=None, activation=None, residual=None, workspace=None, stream=None):
    """kgh_linear: out = activation(x @ weights.T + bias) + residual.

    x [rows, in], weights [out, in], out and residual [rows, out] of one type
    (float32, float16, bfloat16) with any row strides; bias [out] float32;
    activation one of ``ACTIVATIONS``. residual may be out itself. workspace: at
    least ``linear_workspace`` bytes of its own for calls that may overlap."""
    p, device = _linear_params(x, weights, out, bias, activation, residual, workspace)
    _no_gradients("linear", x, weights, out, bias, residual)
    hip_check((_lib or _library()).kgh_linear(device, p, _stream(x, device) if stream is None else stream))
    return out


def rope_axes(x, positions, freqs, out, layout="interleaved", inverse=False, stream=None):
    """kgh_rope_axes: pair p of head h of token t turns by the angle
    sum_a positions[t, a] * freqs[h // (heads // tables), p, a].

    x and out [tokens, heads, dim] of one type with any token and head strides;
    positions [tokens, axes] int32, 1 to 4 axes; freqs [tables, pairs, axes]
    float32, contiguous; layout "interleaved" (channels 2p and 2p + 1) or
    "halves" (p and p + pairs). Channels from 2 * pairs on are copied; inverse
    turns back. out may be x itself."""
    code, device = _first("rope_axes", "x", x)
    xs = _look("rope_axes", "x", x, 3, x.dtype, device)
    os = _look("rope_axes", "out", out, 3, x.dtype, device)
    ps = _look("rope_axes", "positions", positions, 2, _types["int32"], device)
    fs = _look("rope_axes", "freqs", freqs, 3, _types[FP32], device)
    tokens, heads, dim = x.shape
    tables, pairs, axes = freqs.shape
    _shape("rope_axes", "out", out, tokens, heads, dim)
    _shape("rope_axes", "positions", positions, tokens, axes)
    _sizes("rope_axes", tokens, heads, dim, tables, pairs, axes)
    if (fs[0] != pairs * axes and tables > 1) or (fs[1] != axes and pairs > 1):
        _invalid("rope_axes: freqs is not contiguous")
    _no_gradients("rope_axes", x, freqs, out)
    kind = ROPE_LAYOUTS.get(layout)
    if kind is None:
        _invalid(f"rope_axes: unknown layout {layout!r}")
    p = _RopeParams(code, kind, 1 if inverse else 0, axes, tokens, heads, dim, pairs, tables, x.data_ptr(), xs[0], xs[1],
                    positions.data_ptr(), ps[0], freqs.data_ptr(), out.data_ptr(), os[0], os[1])
    hip_check((_lib or _library()).kgh_rope_axes(device, p, _stream(x, device) if stream is None else stream))
    return out


def _attention_params(q, k, v, scale, precise):
    code, device = _first("cross_attention", "q", q)
    dtype = q.dtype
    qs = _look("cross_attention", "q", q, 4, dtype, device)
    ks = _look("cross_attention", "k", k, 4, dtype, device)
    vs = _look("cross_attention", "v", v, 4, dtype, device)
    batch, lq, heads, dq = q.shape
    _, lk, kv_heads, _ = k.shape
    dv = v.shape[3]
    _shape("cross_attention", "k", k, batch, lk, kv_heads, dq)
    _shape("cross_attention", "v", v, batch, lk, kv_heads, dv)
    _sizes("cross_attention", batch, lq, heads, dq, lk, kv_heads, dv)
    if scale is None:
        scale = max(dq, 1) ** -0.5
    return _AttentionParams(code, batch, lq, lk, heads, kv_heads, dq, dv, scale, 1 if precise else 0, q.data_ptr(), qs[:3], k.data_ptr(), ks[:3],
                            v.data_ptr(), vs[:3]), device


def cross_attention_workspace(q, k, v, precise=False) -> int:
    """kgh_cross_attention_workspace: bytes of workspace that ``cross_attention``
    makes use of for tensors of these shapes and types (0: none). A larger one
    serves too."""
    p, device = _attention_params(q, k, v, None, precise)
    n = ctypes.c_uint64()
    hip_check(_library().kgh_cross_attention_workspace(device, p, n))
    return n.value


def cross_attention(q, k, v, out, scale=None, key_lengths=None, key_mask=None, workspace=None, stream=None, precise=False):
    """kgh_cross_attention: softmax(scale * q k^T) v over the keys that take part.

    q [batch, queries, heads, dq], k [batch, keys, kv_heads, dq], v [batch, keys,
    kv_heads, dv], out [batch, queries, heads, dv] of one type, any strides but
    that of the last axis; heads // kv_heads query heads share a kv head. scale
    defaults to dq ** -0.5. key_lengths [batch] int32: keys from there on take no
    part; key_mask [batch, keys] uint8 or bool: nor do those with 0. What k and v
    hold there is not used. A row without a key is zeros. workspace: at least
    ``cross_attention_workspace`` bytes of its own for calls that may overlap;
    without one, long keys are not split over workgroups. precise: in 16 bits the
    softmax's weights keep twice their type's bits for the product with v, which
    those of more than 32 rows (query, head of the group) a kv head do not
    otherwise."""
    p, device = _attention_params(q, k, v, scale, precise)
    os = _look("cross_attention", "out", out, 4, q.dtype, device)
    batch = p.batch
    _shape("cross_attention", "out", out, batch, p.q_len, p.heads, p.v_head_dim)
    p.out, p.out_strides = out.data_ptr(), os[:3]
    if key_lengths is not None:
        ls = _look("cross_attention", "key_lengths", key_lengths, 1, _types["int32"], device)
        _shape("cross_attention", "key_lengths", key_lengths, batch)
        p.key_lengths = key_lengths.data_ptr()
    if key_mask is not None:
        kind = _code("cross_attention", "key_mask", key_mask)
        ms = _look("cross_attention", "key_mask", key_mask, 2, _types[kind if kind in ("uint8", "bool") else "uint8"], device)
        _shape("cross_attention", "key_mask", key_mask, batch, p.k_len)
        p.key_mask, p.key_mask_stride = key_mask.data_ptr(), ms[0]
    _no_gradients("cross_attention", q, k, v, out)
    if workspace is not None:
        p.workspace, p.workspace_bytes = _workspace("cross_attention", workspace, device)
    hip_check((_lib or _library()).kgh_cross_attention(device, p, _stream(q, device) if stream is None else stream))
    return out


def quantize_rows(x, out, scales, stream=None):
    """kgh_quantize_rows: x in 8 bits, a scale for each row: out stands for out *
    scales[:, None].

    x [rows, channels] (float32, float16, bfloat16), out [rows, channels] int8, any row
    strides; scales [rows] float32. Returns out. A row's largest magnitude becomes 127;
    rows of zeros have scale 0, rows with an infinity or NaN zeros and scale NaN."""
    code, device = _first("quantize_rows", "x", x)
    xs = _look("quantize_rows", "x", x, 2, x.dtype, device)
    os = _look("quantize_rows", "out", out, 2, _types["int8"], device)
    _look("quantize_rows", "scales", scales, 1, _types[FP32], device)
    rows, channels = x.shape
    _shape("quantize_rows", "out", out, rows, channels)
    _shape("quantize_rows", "scales", scales, rows)
    _sizes("quantize_rows", rows, channels)
    _no_gradients("quantize_rows", x, scales)
    p = _QuantizeParams(code, channels, rows, x.data_ptr(), xs[0], out.data_ptr(), os[0], scales.data_ptr())
    hip_check((_lib or _library()).kgh_quantize_rows(device, p, _stream(x, device) if stream is None else stream))
    return out


def linear_int8_workspace(x, weights) -> int:
    """kgh_linear_int8_workspace: bytes of workspace that ``linear_int8`` makes use of
    for tensors of these shapes (0: none). A larger one serves too."""
    rows, in_c = x.shape
    _sizes("linear_int8", rows, in_c, weights.shape[0])
    p = _LinearInt8Params(FP32, 0, rows, in_c, weights.shape[0])
    p.out_stride = p.out_channels
    n = ctypes.c_uint64()
    hip_check((_lib or _library()).kgh_linear_int8_workspace(x.get_device(), p, n))
    return n.value


def linear_int8(x, x_scales, weights, weight_scales, out, bias=None, activation=None, residual=None, workspace=None, stream=None):
    """kgh_linear_int8: out = activation((x @ weights.T) * x_scales[:, None] *
    weight_scales + bias) + residual, the products of 8-bit integers and their sums
    exact.

    x [rows, in] and weights [out, in] int8, x_scales [rows] and weight_scales [out]
    float32, as ``quantize_rows`` makes them; out and residual [rows, out] of one type
    (float32, float16, bfloat16); any row strides; bias [out] float32; activation one of
    ``ACTIVATIONS``. residual may be out itself. workspace: at least
    ``linear_int8_workspace`` bytes of its own for calls that may overlap."""
    code, device = _first("linear_int8", "out", out)
    dtype = out.dtype
    i8, f32 = _types["int8"], _types[FP32]
    xs = _look("linear_int8", "x", x, 2, i8, device)
    ws = _look("linear_int8", "weights", weights, 2, i8, device)
    os = _look("linear_int8", "out", out, 2, dtype, device)
    _look("linear_int8", "x_scales", x_scales, 1, f32, device)
    _look("linear_int8", "weight_scales", weight_scales, 1, f32, device)
    rows, in_c = x.shape
    out_c, w_in = weights.shape
    if w_in != in_c:
        _invalid(f"linear_int8: weights have {w_in} input channels, x has {in_c}")
    _sizes("linear_int8", rows, in_c, out_c)
    _shape("linear_int8", "out", out, rows, out_c)
    _shape("linear_int8", "x_scales", x_scales, rows)
    _shape("linear_int8", "weight_scales", weight_scales, out_c)
    act = ACTIVATIONS.get(activation or "identity")
    if act is None:
        _invalid(f"linear_int8: unknown activation {activation!r}")
    bp = None
    rs = space = (None, 0)
    if bias is not None:
        _look("linear_int8", "bias", bias, 1, f32, device)
        _shape("linear_int8", "bias", bias, out_c)
        bp = bias.data_ptr()
    if residual is not None:
        rs = (residual.data_ptr(), _look("linear_int8", "residual", residual, 2, dtype, device)[0])
        _shape("linear_int8", "residual", residual, rows, out_c)
    if workspace is not None:
        space = _workspace("linear_int8", workspace, device)
    _no_gradients("linear_int8", x_scales, weight_scales, out, bias, residual)
    p = _LinearInt8Params(code, act, rows, in_c, out_c, x.data_ptr(), xs[0], x_scales.data_ptr(), weights.data_ptr(), ws[0], weight_scales.data_ptr(),
                          bp, *rs, out.data_ptr(), os[0], *space)
    hip_check((_lib or _library()).kgh_linear_int8(device, p, _stream(out, device) if stream is None else stream))
    return out


def _norm_start(op, x, groups, activation):
    """What both directions' parameters begin with, x's strides and the device."""
    code, device = _first(op, "x", x)
    xs = _look(op, "x", x, 3, x.dtype, device)
    batch, positions, channels = x.shape
    _sizes(op, batch, positions, channels)
    if groups < 1 or channels % groups != 0:
        _invalid(f"{op}: groups must divide channels")
    act = ACTIVATIONS.get(activation or "identity")
    if act is None:
        _invalid(f"{op}: unknown activation {activation!r}")
    return (code, act, batch, positions, channels, groups), xs, device


def _norm_inputs(op, batch, positions, channels, device, weight, bias, lengths, mask):
    """Pointers of the arguments that both directions may have, the last one's stride."""
    wp = bp = lp = mp = None
    ms = 0
    if weight is not None:
        _look(op, "weight", weight, 1, _types[FP32], device)
        _shape(op, "weight", weight, channels)
        wp = weight.data_ptr()
    if bias is not None:
        _look(op, "bias", bias, 1, _types[FP32], device)
        _shape(op, "bias", bias, channels)
        bp = bias.data_ptr()
    if lengths is not None:
        _look(op, "lengths", lengths, 1, _types["int32"], device)
        _shape(op, "lengths", lengths, batch)
        lp = lengths.data_ptr()
    if mask is not None:
        kind = _code(op, "mask", mask)
        ms = _look(op, "mask", mask, 2, _types[kind if kind in ("uint8", "bool") else "uint8"], device)[0]
        _shape(op, "mask", mask, batch, positions)
        mp = mask.data_ptr()
    return wp, bp, lp, mp, ms


def _whole(op, name, t, shape, device):
    """The pointer of a contiguous float32 tensor."""
    strides = _look(op, name, t, len(shape), _types[FP32], device)
    _shape(op, name, t, *shape)
    n = 1
    for size, stride in zip(reversed(shape), reversed(strides)):
        if stride != n and size > 1:
            _invalid(f"{op}: {name} is not contiguous")
        n *= size
    return t.data_ptr()


def group_norm_workspace(x, out, groups) -> int:
    """kgh_group_norm_workspace: bytes of workspace that ``group_norm`` needs for
    tensors of these shapes and types (0: none). A larger one serves too."""
    start, xs, device = _norm_start("group_norm", x, groups, None)
    p = _GroupNormParams(*start)
    if _code("group_norm", "out", out) == "int8":
        p.out_scales = 4
    n = ctypes.c_uint64()
    hip_check((_lib or _library()).kgh_group_norm_workspace(device, p, n))
    return n.value


def group_norm(x, out, groups, weight=None, bias=None, eps=1e-5, activation=None, lengths=None, mask=None, out_scales=None, stats=None,
               workspace=None, stream=None):
    """kgh_group_norm: activation((x - mean) / sqrt(variance + eps) * weight + bias),
    mean and variance of each item over a group's channels at the positions that take
    part.

    x [batch, positions, channels] (float32, float16, bfloat16), out of the same shape
    and type, any strides but that of the last axis; or out int8 and out_scales [batch,
    positions] float32, contiguous: rows in 8 bits as ``quantize_rows`` makes them.
    groups runs of channels; weight and bias [channels] float32; activation one of
    ``ACTIVATIONS``. lengths [batch] int32: positions from there on take no part; mask
    [batch, positions] uint8 or bool: nor do those with 0. What x holds there is not
    used, and out is zero. stats [batch, groups, 2] float32, contiguous, takes mean and
    1 / sqrt(variance + eps) for ``group_norm_backward``. out may be x itself. workspace:
    at least ``group_norm_workspace`` bytes, of its own for calls that may overlap."""
    start, xs, device = _norm_start("group_norm", x, groups, activation)
    _, _, batch, positions, channels, _ = start
    inputs = _norm_inputs("group_norm", batch, positions, channels, device, weight, bias, lengths, mask)
    sp = tp = None
    if out_scales is not None:
        sp = _whole("group_norm", "out_scales", out_scales, (batch, positions), device)
    os = _look("group_norm", "out", out, 3, x.dtype if out_scales is None else _types["int8"], device)
    _shape("group_norm", "out", out, batch, positions, channels)
    if stats is not None:
        tp = _whole("group_norm", "stats", stats, (batch, groups, 2), device)
    _no_gradients("group_norm", x, out, weight, bias)
    space = _workspace("group_norm", workspace, device)
    p = _GroupNormParams(*start, eps, x.data_ptr(), xs[0], xs[1], *inputs, out.data_ptr(), os[0], os[1], sp, tp, *space)
    hip_check((_lib or _library()).kgh_group_norm(device, p, _stream(x, device) if stream is None else stream))
    return out


def group_norm_backward_workspace(x, groups) -> int:
    """kgh_group_norm_backward_workspace: bytes of workspace that
    ``group_norm_backward`` needs for a tensor of this shape and type (0: none). A larger
    one serves too."""
    start, xs, device = _norm_start("group_norm_backward", x, groups, None)
    n = ctypes.c_uint64()
    hip_check((_lib or _library()).kgh_group_norm_backward_workspace(device, _GroupNormBackwardParams(*start), n))
    return n.value


def group_norm_backward(x, grad_out, stats, grad_x, groups, weight=None, bias=None, activation=None, lengths=None, mask=None, grad_weight=None,
                        grad_bias=None, workspace=None, stream=None):
    """kgh_group_norm_backward: the gradients of ``group_norm`` for x (into grad_x,
    which is returned), and where they are given for weight (grad_weight) and bias
    (grad_bias).

    x, grad_out and grad_x [batch, positions, channels] of one type, any strides but
    that of the last axis; stats [batch, groups, 2] of the forward call; weight, bias,
    activation, lengths and mask as they were there; grad_weight and grad_bias [channels]
    float32. grad_x is zero at positions that take no part. workspace: at least
    ``group_norm_backward_workspace`` bytes, of its own for calls that may overlap."""
    op = "group_norm_backward"
    start, xs, device = _norm_start(op, x, groups, activation)
    _, _, batch, positions, channels, _ = start
    inputs = _norm_inputs(op, batch, positions, channels, device, weight, bias, lengths, mask)
    gs = _look(op, "grad_out", grad_out, 3, x.dtype, device)
    os = _look(op, "grad_x", grad_x, 3, x.dtype, device)
    _shape(op, "grad_out", grad_out, batch, positions, channels)
    _shape(op, "grad_x", grad_x, batch, positions, channels)
    tp = _whole(op, "stats", stats, (batch, groups, 2), device)
    wp = bp = None
    if grad_weight is not None:
        wp = _whole(op, "grad_weight", grad_weight, (channels,), device)
    if grad_bias is not None:
        bp = _whole(op, "grad_bias", grad_bias, (channels,), device)
    _no_gradients(op, x, grad_out, grad_x, weight, bias, grad_weight, grad_bias)
    space = _workspace(op, workspace, device)
    p = _GroupNormBackwardParams(*start, x.data_ptr(), xs[0], xs[1], grad_out.data_ptr(), gs[0], gs[1], tp, *inputs, grad_x.data_ptr(), os[0], os[1],
                                 wp, bp, *space)
    hip_check((_lib or _library()).kgh_group_norm_backward(device, p, _stream(x, device) if stream is None else stream))
    return grad_x
