"""Stream operators on device tensors: the layers of a recurrent latent model.

The decoder turns latents into audio, one 40 ms frame of every stream a step.
These are the operators of a model that makes those latents the same way, in
the decoder's own terms: channels-last rows, one call for all streams, a
fixed-size state per stream in a slot of a pool, transactional slot codes.

* ``causal_conv``: short causal depthwise convolution with a carried history;
* ``selective_scan``: selective state space scan with carried states;
* ``group_norm``: group norm with SiLU or the decoder's Snake;
* ``project_int4``: projection by 4-bit weights with group scales.

Rows and sequences. Arrays are torch tensors on one CUDA device (fp32, bf16 or
fp16, adjacent channels, any row stride):

* ``[rows, channels]`` alone: a decoding step, every row a stream of its own;
* ``[n, length, channels]``: n sequences of one length;
* ``[rows, channels]`` with ``offsets`` (int32 ``[n + 1]`` on the device):
  packed sequences, sequence i in rows ``offsets[i]:offsets[i + 1]``, empty
  ones among them. Rows of no sequence keep what ``out`` held.

States. A state tensor is ``[slots, 2, ...]``: two tables per slot.
``codes`` (int32 ``[n]`` on the device, see ``StreamSlots``) name the table a
sequence reads and whether it starts afresh; the advanced state goes to the
other table, so a step that is not committed has changed nothing.

``status`` is an optional int32 tensor of one element, zero before the call:
0x201 after it means offsets that decrease or leave the rows (the call's
outputs are then undefined), 0x202 a code outside the pool (its sequence is
skipped). Without it the same happens silently; either way no memory outside
the arrays is touched.

Coefficients are contiguous fp32; sums, states and statistics run in fp32, and
every output is rounded once to its type. Work is enqueued on the current
stream of the tensors' device without synchronising and may be captured in a
CUDA graph. The operators are for inference: tensors that want gradients or
carry forward derivatives are refused, states and outputs among them. They run
in ``libfav_cuda.so``; there is no CPU path.
"""
from __future__ import annotations

import numpy as np
import torch
from torch.autograd import forward_ad as _forward

from . import _native
from ._native import CONV_ARGS, INT4_ARGS, NORM_ARGS, SCAN_ARGS

__all__ = ["causal_conv", "selective_scan", "group_norm", "project_int4", "quantize_int4", "conv_state",
           "scan_state", "StreamSlots"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "silu": 1, "snake": 2}
_I32, _F32 = torch.int32, torch.float32
_FRESH = 2
_INT = 2 ** 31 - 1   # the library counts in 32 bits, to which ctypes would cut larger numbers
_SLOTS = 2 ** 29
_lib = None
_grad_enabled = torch.is_grad_enabled
_empty_like = torch.empty_like
# A CUDA tensor in hand means that CUDA is initialised: its own getters will do.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


# A step's call must not cost more than its kernel, so plain tensors go to entry
# points that read and check them natively (a fifth of the time that it takes from
# here). What those do not take is checked below, which also says what is wrong.
_KINDS = {torch.Tensor, torch.nn.Parameter, type(None)}
# What the exchange raises of a tensor without plain memory (sparse, quantised, nested).
_UNREADABLE = (RuntimeError, BufferError)
_held = False  # not looked for yet; None where the tensors cannot be read natively


def _native_path(*tensors):
    """The native entry points, if all of ``tensors`` are plain ones without gradients, or None but for the first."""
    global _held
    if tensors[0] is None or _forward._current_level >= 0:
        return None
    if _held is False:
        _held = _native.tensor_functions(torch.Tensor) if torch.cuda.is_available() else None
    if _held is None or not _KINDS.issuperset(map(type, tensors)):
        return None
    if _grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return None
    return _held


def _library(index):
    """The native library, for tensors on CUDA device ``index`` (negative: the CPU)."""
    global _lib
    if index < 0:
        raise RuntimeError("Stream operators run on CUDA tensors; there is no CPU path")
    if _lib is None:
        _lib = _native.load_library()
    return _lib


def _call(lib, function, args, index):
    """Run a C-ABI operator on the current stream of device ``index``."""
    if _current_device() == index:
        status = function(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = function(args, _raw_stream(index))
    if status:
        _native.check(lib, status)


# The checks below run on every call of a step that takes microseconds, so they
# read each tensor attribute once. One that is missing is a ValueError too.
_MISSING = (AttributeError, KeyError, TypeError, RuntimeError)


def _main(x):
    """Checks an operator's first argument; returns its type code and device index."""
    try:
        kind, index = _TYPES[x.dtype], x.get_device()
        if _dense(x, x.dtype, index):
            return kind, index
    except _MISSING:
        pass
    raise ValueError("x must be a dense float32, bfloat16 or float16 tensor")


def _dense(t, dtype, index):
    """Whether t lies in plain memory of device ``index`` (which a negated view does not stand for)."""
    return (t.dtype is dtype and t.get_device() == index and t.layout is torch.strided and not t.is_nested
            and not t.is_neg())


def _no_gradients(*tensors):
    """Refuses tensors, inputs and outputs alike, that want gradients or carry forward derivatives."""
    tensors = [t for t in tensors if isinstance(t, torch.Tensor) and t.is_floating_point()]
    if _grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("Stream operators have no gradients; call them under torch.no_grad()")
    if _forward._current_level >= 0 and any(_forward.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("Stream operators have no gradients, forward ones neither; detach their tensors")


def _array(t, name, dtype, index, shape):
    """Address and row stride of an array of x's type with adjacent channels."""
    try:
        good = _dense(t, dtype, index) and t.shape == shape
    except _MISSING:
        good = False
    if not good:
        raise ValueError(f"{name} must be a {dtype} tensor of shape {list(shape)} on x's device")
    strides = t.stride()
    if strides[-1] != 1 and shape[-1] != 1:
        raise ValueError(f"{name} must have adjacent channels (stride 1)")
    if len(shape) == 2:
        return t.data_ptr(), strides[0] if shape[0] != 1 else shape[1]
    return t.data_ptr(), _row_stride(name, shape, strides)


def _row_stride(name, shape, strides):
    """The one stride between the rows of ``[n, length, ...]``."""
    if shape[1] == 1:
        return strides[0]
    if shape[0] != 1 and strides[0] != shape[1] * strides[1]:
        raise ValueError(f"{name} must have one stride between all its rows")
    return strides[1]


def _vector(t, name, index, shape):
    """Address of a contiguous fp32 coefficient array (0 for None)."""
    if t is None:
        return 0
    try:
        if _dense(t, _F32, index) and t.shape == shape and t.is_contiguous():
            return t.data_ptr()
    except _MISSING:
        pass
    raise ValueError(f"{name} must be a contiguous float32 tensor of shape {list(shape)} on x's device")


def _index(t, name, index, count):
    try:
        if _dense(t, _I32, index) and t.shape == (count,) and t.is_contiguous():
            return t.data_ptr()
    except _MISSING:
        pass
    raise ValueError(f"{name} must be a contiguous int32 tensor of {count} elements on x's device")


def _sequences(shape, offsets, index):
    """(sequences, length, rows, offsets address) of x; length 0 with offsets."""
    if offsets is not None:
        if len(shape) != 2:
            raise ValueError("Packed sequences (offsets) require x of shape [rows, channels]")
        count = offsets.shape[0] if isinstance(offsets, torch.Tensor) and offsets.dim() else 0
        if count < 1:
            raise ValueError("offsets must hold n + 1 elements")
        n, length, rows, at = count - 1, 0, shape[0], _index(offsets, "offsets", index, count)
    elif len(shape) == 2:
        n, length, rows, at = shape[0], 1, shape[0], 0
    elif len(shape) == 3:
        if shape[1] < 1:
            raise ValueError("Sequences without offsets must have at least one row")
        n, length, rows, at = shape[0], shape[1], shape[0] * shape[1], 0
    else:
        raise ValueError("x must have shape [rows, channels] or [n, length, channels]")
    if n > _INT or rows > _INT or shape[-1] > _INT:
        raise ValueError("x has too many rows or channels: each below 2^31")
    return n, length, rows, at


def _states(state, codes, dtype, index, n, shape):
    """Addresses of a state pool and its codes, and its slots (0s for None)."""
    if state is None and codes is None:
        return 0, 0, 0
    if state is None or codes is None:
        raise ValueError("state and codes go together")
    try:
        held = state.shape
        good = _dense(state, dtype, index) and held[1:] == shape and state.is_contiguous()
    except _MISSING:
        good = False
    if not good:
        raise ValueError(f"state must be a contiguous {dtype} tensor of shape {['slots', *shape]} on x's device")
    if held[0] < n:
        raise ValueError(f"{n} sequences need at least as many slots; state has {held[0]}")
    if held[0] > _SLOTS:
        raise ValueError("state has too many slots: up to 2^29")
    return state.data_ptr(), _index(codes, "codes", index, n), held[0]


def causal_conv(x, weight, bias=None, *, activation=None, offsets=None, state=None, codes=None, status=None, out=None):
    """Causal depthwise convolution over each sequence's rows, 2 to 8 taps.

    ``y[t, c] = act(bias[c] + sum_j weight[c, j] * x[t - (taps - 1) + j, c])``
    with ``weight`` ``[channels, taps]`` (the last tap meets the newest row),
    ``bias`` ``[channels]`` and ``activation`` None or ``"silu"``. Rows before a
    sequence's first come from ``state`` ``[slots, 2, taps - 1, channels]`` (x's
    type, oldest first; ``conv_state`` makes one) or are zero.
    """
    native = _native_path(x, weight, bias, offsets, state, codes, status, out)
    if native is not None and (activation is None or activation == "silu"):
        try:
            y = _empty_like(x) if out is None else out
            if native.fav_causal_conv_tensors(x, weight, bias, offsets, state, codes, status, y,
                                              _ACTIVATIONS[activation]) == 0:
                return y
        except _UNREADABLE:
            pass
    kind, index = _main(x)
    _no_gradients(x, weight, bias, state, out)
    shape, dtype = x.shape, x.dtype
    n, length, rows, offsets_at = _sequences(shape, offsets, index)
    channels = shape[-1]
    taps = weight.shape[1] if isinstance(weight, torch.Tensor) and weight.dim() == 2 else 0
    if not 2 <= taps <= 8:
        raise ValueError("weight must have shape [channels, taps] with 2 to 8 taps")
    if activation is not None and activation != "silu":
        raise ValueError("activation must be None or 'silu'")
    weight_at = _vector(weight, "weight", index, (channels, taps))
    bias_at = _vector(bias, "bias", index, (channels,))
    x_at, x_stride = _array(x, "x", dtype, index, shape)
    pool_at, codes_at, slots = _states(state, codes, dtype, index, n, (2, taps - 1, channels))
    status_at = _index(status, "status", index, 1) if status is not None else 0
    lib = _library(index)
    if out is None:  # contiguous: x's rows have one stride, or lie that way themselves
        out = _empty_like(x)
        y_at, y_stride = out.data_ptr(), channels
    else:
        y_at, y_stride = _array(out, "out", dtype, index, shape)
    if n:
        _call(lib, lib.fav_causal_conv,
              CONV_ARGS(x_at, y_at, x_stride, y_stride, weight_at, bias_at, pool_at, codes_at, offsets_at, status_at,
                        kind, channels, taps, _ACTIVATIONS[activation], n, length, rows, slots), index)
    return out


def _maps(t, name, dtype, index, lead, groups, states):
    """Address, row stride and group stride of an input or output map."""
    shape = (*lead, groups, states)
    try:
        good = _dense(t, dtype, index) and t.shape == shape
    except _MISSING:
        good = False
    if not good:
        raise ValueError(f"{name} must be a {dtype} tensor of shape {list(shape)} on x's device")
    strides = t.stride()
    if strides[-1] != 1 and states != 1:
        raise ValueError(f"{name} must have adjacent states (stride 1)")
    return (t.data_ptr(), strides[0] if len(lead) == 1 else _row_stride(name, shape, strides),
            strides[-2] if groups > 1 else 0)


def selective_scan(x, dt, a, b, c, *, d=None, z=None, dt_bias=None, softplus=True, offsets=None, state=None,
                   codes=None, status=None, out=None):
    """Selective state space scan over each sequence's rows.

    Channel c of group g keeps N states; ``delta = softplus(dt + dt_bias)`` (or
    the sum itself), and row by row

    ``h[n, c] = exp(delta * a[n, c]) * h[n, c] + delta * x[t, c] * b[t, g, n]``
    ``y[t, c] = (sum_n c[t, g, n] * h[n, c] + d[c] * x[t, c]) * silu(z[t, c])``

    ``dt`` and ``z`` are shaped like ``x``; ``b`` and ``c`` are
    ``[..., groups, N]`` over the same rows (groups divide the channels); ``a``
    is ``[N, channels]`` and finite, and ``d`` and ``dt_bias`` are ``[channels]``. N is 1 to
    128. ``state`` is ``[slots, 2, N, channels]`` fp32 (``scan_state``).
    """
    native = _native_path(x, dt, a, b, c, d, z, dt_bias, offsets, state, codes, status, out)
    if native is not None:
        arrays = (x, dt, a, b, c, d, z, dt_bias, offsets, state, codes, status)
        softplus = bool(softplus)
        try:
            y = _empty_like(x) if out is None else out
            result = native.fav_selective_scan_tensors(*arrays, None, y, softplus)
            if result > 64:
                workspace = x.new_empty(result, dtype=torch.uint8)
                result = native.fav_selective_scan_tensors(*arrays, workspace, y, softplus)
            if result == 0:
                return y
        except _UNREADABLE:
            pass
    kind, index = _main(x)
    _no_gradients(x, dt, a, b, c, d, z, dt_bias, state, out)
    shape, dtype = x.shape, x.dtype
    n, length, rows, offsets_at = _sequences(shape, offsets, index)
    channels = shape[-1]
    states = a.shape[0] if isinstance(a, torch.Tensor) and a.dim() == 2 else 0
    if not 1 <= states <= 128:
        raise ValueError("a must have shape [states, channels] with 1 to 128 states")
    groups = b.shape[-2] if isinstance(b, torch.Tensor) and b.dim() == len(shape) + 1 else 0
    if groups < 1 or channels % groups:
        raise ValueError("b must have shape [..., groups, states] with groups that divide the channels")
    x_at, x_stride = _array(x, "x", dtype, index, shape)
    dt_at, dt_stride = _array(dt, "dt", dtype, index, shape)
    z_at, z_stride = _array(z, "z", dtype, index, shape) if z is not None else (0, 0)
    lead = shape[:-1]
    b_at, b_stride, b_group = _maps(b, "b", dtype, index, lead, groups, states)
    c_at, c_stride, c_group = _maps(c, "c", dtype, index, lead, groups, states)
    a_at = _vector(a, "a", index, (states, channels))
    d_at = _vector(d, "d", index, (channels,))
    bias_at = _vector(dt_bias, "dt_bias", index, (channels,))
    pool_at, codes_at, slots = _states(state, codes, _F32, index, n, (2, states, channels))
    status_at = _index(status, "status", index, 1) if status is not None else 0
    lib = _library(index)
    if out is None:  # contiguous: x's rows have one stride, or lie that way themselves
        out = _empty_like(x)
        y_at, y_stride = out.data_ptr(), channels
    else:
        y_at, y_stride = _array(out, "out", dtype, index, shape)
    if not n:
        return out
    fixed = (x_at, dt_at, z_at, b_at, c_at, y_at, x_stride, dt_stride, z_stride, b_stride, b_group, c_stride, c_group,
             y_stride, a_at, d_at, bias_at, pool_at, codes_at, offsets_at, status_at)
    sizes = (kind, channels, states, groups, bool(softplus), n, length, rows, slots)
    args = SCAN_ARGS(*fixed, 0, 0, *sizes)
    if length != 1:
        need = lib.fav_selective_scan_workspace_bytes(args)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
            args = SCAN_ARGS(*fixed, workspace.data_ptr(), need, *sizes)
    _call(lib, lib.fav_selective_scan, args, index)
    return out


def group_norm(x, groups, weight=None, bias=None, *, eps=1e-5, activation=None, alpha=None, reciprocal=None,
               offsets=None, status=None, out=None):
    """Group norm with an activation, channels last.

    ``y = act((x - mean) / sqrt(variance + eps) * weight + bias)`` with the mean
    and the biased variance over a sequence's rows and the neighbouring
    ``channels / groups`` channels of a group; of ``[rows, channels]`` without
    ``offsets`` every row is normalised by itself, as a step needs it.
    ``activation`` is None, ``"silu"`` or ``"snake"``, the decoder's
    ``v + reciprocal * sin(alpha * v)**2`` with ``[channels]`` coefficients.
    """
    if type(groups) is int and groups <= _INT and activation in _ACTIVATIONS and eps >= 0:
        native = _native_path(x, weight, bias, alpha, reciprocal, offsets, status, out)
        if native is not None:
            try:
                y = _empty_like(x) if out is None else out
                if native.fav_group_norm_tensors(x, weight, bias, alpha, reciprocal, offsets, status, y, groups, eps,
                                                 _ACTIVATIONS[activation]) == 0:
                    return y
            except _UNREADABLE:
                pass
    kind, index = _main(x)
    _no_gradients(x, weight, bias, alpha, reciprocal, out)
    shape, dtype = x.shape, x.dtype
    n, length, rows, offsets_at = _sequences(shape, offsets, index)
    channels = shape[-1]
    if type(groups) is not int or groups < 1 or channels % groups:
        raise ValueError("groups must be a positive int that divides the channels")
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be None, 'silu' or 'snake'")
    if (activation == "snake") != (alpha is not None) or (activation == "snake") != (reciprocal is not None):
        raise ValueError("alpha and reciprocal belong to activation='snake'")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    per = (channels,)
    coefficients = (_vector(weight, "weight", index, per), _vector(bias, "bias", index, per),
                    _vector(alpha, "alpha", index, per), _vector(reciprocal, "reciprocal", index, per))
    x_at, x_stride = _array(x, "x", dtype, index, shape)
    status_at = _index(status, "status", index, 1) if status is not None else 0
    lib = _library(index)
    if out is None:  # contiguous: x's rows have one stride, or lie that way themselves
        out = _empty_like(x)
        y_at, y_stride = out.data_ptr(), channels
    else:
        y_at, y_stride = _array(out, "out", dtype, index, shape)
    if n:
        _call(lib, lib.fav_group_norm,
              NORM_ARGS(x_at, y_at, x_stride, y_stride, *coefficients, offsets_at, status_at, eps, kind, channels,
                        groups, _ACTIVATIONS[activation], n, length, rows), index)
    return out


def project_int4(x, weight, scales, bias=None, *, group, out=None):
    """Rows times 4-bit weights: ``y = x @ w.T + bias`` for the rows of a step.

    ``w[r, k] = (q[r, k] - 8) * scales[r, k // group]`` with ``q`` in 0..15, two
    to a byte along k, the even k in the low half: ``weight`` is uint8
    ``[out, depth / 2]``, ``scales`` fp32 ``[out, ceil(depth / group)]``
    (``quantize_int4`` makes both), ``x`` ``[rows, depth]``. ``group`` and the
    depth are multiples of 32.
    """
    native = _native_path(x, weight, scales, bias, out)
    if (native is not None and type(group) is int and group <= _INT and weight is not None and x.dim() == 2
            and weight.dim() == 2):
        try:
            y = x.new_empty((x.shape[0], weight.shape[0])) if out is None else out
            if native.fav_project_int4_tensors(x, weight, scales, bias, y, group) == 0:
                return y
        except _UNREADABLE:
            pass
    kind, index = _main(x)
    _no_gradients(x, scales, bias, out)
    shape, dtype = x.shape, x.dtype
    if len(shape) != 2:
        raise ValueError("x must have shape [rows, depth]")
    rows, depth = shape
    if type(group) is not int or group < 32 or group % 32 or depth < 32 or depth % 32:
        raise ValueError("group and the depth must be positive multiples of 32")
    try:
        packed = weight.shape
        good = (_dense(weight, torch.uint8, index) and len(packed) == 2 and packed[1] == depth // 2
                and weight.is_contiguous())
    except _MISSING:
        good = False
    if not good:
        raise ValueError(f"weight must be a contiguous uint8 tensor of shape ['out', {depth // 2}] on x's device")
    weight_at = weight.data_ptr()
    if weight_at % 16:
        raise ValueError("weight must be 16-byte aligned")
    if scales is None:
        raise ValueError("scales are required")
    width = packed[0]
    if rows > _INT or depth > _INT or width > _INT:
        raise ValueError("x or weight is too large: each size below 2^31")
    scales_at = _vector(scales, "scales", index, (width, -(-depth // group)))
    if group > _INT:   # one scale a row, as for any group that is wider than the depth
        group = 2 ** 30
    bias_at = _vector(bias, "bias", index, (width,))
    x_at, x_stride = _array(x, "x", dtype, index, shape)
    lib = _library(index)
    if out is None:
        out = x.new_empty((rows, width))
        y_at, y_stride = out.data_ptr(), width
    else:
        y_at, y_stride = _array(out, "out", dtype, index, (rows, width))
    if rows and width:
        _call(lib, lib.fav_project_int4,
              INT4_ARGS(x_at, y_at, x_stride, y_stride, weight_at, scales_at, bias_at, kind, rows, depth, width, group),
              index)
    return out


def quantize_int4(weight, group):
    """4-bit codes and group scales of ``weight`` ``[out, depth]`` for ``project_int4``.

    Symmetric: a group's scale is its largest magnitude over 7 (1 for a group of
    zeros), codes round to nearest, ties to even.
    """
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError("weight must be a floating point tensor of shape [out, depth]")
    weight = weight.detach()
    width, depth = weight.shape
    if type(group) is not int or group < 32 or group % 32 or depth < 32 or depth % 32:
        raise ValueError("group and the depth must be positive multiples of 32")
    groups = -(-depth // group)
    w = torch.zeros((width, groups * group), dtype=_F32, device=weight.device)
    w[:, :depth] = weight
    w = w.view(width, groups, group)
    scales = w.abs().amax(2) / 7
    if not torch.isfinite(scales).all():
        raise ValueError("weight must contain only finite values")
    scales[scales == 0] = 1
    q = (torch.round(w / scales[:, :, None]).clamp(-7, 7) + 8).to(torch.uint8).view(width, -1)[:, :depth]
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), scales.contiguous()


def conv_state(slots, channels, taps, *, dtype=torch.bfloat16, device="cuda"):
    """A zeroed state pool of ``causal_conv``."""
    return torch.zeros((slots, 2, taps - 1, channels), dtype=dtype, device=device)


def scan_state(slots, channels, states, *, device="cuda"):
    """A zeroed state pool of ``selective_scan``."""
    return torch.zeros((slots, 2, states, channels), dtype=_F32, device=device)


class StreamSlots:
    """Read tables and fresh starts of a pool's slots, as the decoder keeps its own.

    One ``StreamSlots`` serves every layer of a model, since all layers of a
    step advance together: ``codes(slots)`` before the step, and
    ``commit(slots)`` once it has succeeded. A step that is not committed
    leaves every state as it was. Slots start afresh until their first commit
    and again after ``reset``. Codes are uploaded without waiting for the device;
    the upload is no part of a captured step, whose codes are written before its
    replay (``out``).
    """

    def __init__(self, slots, *, device="cuda"):
        if type(slots) is not int or not 1 <= slots <= _SLOTS:
            raise ValueError("slots must be a positive int, up to 2^29")
        self.device = torch.device(device)
        self._table = np.zeros(slots, np.int32)
        self._fresh = np.ones(slots, np.int32)

    def _checked(self, slots):
        index = np.asarray(slots)
        if index.size == 0:
            index = index.astype(np.int64)
        if index.ndim != 1 or index.dtype.kind not in "iu":
            raise ValueError("slots must be a sequence of ints")
        if index.size and (index.min() < 0 or index.max() >= len(self._table)):
            raise ValueError(f"slots must lie in [0, {len(self._table)})")
        if len(np.unique(index)) != index.size:
            raise ValueError("A slot may appear only once per step")
        return index

    def codes(self, slots, out=None):
        """The slot codes of a step over distinct ``slots``, on the device, in ``out`` if given."""
        index = self._checked(slots)
        if out is not None and not (isinstance(out, torch.Tensor) and out.dtype is _I32 and out.shape == index.shape
                                    and out.is_contiguous() and out.device.type == self.device.type):
            raise ValueError(f"out must be a contiguous int32 tensor of {index.size} elements on the slots' device")
        codes = torch.from_numpy(
            (index.astype(np.int32) << 2) | (self._fresh[index] * _FRESH) | self._table[index])
        if self.device.type == "cuda":
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("A capture would keep these codes for good; write the codes of a replay into "
                                   "the captured tensor before it (out=)")
            codes = codes.pin_memory()   # its allocator keeps the memory until the copy from it is done
        if out is None:
            return codes.to(self.device, non_blocking=True)
        return out.copy_(codes, non_blocking=True)

    def commit(self, slots):
        index = self._checked(slots)
        self._table[index] ^= 1
        self._fresh[index] = 0

    def reset(self, slots):
        self._fresh[self._checked(slots)] = 1
