"""ctypes binding of ``libfav_cuda.so`` (declarations in ``include/fast_audiovae_cuda.h``).

Loading never falls back to anything: a missing or unloadable library raises.
"""
from __future__ import annotations

import ctypes as ct
import struct as pack
import threading
from pathlib import Path

import numpy as np

from . import weights as W

LIBRARY = Path(__file__).resolve().parent / "libfav_cuda.so"
ABI_VERSION = 1
SLOT_FLOATS = 161856
SLOT_STRIDE_FLOATS = 2 * SLOT_FLOATS + 64
NUM_COEFFICIENTS = 188

STATUS = {0: "FAV_OK", 1: "FAV_INVALID_ARGUMENT", 2: "FAV_UNSUPPORTED", 3: "FAV_OVERLAP",
          4: "FAV_SIZE_OVERFLOW", 5: "FAV_DEVICE_ERROR", 6: "FAV_TIMEOUT"}

_P = ct.c_void_p


def _struct(name, fields):
    """A ctypes structure from ``"type: name name ..."`` lines in the header's order."""
    kinds = {"ptr": ct.c_void_p, "i64": ct.c_int64, "size": ct.c_size_t, "f32": ct.c_float, "i32": ct.c_int32}
    return type(name, (ct.Structure,), {"_fields_": [
        (field, kinds[kind]) for kind, _, names in (line.partition(":") for line in fields)
        for field in names.split()]})


def _packer(struct):
    """``struct``'s C image from its fields' values in order, as bytes a call can be given (a
    third of the time that a ctypes structure takes to fill)."""
    letters = {ct.c_void_p: "P", ct.c_int64: "q", ct.c_size_t: "N", ct.c_float: "f", ct.c_int32: "i"}
    image = pack.Struct("@" + "".join(letters[kind] for _, kind in struct._fields_) + "0P")
    assert image.size == ct.sizeof(struct)
    return image.pack


# Argument structures of the stream operators (fav_conv_args and so on).
ConvArgs = _struct("ConvArgs", [
    "ptr: x y", "i64: x_stride y_stride", "ptr: weight bias state_pool slot_codes offsets status",
    "i32: type channels taps activation n length rows num_slots"])
ScanArgs = _struct("ScanArgs", [
    "ptr: x dt z b c y",
    "i64: x_stride dt_stride z_stride b_stride b_group_stride c_stride c_group_stride y_stride",
    "ptr: a d dt_bias state_pool slot_codes offsets status workspace", "size: workspace_bytes",
    "i32: type channels states groups softplus n length rows num_slots"])
NormArgs = _struct("NormArgs", [
    "ptr: x y", "i64: x_stride y_stride", "ptr: weight bias alpha reciprocal offsets status", "f32: eps",
    "i32: type channels groups activation n length rows"])
Int4Args = _struct("Int4Args", [
    "ptr: x y", "i64: x_stride y_stride", "ptr: weight scales bias", "i32: type rows depth out group"])

CONV_ARGS, SCAN_ARGS, NORM_ARGS, INT4_ARGS = map(_packer, (ConvArgs, ScanArgs, NormArgs, Int4Args))

# Every symbol the header declares, with its ctypes signature.
SIGNATURES = {
    "fav_abi_version": ([], ct.c_int32),
    "fav_last_error": ([], ct.c_char_p),
    "fav_status_string": ([ct.c_int32], ct.c_char_p),
    "fav_device_supported": ([], ct.c_int32),
    "fav_host_device_pointer": ([ct.c_void_p, ct.POINTER(ct.c_void_p)], ct.c_int32),
    "fav_plan_create": ([ct.POINTER(ct.POINTER(ct.c_float)), ct.c_int32, ct.c_int32, ct.POINTER(_P)], ct.c_int32),
    "fav_plan_destroy": ([_P], None),
    "fav_plan_bytes": ([_P], ct.c_size_t),
    "fav_state_pool_bytes": ([ct.c_int32], ct.c_size_t),
    "fav_step_workspace_bytes": ([ct.c_int32, ct.c_int32], ct.c_size_t),
    "fav_step": ([_P, _P, ct.c_int32, _P, ct.c_int32, ct.c_int32, _P, _P, _P, ct.c_size_t, _P, _P], ct.c_int32),
    "fav_debug_step_unfused": ([_P, _P, ct.c_int32, _P, ct.c_int32, ct.c_int32, _P, _P, _P, ct.c_size_t, _P, _P],
                               ct.c_int32),
    "fav_step_static": ([_P, _P, ct.c_int32, _P, ct.c_int32, ct.c_int32, _P, _P, _P, _P], ct.c_int32),
    "fav_batch_workspace_bytes": ([ct.c_int32, ct.c_int32], ct.c_size_t),
    "fav_plan_workspace_bytes": ([_P, ct.c_int32, ct.c_int32], ct.c_size_t),
    "fav_plan_batch_workspace_bytes": ([_P, ct.c_int32, ct.c_int32], ct.c_size_t),
    "fav_plan_precision": ([_P], ct.c_int32),
    "fav_decode_batch": ([_P, _P, ct.c_int32, ct.c_int32, ct.c_int32, _P, _P, ct.c_size_t, _P, _P], ct.c_int32),
    "fav_step_profile": ([_P, _P, ct.c_int32, _P, ct.c_int32, ct.c_int32, _P, _P, _P, ct.c_size_t, _P,
                          ct.POINTER(ct.c_float), _P], ct.c_int32),
    "fav_debug_step_layers": ([_P, _P, ct.c_int32, _P, ct.c_int32, ct.c_int32, _P, _P, ct.c_size_t, _P,
                               ct.c_int32, ct.POINTER(ct.c_void_p), _P], ct.c_int32),
    "fav_debug_step_gated": ([_P, _P, ct.c_int32, _P, ct.c_int32, ct.c_int32, _P, _P, _P, ct.c_size_t, _P,
                              ct.c_int32, ct.c_uint32, _P, _P], ct.c_int32),
    "fav_causal_conv": ([_P, _P], ct.c_int32),
    "fav_selective_scan": ([_P, _P], ct.c_int32),
    "fav_selective_scan_workspace_bytes": ([_P], ct.c_size_t),
    "fav_group_norm": ([_P, _P], ct.c_int32),
    "fav_project_int4": ([_P, _P], ct.c_int32),
    "fav_bind_tensors": ([_P, _P], ct.c_int32),
    "fav_causal_conv_tensors": ([ct.py_object] * 8 + [ct.c_int32], ct.c_int32),
    "fav_selective_scan_tensors": ([ct.py_object] * 14 + [ct.c_int32], ct.c_int64),
    "fav_group_norm_tensors": ([ct.py_object] * 8 + [ct.c_int32, ct.c_float, ct.c_int32], ct.c_int32),
    "fav_project_int4_tensors": ([ct.py_object] * 5 + [ct.c_int32], ct.c_int32),
    "fav_test_gemm": ([_P, ct.c_int32, ct.c_int32, _P, ct.c_int32, ct.c_int32, _P, _P], ct.c_int32),
    "fav_test_sine": ([_P, ct.c_int32, _P, _P], ct.c_int32),
}

_lock = threading.Lock()
_lib = None


class NativeError(RuntimeError):
    def __init__(self, status, message):
        super().__init__(f"{STATUS.get(status, status)}: {message}")
        self.status = status


def load_library(path=None):
    """Load (once) and type the CUDA library; raises if it is absent or mismatched."""
    global _lib
    with _lock:
        if _lib is not None and path is None:
            return _lib
        target = Path(path) if path else LIBRARY
        if not target.is_file():
            raise RuntimeError(f"CUDA decoder library {target} is not built; run fast_audiovae.build")
        lib = ct.CDLL(str(target))
        for name, (args, res) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.argtypes = args
            fn.restype = res
        if lib.fav_abi_version() != ABI_VERSION:
            raise RuntimeError("CUDA decoder ABI version mismatch")
        if path is None:
            _lib = lib
        return lib


def tensor_functions(tensor_type):
    """The entry points that read tensor objects themselves, as functions that are called with the
    interpreter's lock (which they give back while they launch); None when ``tensor_type`` has no DLPack 1.x C exchange interface."""
    lib = load_library()
    capsule = getattr(tensor_type, "__dlpack_c_exchange_api__", None)
    if capsule is None:
        return None
    pointer = ct.PYFUNCTYPE(ct.c_void_p, ct.py_object, ct.c_char_p)(("PyCapsule_GetPointer", ct.pythonapi))
    if lib.fav_bind_tensors(pointer(capsule, b"dlpack_exchange_api"), id(None)) != 0:
        return None
    held = ct.PyDLL(str(LIBRARY))
    for name in ("fav_causal_conv_tensors", "fav_selective_scan_tensors", "fav_group_norm_tensors",
                 "fav_project_int4_tensors"):
        fn = getattr(held, name)
        fn.argtypes, fn.restype = SIGNATURES[name]
    return held


def check(lib, status):
    if status != 0:
        raise NativeError(status, lib.fav_last_error().decode(errors="replace"))


def coefficient_list(weights):
    """The 188 coefficient arrays in the C ABI's canonical order (contiguous fp32)."""
    W.validate_weights(weights)
    names = list(W.weight_shapes())
    assert len(names) == NUM_COEFFICIENTS
    return [np.ascontiguousarray(weights[n], dtype=np.float32) for n in names]


class Plan:
    """Owns an ``fav_plan`` (immutable packed weights on the current device)."""

    def __init__(self, weights, precision=0):
        self.lib = load_library()
        arrays = coefficient_list(weights)
        self._keep = arrays
        ptrs = (ct.POINTER(ct.c_float) * len(arrays))(*[a.ctypes.data_as(ct.POINTER(ct.c_float)) for a in arrays])
        handle = ct.c_void_p()
        check(self.lib, self.lib.fav_plan_create(ptrs, len(arrays), precision, ct.byref(handle)))
        self.handle = handle
        self._keep = None

    @property
    def device_bytes(self):
        return int(self.lib.fav_plan_bytes(self.handle))

    def close(self):
        if getattr(self, "handle", None):
            self.lib.fav_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
