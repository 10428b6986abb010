"""svox_amd.csrc.decoder -- the ctypes mirror of include/svox_decoder.h and the loader of libsvox_decoder.so.

The calls of svox_amd.decoder are made in native code (decoder_shim.cpp); the signatures here are what a caller of the C ABI
binds, and what the tests compare with the header.  The reference has no such operators.
"""
import ctypes
import os

HERE = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(HERE, "libsvox_decoder.so")

ABI_VERSION = 1   # SVOX_DECODER_ABI_VERSION of include/svox_decoder.h
F32, F16, BF16 = 0, 1, 2
ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}

c_void_p, c_int32, c_int64, c_float = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class LayerNormC(ctypes.Structure):
    _fields_ = [("x", c_void_p), ("weight", c_void_p), ("bias", c_void_p), ("rows", c_int64), ("x_stride", c_int64),
                ("dim", c_int32), ("dtype", c_int32), ("eps", c_float)]


class GatedFfnC(ctypes.Structure):
    _fields_ = [("x", c_void_p), ("w_gate", c_void_p), ("w_up", c_void_p), ("w_down", c_void_p), ("b_gate", c_void_p),
                ("b_up", c_void_p), ("b_down", c_void_p), ("residual", c_void_p), ("rows", c_int64), ("x_stride", c_int64),
                ("residual_stride", c_int64), ("dim", c_int32), ("hidden", c_int32), ("out", c_int32), ("dtype", c_int32),
                ("activation", c_int32)]


class GatedFfnGradsC(ctypes.Structure):
    _fields_ = [("x", c_void_p), ("w_gate", c_void_p), ("w_up", c_void_p), ("w_down", c_void_p), ("b_gate", c_void_p),
                ("b_up", c_void_p), ("b_down", c_void_p)]


P = ctypes.POINTER

# name -> (restype, argtypes); the entry points of include/svox_decoder.h
SIGNATURES = {
    "svox_decoder_abi_version": (ctypes.c_int, []),
    "svox_decoder_last_error": (ctypes.c_char_p, []),
    "svox_layer_norm": (ctypes.c_int, [P(LayerNormC), c_void_p, c_void_p, c_void_p]),
    "svox_layer_norm_backward": (
        ctypes.c_int, [P(LayerNormC), c_void_p, c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "svox_layer_norm_workspace_bytes": (c_int64, [P(LayerNormC), c_int32]),
    "svox_gated_ffn": (ctypes.c_int, [P(GatedFfnC), c_void_p, c_void_p, c_int64, c_void_p]),
    "svox_gated_ffn_backward": (
        ctypes.c_int, [P(GatedFfnC), c_void_p, c_int64, P(GatedFfnGradsC), c_void_p, c_int64, c_void_p]),
    "svox_gated_ffn_workspace_bytes": (c_int64, [P(GatedFfnC), c_int32]),
}

_lib = None
_native = None


def load_library():
    """libsvox_decoder.so with its argument types (once).  Raises if it is not built, or built from other sources."""
    global _lib
    if _lib is None:
        import torch  # noqa: F401  (loads the HIP runtime the library binds to)
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: the HIP extension has not been built "
                               "(run `python -m svox_amd.csrc.build`); there is no CPU fallback")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (restype, argtypes) in SIGNATURES.items():
            fn = getattr(lib, name, None)
            if fn is None:
                raise RuntimeError(f"{LIB_PATH} does not export {name}: it was built from other sources, build it again")
            fn.restype, fn.argtypes = restype, argtypes
        if lib.svox_decoder_abi_version() != ABI_VERSION:
            raise RuntimeError(f"{LIB_PATH} has ABI version {lib.svox_decoder_abi_version()}, this package expects {ABI_VERSION}: "
                               "build it again")
        _lib = lib
    return _lib


def native():
    """The extension module decoder_shim.cpp is built into, bound to the library.  Raises if it is not built."""
    global _native
    if _native is None:
        load_library()
        try:
            from .. import _decoder_shim
        except ImportError as e:
            raise RuntimeError(f"the host extension of svox_amd.csrc.decoder cannot be loaded ({e}): build it "
                               "(run `python -m svox_amd.csrc.build`)") from e
        _decoder_shim.init(LIB_PATH)
        _native = _decoder_shim
    return _native
