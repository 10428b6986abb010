"""svox_amd.csrc.network -- the ctypes mirror of include/svox_network.h and the loader of libsvox_network.so.

The calls of svox_amd.network are made in native code (network_shim.cpp); the signatures here are what a caller of the C ABI
binds, and what the tests compare with the header.  The reference has no such operators.
"""
import ctypes
import os

HERE = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(HERE, "libsvox_network.so")

ABI_VERSION = 1   # SVOX_NETWORK_ABI_VERSION of include/svox_network.h

c_void_p, c_int32, c_int64, c_float, c_double = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_double


class ClipTensorC(ctypes.Structure):
    _fields_ = [("from_", c_void_p), ("to", c_void_p), ("count", c_int64), ("dtype", c_int32)]


class RotateHeadsC(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("k", c_void_p), ("q_weight", c_void_p), ("k_weight", c_void_p), ("positions", c_void_p), ("frequencies", c_void_p),
                ("rows", c_int64), ("q_stride", c_int64), ("q_head", c_int64), ("k_stride", c_int64), ("k_head", c_int64), ("heads", c_int32),
                ("kv_heads", c_int32), ("dim", c_int32), ("rotated", c_int32), ("axes", c_int32), ("interleaved", c_int32), ("dtype", c_int32),
                ("position_type", c_int32), ("eps", c_float)]


class AttentionC(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("k", c_void_p), ("v", c_void_p), ("offsets", c_void_p), ("key_offsets", c_void_p), ("queries", c_int64),
                ("keys", c_int64), ("sequences", c_int64), ("q_stride", c_int64), ("q_head", c_int64), ("k_stride", c_int64), ("k_head", c_int64),
                ("v_stride", c_int64), ("v_head", c_int64), ("heads", c_int32), ("kv_heads", c_int32), ("dim", c_int32), ("dtype", c_int32),
                ("wide_offsets", c_int32), ("causal", c_int32), ("scale", c_float)]


class AttentionGradsC(ctypes.Structure):
    _fields_ = [("out", c_void_p), ("lse", c_void_p), ("rest", c_void_p), ("grad", c_void_p), ("grad_stride", c_int64), ("grad_head", c_int64), ("q", c_void_p),
                ("k", c_void_p), ("v", c_void_p)]


P = ctypes.POINTER

# name -> (restype, argtypes); the entry points of include/svox_network.h
SIGNATURES = {
    "svox_network_abi_version": (ctypes.c_int, []),
    "svox_network_last_error": (ctypes.c_char_p, []),
    "svox_clip_norm": (ctypes.c_int, [P(ClipTensorC), c_int64, c_double, c_void_p, c_void_p, c_int64, c_void_p]),
    "svox_clip_norm_workspace_bytes": (c_int64, [P(ClipTensorC), c_int64]),
    "svox_rotate_heads": (ctypes.c_int, [P(RotateHeadsC), c_void_p, c_void_p, c_void_p]),
    "svox_rotate_heads_backward": (
        ctypes.c_int, [P(RotateHeadsC), c_void_p, c_void_p, P(c_int64), c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "svox_rotate_heads_workspace_bytes": (c_int64, [P(RotateHeadsC), c_int32]),
    "svox_attention": (ctypes.c_int, [P(AttentionC), c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "svox_attention_backward": (ctypes.c_int, [P(AttentionC), P(AttentionGradsC), c_void_p, c_int64, c_void_p]),
    "svox_attention_workspace_bytes": (c_int64, [P(AttentionC), c_int32]),
}

_lib = None
_native = None


def load_library():
    """libsvox_network.so with its argument types (once).  Raises if it is not built, or built from other sources."""
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
        if lib.svox_network_abi_version() != ABI_VERSION:
            raise RuntimeError(f"{LIB_PATH} has ABI version {lib.svox_network_abi_version()}, this package expects {ABI_VERSION}: "
                               "build it again")
        _lib = lib
    return _lib


def native():
    """The extension module network_shim.cpp is built into, bound to the library.  Raises if it is not built."""
    global _native
    if _native is None:
        load_library()
        try:
            from .. import _network_shim
        except ImportError as e:
            raise RuntimeError(f"the host extension of svox_amd.csrc.network cannot be loaded ({e}): build it "
                               "(run `python -m svox_amd.csrc.build`)") from e
        _network_shim.init(LIB_PATH)
        _native = _network_shim
    return _native
