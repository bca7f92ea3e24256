"""include/afc_ops.h for ctypes: what a host program without torch binds (tests/test_ops.py checks it against the header)."""
import ctypes as C

from rlfluidcontrol_amd import ops

SYMBOLS = ["afc_ops_last_error", "afc_conv", "afc_conv_grad", "afc_conv_workspace", "afc_conv_step", "afc_scan", "afc_scan_grad",
           "afc_scan_workspace", "afc_scan_step", "afc_clip", "afc_clip_workspace"]


class Seq(C.Structure):
    """struct afc_seq"""
    _fields_ = [("data", C.c_void_p), ("stride_batch", C.c_int64), ("stride_length", C.c_int64), ("stride_group", C.c_int64)]


class ConvArgs(C.Structure):
    """struct afc_conv_args"""
    _fields_ = [("device", C.c_int32), ("dtype", C.c_int32), ("taps", C.c_int32), ("silu", C.c_int32),
                ("batch", C.c_int64), ("length", C.c_int64), ("width", C.c_int64), ("x", Seq), ("y", Seq),
                ("weight", C.c_void_p), ("bias", C.c_void_p), ("initial_state", C.c_void_p), ("final_state", C.c_void_p),
                ("lengths", C.c_void_p), ("dy", Seq), ("dfinal_state", C.c_void_p), ("dx", Seq), ("dweight", C.c_void_p),
                ("dbias", C.c_void_p), ("dinitial_state", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


class ScanArgs(C.Structure):
    """struct afc_scan_args"""
    _fields_ = [("device", C.c_int32), ("dtype", C.c_int32), ("softplus", C.c_int32), ("state", C.c_int32),
                ("batch", C.c_int64), ("length", C.c_int64), ("width", C.c_int64), ("groups", C.c_int64),
                ("x", Seq), ("dt", Seq), ("b", Seq), ("c", Seq), ("z", Seq), ("y", Seq), ("a", C.c_void_p), ("d", C.c_void_p),
                ("dt_bias", C.c_void_p), ("initial_state", C.c_void_p), ("final_state", C.c_void_p), ("lengths", C.c_void_p),
                ("checkpoints", C.c_void_p), ("dy", Seq), ("dfinal_state", C.c_void_p), ("dx", Seq), ("ddt", Seq), ("db", Seq),
                ("dc", Seq), ("dz", Seq), ("da", C.c_void_p), ("dd", C.c_void_p), ("ddt_bias", C.c_void_p),
                ("dinitial_state", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


class ClipArgs(C.Structure):
    """struct afc_clip_args"""
    _fields_ = [("device", C.c_int32), ("count", C.c_int32), ("inp", C.c_void_p), ("out", C.c_void_p), ("numel", C.c_void_p),
                ("in_dtype", C.c_void_p), ("out_dtype", C.c_void_p), ("max_norm", C.c_float), ("norm", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


def load():
    L = C.CDLL(ops.LIB_PATH)
    L.afc_ops_last_error.restype = C.c_char_p
    u64 = C.POINTER(C.c_uint64)
    for f in ("afc_conv", "afc_conv_grad", "afc_conv_step"):
        getattr(L, f).argtypes = [C.POINTER(ConvArgs), C.c_void_p]
    for f in ("afc_scan", "afc_scan_grad", "afc_scan_step"):
        getattr(L, f).argtypes = [C.POINTER(ScanArgs), C.c_void_p]
    L.afc_clip.argtypes = [C.POINTER(ClipArgs), C.c_void_p]
    L.afc_conv_workspace.argtypes = [C.POINTER(ConvArgs), u64]
    L.afc_scan_workspace.argtypes = [C.POINTER(ScanArgs), u64, u64, u64]
    L.afc_clip_workspace.argtypes = [C.POINTER(ClipArgs), u64]
    return L
