"""ctypes view of the linear attention of include/rxmet_b200_mixer.h (test infrastructure)."""
import ctypes as C

from rx_met_b200 import _cabi


class Heads(C.Structure):
    """``rxmet_head_tensor``."""
    _fields_ = [("data", C.c_void_p), ("stride_b", C.c_int64), ("stride_t", C.c_int64), ("stride_h", C.c_int64), ("heads", C.c_int32)]

    @classmethod
    def of(cls, t):
        return cls(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2), t.shape[2])


class Problem(C.Structure):
    """``rxmet_decayed_attention``."""
    _fields_ = [(n, C.c_int32) for n in ("batch", "tokens", "heads", "key_dim", "value_dim", "type")] + [(n, Heads) for n in "qkv"] + \
        [("log_decay", C.c_void_p), ("lengths", C.c_void_p), ("scale", C.c_float)]


def library():
    lib = _cabi.load_library()
    lib.rxmet_last_error.restype = C.c_char_p
    lib.rxmet_decayed_attention_workspace_bytes.restype = C.c_size_t
    return lib
