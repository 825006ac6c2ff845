"""The argument structs of csrc/include/tcpxb/train.h, for calls of the C entries themselves."""
import ctypes

from nccl_plugin_gpudirecttcpx_b200.utils import native

_vp, _i32, _i64, _f32, _f64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_double


def _heads(*names):
    return [f for n in names for f in ((n, _vp), (n + "_b", _i64), (n + "_s", _i64), (n + "_h", _i64))]


def _all(kind, names):
    return [(n, kind) for n in names.split()]


class Attention(ctypes.Structure):
    _fields_ = (_heads("q", "k", "v") + _all(_vp, "out lse") + _heads("dout") + _all(_vp, "dq dk dv delta key_lengths") +
                _all(_i32, "b sq sk heads kv_heads d") + [("scale", _f32)] + _all(_i32, "causal dtype device") + [("status", _vp)])


class NormRope(ctypes.Structure):
    _fields_ = (_heads("q", "k") + _all(_vp, "wq wk cos sin pos q_out k_out") + _heads("dq_out", "dk_out") + _all(_vp, "dq dk dwq dwk partial") +
                _all(_i32, "b s heads kv_heads d positions") + [("eps", _f32)] + _all(_i32, "dtype device"))


class AdamwTensor(ctypes.Structure):
    _fields_ = _all(_vp, "p g m v m_scale v_scale master step") + [("n", _i64)]


class Adamw(ctypes.Structure):
    _fields_ = (_all(_f64, "lr beta1 beta2 eps weight_decay") + [("grad_norm", _vp), ("max_norm", _f32)] +
                _all(_i32, "compute_norm state_bits dtype device") + [("scratch", _vp)])


def library():
    lib = native.load("libtcpxb_train.so")
    lib.tcpxb_train_last_error.restype = ctypes.c_char_p
    for name, *args in (("attention_forward", _vp, _vp), ("attention_backward", _vp, _vp), ("norm_rope_forward", _vp, _vp), ("norm_rope_backward", _vp, _vp),
                        ("adamw_step", _vp, _i32, _vp, _vp), ("grad_norm", _vp, _i32, _i32, _i32, _vp, _vp, _vp)):
        getattr(lib, "tcpxb_" + name).argtypes = args
    return lib
