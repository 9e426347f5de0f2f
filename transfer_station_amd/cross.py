"""Python mirror of cross attention's entry points (include/attn_flash.h): attention of ragged batches of rows to
encoder states of another length, with the log-sum-exp, and its gradients. No counterpart in the reference.

Device memory is given as DeviceBuffer or raw addresses, as everywhere in this package; Spans, CrossCall and Rows are
made once and kept for as long as their tensors live."""
import ctypes

from ._lib import lib
from .attn import _addr, parse_plan
from .paged import _Struct

ATTN_TOKEN_MAX = 1 << 22


class Spans(_Struct):
    """struct attn_spans: each sequence's rows of a token tensor of T rows, max at most (a bound). With len, sequence b
    has len[b] rows from start[b] on, else those up to start[b + 1]."""
    _fields_ = [("start", ctypes.c_void_p), ("len", ctypes.c_void_p), ("T", ctypes.c_int32),
                ("max", ctypes.c_int32)]

    def __init__(self, start, T, max, len=None):
        super().__init__(_addr(start), _addr(len), T, max)


class CrossCall(_Struct):
    """struct attn_cross_call: the rows and states of B sequences, their heads and the scale (0: 1/sqrt(D))."""
    _fields_ = [("q", Spans), ("k", Spans), ("B", ctypes.c_int32), ("Hq", ctypes.c_int32),
                ("Hkv", ctypes.c_int32), ("D", ctypes.c_int32), ("scale", ctypes.c_float)]

    def __init__(self, q, k, B, Hq, Hkv, D, scale=0.0):
        super().__init__(q, k, B, Hq, Hkv, D, scale)


def attn_cross_scratch_bytes(call):
    return lib().attn_cross_scratch_bytes(call._at)


def attn_cross_grad_scratch_bytes(call):
    return lib().attn_cross_grad_scratch_bytes(call._at)


def attn_cross(call, q, k, v, o, lse, scratch):
    """Attention of each sequence's rows over its states, o in bf16, and each row's log-sum-exp (lse may be None)."""
    lib().attn_cross(call._at, q._at, k._at, v._at, o._at, _addr(lse), _addr(scratch))


def attn_cross_grad(call, q, k, v, o, lse, d_o, dq, dk, dv, scratch):
    """The gradients of q, k and v from that of o, and from the o and lse that attn_cross left."""
    lib().attn_cross_grad(call._at, q._at, k._at, v._at, o._at, _addr(lse), d_o._at, dq._at, dk._at, dv._at,
                          _addr(scratch))


def attn_cross_plan(call, grad=False):
    """The kernels such a call launches, as attn_flash_plan gives them; nothing is launched."""
    buf = ctypes.create_string_buffer(4096)
    n = lib().attn_cross_plan(call._at, int(bool(grad)), buf, len(buf))
    if n < 0:
        raise RuntimeError("attn_cross_plan: the plan does not fit the buffer")
    return parse_plan(buf.value.decode())
