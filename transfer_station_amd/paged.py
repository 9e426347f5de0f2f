"""Python mirror of the paged KV cache's entry points (include/attn_flash.h): appending tokens, reading rows
back, and attention over the cache, in bf16 or in 4 bits. No counterpart in the reference.

Device memory is given as DeviceBuffer or raw addresses, as everywhere in this package; KvCache, Rows and
Scores are made once and kept for as long as their tensors live. T, max_q and max_kv are bounds, which choose kernels and
cut the work; the header says what loose ones cost."""
import ctypes

from ._lib import lib
from .attn import _addr, parse_plan

ATTN_KV_BF16 = 16
ATTN_KV_FP4 = 4
ATTN_KV_PAGE_MIN = 16
ATTN_KV_PAGE_MAX = 256


class _Struct(ctypes.Structure):
    """A struct whose address is taken once: a call of a few microseconds makes no new pointers."""

    def __init__(self, *fields):
        super().__init__(*fields)
        self._at = ctypes.addressof(self)


class KvCache(_Struct):
    """struct attn_kv_cache: the pages, the table, the lengths and the starts of a call's sequences."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("table", ctypes.c_void_p),
                ("kv_len", ctypes.c_void_p), ("q_start", ctypes.c_void_p), ("B", ctypes.c_int32),
                ("table_cols", ctypes.c_int32), ("pages", ctypes.c_int32), ("page", ctypes.c_int32),
                ("Hkv", ctypes.c_int32), ("D", ctypes.c_int32), ("bits", ctypes.c_int32)]

    def __init__(self, k, v, table, kv_len, q_start, B, table_cols, pages, page, Hkv, D,
                 bits=ATTN_KV_BF16, k_scale=None, v_scale=None):
        super().__init__(_addr(k), _addr(v), _addr(k_scale), _addr(v_scale), _addr(table),
                         _addr(kv_len), _addr(q_start), B, table_cols, pages, page, Hkv, D, bits)


class Rows(_Struct):
    """struct attn_rows: a token tensor [T][heads][D] in bf16, strides in elements."""
    _fields_ = [("data", ctypes.c_void_p), ("token", ctypes.c_int64), ("head", ctypes.c_int64)]

    def __init__(self, data, token, head):
        super().__init__(_addr(data), token, head)


class Scores(_Struct):
    """struct attn_scores: scale (0: 1/sqrt(D)), softcap (0: none), slopes (device, [Hq], or None)."""
    _fields_ = [("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("slopes", ctypes.c_void_p)]

    def __init__(self, scale=0.0, softcap=0.0, slopes=None):
        super().__init__(scale, softcap, _addr(slopes))


def _at(s):
    return None if s is None else s._at


def attn_kv_append(cache, q, q_out, k, v, T, Hq, rope, rope_rows, rot, pairs=0, max_q=1):
    """Writes k and v of a call's tokens into the cache, k rotated, and the rotated q to q_out."""
    lib().attn_kv_append(cache._at, _at(q), _at(q_out), k._at, v._at, int(T), int(Hq), _addr(rope),
                         int(rope_rows), int(rot), int(bool(pairs)), int(max_q))


def attn_kv_read(cache, k, v, T, max_q=1):
    """A call's rows of the cache to k and v, in bf16."""
    lib().attn_kv_read(cache._at, k._at, v._at, int(T), int(max_q))


def attn_paged(cache, q, o, T, Hq, causal, scores, max_q, max_kv, scratch):
    """Attention of a call's rows over their sequences' caches. Stream-ordered; scratch is an attn_flash
    scratch of the cache's D."""
    lib().attn_paged(cache._at, q._at, o._at, int(T), int(Hq), int(bool(causal)), _at(scores), int(max_q),
                     int(max_kv), _addr(scratch))


def attn_paged_plan(cache, T, Hq, causal, scores, max_q, max_kv):
    """The kernels such a call launches, as attn_flash_plan gives them; nothing is launched."""
    buf = ctypes.create_string_buffer(4096)
    n = lib().attn_paged_plan(cache._at, int(T), int(Hq), int(bool(causal)), _at(scores), int(max_q),
                              int(max_kv), buf, len(buf))
    if n < 0:
        raise RuntimeError("attn_paged_plan: the plan does not fit the buffer")
    return parse_plan(buf.value.decode())
