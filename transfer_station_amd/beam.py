"""Python mirror of beam search's entry points (include/attn_flash.h): the continuations that go on, and the paged
cache's sequences following them. No counterpart in the reference."""
import ctypes

from ._lib import lib
from .attn import _addr
from .paged import _Struct

ATTN_BEAMS_MAX = 256
ATTN_BEAM_K_MAX = 64
ATTN_BEAM_V_MAX = 1 << 20
ATTN_REORDER_MAX = 32


class Beams(_Struct):
    """struct attn_beams: the logits (bits 16: bf16, 32: fp32) and scores of B entries' beams."""
    _fields_ = [("logits", ctypes.c_void_p), ("row", ctypes.c_int64), ("scores", ctypes.c_void_p),
                ("done", ctypes.c_void_p), ("bits", ctypes.c_int32), ("B", ctypes.c_int32),
                ("beams", ctypes.c_int32), ("V", ctypes.c_int32), ("K", ctypes.c_int32),
                ("done_token", ctypes.c_int32)]

    def __init__(self, logits, row, bits, B, beams, V, K, scores, done=None, done_token=0):
        super().__init__(_addr(logits), row, _addr(scores), _addr(done), bits, B, beams, V, K, done_token)


def attn_beam_scratch_bytes(beams):
    return lib().attn_beam_scratch_bytes(beams._at)


def attn_beam_select(beams, score, token, parent, scratch):
    """The K best continuations of each entry's beams: score (float32), token and parent (int32), [B][K] each."""
    lib().attn_beam_select(beams._at, _addr(score), _addr(token), _addr(parent), _addr(scratch))


def attn_kv_reorder(cache, parent, beams, tables=1):
    """Sequence b of the cache continues parent[b], a member of its group of `beams` sequences."""
    lib().attn_kv_reorder(cache._at, _addr(parent), int(beams), int(bool(tables)))
