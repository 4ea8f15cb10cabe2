"""Paged key/value cache over the C ABI: rotary embedding with the append (16 bits, or 8 or 4 as it is written), reading the cache
back, and attention of new tokens over it, for batches of sequences, prompts and single tokens.

The one-token operators of :mod:`mlxl3_b200.decoder` (``rope_append``, ``attention_decode``) work on a cache
[kv_heads, max_ctx, head_dim]; that is a pool of one page of ``max_ctx`` rows here.  All pointers are device pointers, calls allocate
nothing and can be recorded into a graph; rows, lengths and pages are read on the device.
"""
from __future__ import annotations

import ctypes
import math
from ctypes import byref, c_float, c_int, c_int64, c_size_t, c_void_p

import numpy as np

from . import _lib
from ._lib import B200Exl3Error, F16
from .linear import new_workspace
from .runtime import DEFAULT_STREAM, DeviceBuffer, Stream


class KvCache(ctypes.Structure):
    """``b200exl3_kv_cache``: a pool of ``pages`` pages of ``page_size`` tokens.  Without pointers it owns its memory (zeroed)."""
    _fields_ = [("d_k", c_void_p), ("d_v", c_void_p), ("d_k_scale", c_void_p), ("d_v_scale", c_void_p), ("pages", c_int64),
                ("page_size", c_int), ("kv_heads", c_int), ("head_dim", c_int), ("dtype", c_int), ("bits", c_int)]

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: int = F16, bits: int = 16, d_k: int = 0, d_v: int = 0,
                 d_k_scale: int = 0, d_v_scale: int = 0):
        self._owned = []
        if not d_k and not d_v:
            vectors = pages * kv_heads * page_size
            for nbytes in [vectors * head_dim * bits // 8] * 2 + [vectors * 4] * (2 if bits != 16 else 0):
                buf = DeviceBuffer(nbytes)
                buf.fill(0)
                self._owned.append(buf)
            DEFAULT_STREAM.sync()                # calls on other streams do not wait for it
            d_k, d_v, d_k_scale, d_v_scale = ([b.ptr for b in self._owned] + [0, 0])[:4]
        super().__init__(d_k, d_v, d_k_scale, d_v_scale, pages, page_size, kv_heads, head_dim, dtype, bits)

    @property
    def bytes_per_token(self) -> int:
        return 2 * self.kv_heads * (self.head_dim * self.bits // 8 + (4 if self.bits != 16 else 0))


class KvBatch(ctypes.Structure):
    """``b200exl3_kv_batch``: device arrays ``row_start [batch + 1]``, ``length [batch]`` and ``page_table [batch, table_width]`` (int32),
    and how many rows the row buffers have."""
    _fields_ = [("d_row_start", c_void_p), ("d_length", c_void_p), ("d_page_table", c_void_p), ("rows", c_int64), ("batch", c_int),
                ("table_width", c_int)]

    def __init__(self, d_row_start: int, d_length: int, d_page_table: int, batch: int, table_width: int, rows: int):
        super().__init__(d_row_start, d_length, d_page_table, rows, batch, table_width)


class Rope(ctypes.Structure):
    """``b200exl3_rope``: ``d_turns`` holds ``rotated / 2`` float64 (``rope_turns``)."""
    _fields_ = [("d_turns", c_void_p), ("rotated", c_int), ("interleaved", c_int), ("magnitude", c_float)]

    def __init__(self, d_turns: int, rotated: int, interleaved: bool = False, magnitude: float = 1.0):
        super().__init__(d_turns, rotated, int(interleaved), magnitude)


def rope_turns(rotated: int, theta: float, stretch: float = 1.0, low_freq: float = 0.0, high_freq: float = 0.0, original_ctx: int = 0) -> np.ndarray:
    """Turns per position of every rotated pair, theta^(-2j / rotated) / 2 pi in float64.  ``stretch`` > 1 reaches ``stretch`` times as far:
    every frequency is divided by it, or, with ``original_ctx``, only those that turn fewer than ``low_freq`` times in the original context;
    those that turn more than ``high_freq`` times stay, and between the two the division fades in."""
    if rotated <= 0 or rotated % 2 or theta <= 1.0 or stretch <= 0.0:
        raise B200Exl3Error("invalid rotary frequencies")
    turns = theta ** (-2.0 * np.arange(rotated // 2, dtype=np.float64) / rotated) / (2.0 * math.pi)
    if not original_ctx:
        return turns / stretch
    if not high_freq > low_freq:
        raise B200Exl3Error("invalid rotary frequencies")
    keep = np.clip((turns * original_ctx - low_freq) / (high_freq - low_freq), 0.0, 1.0)
    return turns * (keep + (1.0 - keep) / stretch)


def append(cache: KvCache, batch: KvBatch, d_k: int, d_v: int, rope: Rope | None = None, d_q: int = 0, heads: int = 0, d_q_out: int = 0,
           q_stride: int = 0, q_out_stride: int = 0, k_stride: int = 0, v_stride: int = 0, stream: Stream = DEFAULT_STREAM) -> None:
    """Rotates q (into ``d_q_out``, which may be ``d_q``) and k by their positions and writes k and v to the cache.  Strides are elements
    from row to row, 0 for rows without gaps."""
    _lib.call("b200exl3_kv_append", byref(cache), byref(batch), None if rope is None else byref(rope), d_q, q_stride, heads, d_q_out,
              q_out_stride, d_k, k_stride, d_v, v_stride, stream.handle)


def read(cache: KvCache, batch: KvBatch, dtype: int, d_k: int, d_v: int, stream: Stream = DEFAULT_STREAM) -> None:
    """Keys and values of the batch's rows, [rows, kv_heads, head_dim] in ``dtype``; either pointer may be 0."""
    _lib.call("b200exl3_kv_read", byref(cache), byref(batch), dtype, d_k, d_v, stream.handle)


def attention_workspace_bytes(cache: KvCache, heads: int, max_new: int) -> int:
    out = c_size_t()
    _lib.call("b200exl3_kv_attention_workspace_bytes", byref(cache), heads, max_new, byref(out))
    return out.value


def new_attention_workspace(cache: KvCache, batch: KvBatch, heads: int, max_new: int = 0) -> DeviceBuffer:
    """Scratch of ``attention`` for batches of up to ``max_new`` rows per sequence (0: all rows of ``batch``)."""
    return new_workspace(attention_workspace_bytes(cache, heads, max_new or batch.rows))


def attention(cache: KvCache, batch: KvBatch, d_q: int, heads: int, scale: float, d_out: int, workspace: DeviceBuffer, max_new: int = 0,
              window: int = 0, q_stride: int = 0, out_stride: int = 0, stream: Stream = DEFAULT_STREAM) -> None:
    """softmax(q k^T * scale) v of every row over the tokens up to its own; with ``window`` the last ``window`` of them.  ``max_new`` bounds
    the rows of one sequence (1 for a step of single tokens)."""
    _lib.call("b200exl3_kv_attention", byref(cache), byref(batch), d_q, q_stride, heads, scale, window, max_new, d_out, out_stride,
              workspace.ptr, workspace.nbytes, stream.handle)
