"""Attention sessions on the HIP backend: the new rows of many sequences over a
paged cache of keys and values.

An ``AttentionLayout`` is a layer's heads and types; ``HipAttentionSession`` holds
the pages of its layers (or the caller's) and runs, on the device, packed prompts
of several lengths, one row of each sequence, or trees of drafted tokens: what the
reference's step functions do one token at a time (llambda.lisp:5122-5167,
5951-6018).  Rows are those of the projection sessions around it, which may lie
side by side in one buffer.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import numpy as np

from . import native
from .hip_backend import HipBackendError, _check

# LLAMBDA_HIP_TYPE_*
TYPE_TAGS = {"f32": 0, "f16": 1, "bf16": 30}
# elements of the types on the host; numpy has no bf16, whose bits are taken
HOST_TYPES = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


@dataclass
class AttentionLayout:
    heads: int
    kv_heads: int
    head_dim: int
    scale: Optional[float] = None   # None: 1 / sqrt(head_dim)
    row_type: str = "f32"           # of q, k, v and the output
    cache_type: str = "f16"         # any below f32 rows, else the rows'


class HipAttentionSession:
    """`layers` layers' pages of `page_tokens` tokens, in device memory of the session's own
    (zeroed) or the caller's (key_pages_ptr, value_pages_ptr [layers][pages][kv_heads]
    [page_tokens][head_dim] of the cache's type); max_tokens and max_sequences bound a call."""

    def __init__(self, layout: AttentionLayout, *, pages: int, page_tokens: int = 64, max_context: int,
                 max_tokens: int = 4096, max_sequences: int = 1, layers: int = 1, key_pages_ptr: int = 0,
                 value_pages_ptr: int = 0):
        self.pointer = None
        self.layout = layout
        self.page_tokens = page_tokens
        for t in (layout.row_type, layout.cache_type):
            if t not in TYPE_TAGS:
                raise HipBackendError(f"HIP attention has no type {t!r}; they are {', '.join(TYPE_TAGS)}.")
        if layout.scale is not None and not np.float32(layout.scale) > 0:  # 0 is the default's
            raise HipBackendError(f"HIP attention scale {layout.scale} is not positive.")
        d = native.AttentionDesc()
        d.heads, d.kv_heads, d.head_dim = layout.heads, layout.kv_heads, layout.head_dim
        d.scale = 0.0 if layout.scale is None else layout.scale
        d.row_type, d.cache_type = TYPE_TAGS[layout.row_type], TYPE_TAGS[layout.cache_type]
        d.layers, d.page_tokens, d.pages, d.max_context = layers, page_tokens, pages, max_context
        d.max_tokens, d.max_sequences = max_tokens, max_sequences
        d.key_pages = key_pages_ptr or None
        d.value_pages = value_pages_ptr or None
        handle = ctypes.c_void_p()
        _check(native.lib().llambda_hip_attention_session_create(ctypes.byref(d), ctypes.byref(handle)),
               "HIP attention session creation")
        self.pointer = handle.value

    def close(self) -> None:
        if self.pointer:
            native.lib().llambda_hip_attention_session_destroy(self.pointer)
            self.pointer = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass

    def _live(self):
        if not self.pointer:
            raise HipBackendError("HIP attention session is closed.")
        return self.pointer

    def run_device(self, q_ptr: int, k_ptr: int, v_ptr: int, output_ptr: int, tokens: int, context_ptr: int,
                   table_ptr: int, sequences: int, *, offsets_ptr: int = 0, parents_ptr: int = 0, layer: int = 0,
                   q_stride: int = 0, k_stride: int = 0, v_stride: int = 0, output_stride: int = 0,
                   table_stride: int = 0, stream: int = 0) -> None:
        """Sequence i's rows [offsets[i], offsets[i + 1]) behind context[i] cached tokens (int32 lists
        on the device); no offsets: one row each.  parents: the rows are trees.  Strides in elements,
        0 = dense.  Next tokens of many sequences and long prompts are faster in calls of their own."""
        rows = native.AttentionRows(q_ptr or None, k_ptr or None, v_ptr or None, output_ptr or None,
                                    q_stride, k_stride, v_stride, output_stride)
        batch = native.AttentionBatch(tokens, sequences, offsets_ptr or None, context_ptr or None,
                                      table_ptr or None, table_stride, parents_ptr or None)
        _check(native.lib().llambda_hip_attention_session_run_device(
            self._live(), layer, ctypes.byref(rows), ctypes.byref(batch), stream or None), "HIP attention device run")

    def accept_device(self, context_ptr: int, table_ptr: int, paths_ptr: int, counts_ptr: int, sequences: int,
                      path_stride: int, *, table_stride: int = 0, stream: int = 0) -> None:
        """Move the keys and values of counts[i] accepted nodes, paths[i][0] < paths[i][1] < ..., of
        each sequence's tree behind its cached tokens, in all layers."""
        _check(native.lib().llambda_hip_attention_session_accept_device(
            self._live(), context_ptr or None, table_ptr or None, table_stride, paths_ptr or None, path_stride,
            counts_ptr or None, sequences, stream or None), "HIP attention accept")

    def sync(self, stream: int = 0) -> None:
        """Wait for `stream`; raises if the device refused sequences of a call."""
        _check(native.lib().llambda_hip_attention_session_sync(self._live(), stream or None), "HIP attention sync")

    def _rows(self, a, heads: int, kind: str, what: str) -> np.ndarray:
        a = np.asarray(a)
        if kind == "bf16" and a.dtype != np.uint16:
            raise HipBackendError(f"HIP attention {what} of bf16 are taken as their bits (uint16), not {a.dtype}.")
        a = np.ascontiguousarray(a, dtype=HOST_TYPES[kind])
        width = heads * self.layout.head_dim
        if a.size % width:
            raise HipBackendError(f"HIP attention {what} has {a.size} elements, not rows of {width}.")
        return a.reshape(-1, heads, self.layout.head_dim)

    @staticmethod
    def _whole(a, what: str, used: Optional[int] = None) -> np.ndarray:
        """Whole numbers as int32; the first `used` (all, if None) have to fit it, the others are not read."""
        a = np.asarray(a).reshape(-1)
        if a.size and a.dtype.kind not in "iu":
            raise HipBackendError(f"HIP attention {what} must be whole numbers, not {a.dtype}.")
        ends = np.iinfo(np.int32)
        far = (a[:used] < ends.min) | (a[:used] > ends.max)
        if far.any():
            raise HipBackendError(f"HIP attention {what} holds {a[:used][far][0]}, which does not fit 32 bits.")
        return np.ascontiguousarray(a, dtype=np.int32)

    def _table(self, table: Sequence[int], positions: int) -> np.ndarray:
        t = self._whole(table, "table", -(-max(positions, 0) // self.page_tokens))
        if positions > t.size * self.page_tokens:
            raise HipBackendError(f"HIP attention table of {t.size} pages does not hold {positions} tokens.")
        return t

    def run(self, q, k, v, table: Sequence[int], context: int = 0, *, parents: Optional[Sequence[int]] = None,
            layer: int = 0) -> np.ndarray:
        """Host rows q [tokens][heads][head_dim], k and v [tokens][kv_heads][head_dim] of one sequence
        whose pages are `table`, behind `context` cached tokens."""
        L = self.layout
        q, k, v = (self._rows(a, n, L.row_type, w) for a, n, w in
                   ((q, L.heads, "q"), (k, L.kv_heads, "k"), (v, L.kv_heads, "v")))
        if not len(q) == len(k) == len(v):
            raise HipBackendError(f"HIP attention has {len(q)}, {len(k)} and {len(v)} rows of q, k and v.")
        t = self._table(table, context + len(q))
        p = None
        if parents is not None:
            p = self._whole(parents, "parents")
            if p.size != len(q):
                raise HipBackendError(f"HIP attention has {p.size} parents of {len(q)} rows.")
        y = np.empty_like(q)
        _check(native.lib().llambda_hip_attention_session_run(
            self._live(), layer, q.ctypes.data, k.ctypes.data, v.ctypes.data, y.ctypes.data, len(q), context,
            t.ctypes.data, None if p is None else p.ctypes.data), "HIP attention run")
        return y

    def write(self, table: Sequence[int], first: int, keys, values, *, layer: int = 0) -> None:
        """Put keys and values [count][kv_heads][head_dim] at positions `first` and on."""
        L = self.layout
        k, v = (self._rows(a, L.kv_heads, L.cache_type, w) for a, w in ((keys, "keys"), (values, "values")))
        if len(k) != len(v):
            raise HipBackendError(f"HIP attention has {len(k)} rows of keys and {len(v)} of values.")
        t = self._table(table, first + len(k))
        _check(native.lib().llambda_hip_attention_session_write(
            self._live(), layer, t.ctypes.data, first, len(k), k.ctypes.data, v.ctypes.data), "HIP attention write")

    def read(self, table: Sequence[int], first: int, count: int, *, layer: int = 0) -> Tuple[np.ndarray, np.ndarray]:
        """Keys and values [count][kv_heads][head_dim] at positions `first` and on."""
        L = self.layout
        t = self._table(table, first + count)
        shape = (max(count, 0), L.kv_heads, L.head_dim)
        k, v = (np.empty(shape, dtype=HOST_TYPES[L.cache_type]) for _ in range(2))
        _check(native.lib().llambda_hip_attention_session_read(
            self._live(), layer, t.ctypes.data, first, count, k.ctypes.data, v.ctypes.data), "HIP attention read")
        return k, v
