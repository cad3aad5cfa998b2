"""Token sampling on the device: the host side of llambda_hip_sampler_*.

Mirrors the reference's ``sample-token-id-from-logits`` (llambda.lisp:1272-1317)
keyword for keyword -- history, repetition-penalty (1.15), top-k (40, NIL ->
40), top-p (0.95, NIL -> 0.95), temperature (1.0) and an explicit
random-value in [0, 1) -- and its argument errors.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np

from . import native

DEFAULT_TOP_K = 40      # llambda.lisp:32
DEFAULT_TOP_P = 0.95    # llambda.lisp:33


class SamplingError(RuntimeError):
    pass


def _params(history, repetition_penalty, top_k, top_p, temperature, random_value, keep):
    p = native.Sampling()
    if history is not None and len(history):
        h = np.ascontiguousarray(history, dtype=np.int64)
        keep.append(h)
        p.history, p.history_count = h.ctypes.data, h.size
    p.repetition_penalty = repetition_penalty
    p.top_k = DEFAULT_TOP_K if top_k is None else int(top_k)
    p.top_p = DEFAULT_TOP_P if top_p is None else float(top_p)
    p.temperature = temperature
    p.random_value = random_value
    return p


class HipSampler:
    """Device scratch for logits rows of up to `vocab` entries."""

    def __init__(self, vocab: int):
        handle = ctypes.c_void_p()
        if native.lib().llambda_hip_sampler_create(vocab, ctypes.byref(handle)) != 0:
            raise SamplingError(native.last_error())
        self._h = handle
        self.vocab = vocab

    def close(self) -> None:
        if getattr(self, "_h", None):
            native.lib().llambda_hip_sampler_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass

    def sample(self, logits, *, random_value: float, history: Optional[Sequence[int]] = None,
               repetition_penalty: float = 1.15, top_k: Optional[int] = DEFAULT_TOP_K,
               top_p: Optional[float] = DEFAULT_TOP_P, temperature: float = 1.0,
               device_count: Optional[int] = None) -> int:
        """logits: a host array, or a device pointer (int) with device_count
        entries.  The logits are not modified."""
        keep = []
        p = _params(history, repetition_penalty, top_k, top_p, temperature, random_value, keep)
        tok = ctypes.c_int64()
        if isinstance(logits, int):
            ptr, n, dev = logits, int(device_count), 1
        else:
            a = np.ascontiguousarray(logits, dtype=np.float32)
            keep.append(a)
            ptr, n, dev = a.ctypes.data, a.size, 0
        if native.lib().llambda_hip_sampler_sample(self._h, ptr, n, dev, ctypes.byref(p),
                                                   ctypes.byref(tok)) != 0:
            raise SamplingError(native.last_error())
        return tok.value

    def sample_session(self, session, *, random_value: float, history=None,
                       repetition_penalty: float = 1.15, top_k=DEFAULT_TOP_K,
                       top_p=DEFAULT_TOP_P, temperature: float = 1.0) -> int:
        """Sample from a HipLlamaSession's own logits (after step_device with
        logits_ptr=0)."""
        keep = []
        p = _params(history, repetition_penalty, top_k, top_p, temperature, random_value, keep)
        tok = ctypes.c_int64()
        if native.lib().llambda_hip_llama_session_sample(session._h, self._h, ctypes.byref(p),
                                                         ctypes.byref(tok)) != 0:
            raise SamplingError(native.last_error())
        return tok.value


def _per_row(value, rows: int, dtype) -> np.ndarray:
    """One number or one per row as `rows` of `dtype` (int32: whole numbers only; those beyond it are its ends)."""
    v = np.asarray(value)
    if np.dtype(dtype) == np.int32:
        if v.dtype.kind not in "iubf" or (v.dtype.kind == "f" and not np.all(np.floor(v) == v)):
            raise SamplingError(f"TOP-K must be whole numbers, got {value}.")
        ends = np.iinfo(np.int32)
        v = v.astype(np.float64 if v.dtype.kind == "f" else np.uint64 if v.dtype.kind == "u" else np.int64)
        v = np.minimum(v if v.dtype.kind == "u" else np.maximum(v, ends.min), ends.max)
    return np.ascontiguousarray(np.broadcast_to(v.astype(dtype), (rows,)))


def _random_per_row(value, rows: int) -> np.ndarray:
    """Numbers in [0, 1) in float32: those of more digits that would round to 1 become the largest below it."""
    v = np.asarray(value, dtype=np.float64)
    return _per_row(np.where(v < 1, np.minimum(v, 1 - 2.0 ** -24), v), rows, np.float32)


class HipBatchSampler:
    """One token per row of a batch of logits (llambda_hip_batch_sampler_*): temperature, top-k,
    top-p and min-p of each row's own, from given random numbers, in 64 bits."""

    def __init__(self, vocab: int, max_rows: int):
        self._h = None
        handle = ctypes.c_void_p()
        if native.lib().llambda_hip_batch_sampler_create(vocab, max_rows, ctypes.byref(handle)) != 0:
            raise SamplingError(native.last_error())
        self._h = handle
        self.vocab = vocab
        self.max_rows = max_rows

    def close(self) -> None:
        if getattr(self, "_h", None):
            native.lib().llambda_hip_batch_sampler_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass

    def sample_device(self, logits_ptr: int, rows: int, tokens_ptr: int, random_ptr: int, *,
                      temperature_ptr: int = 0, top_k_ptr: int = 0, top_p_ptr: int = 0,
                      min_p_ptr: int = 0, count: Optional[int] = None, stream: int = 0) -> None:
        """Device pointers: logits [rows][count] (the vocabulary by default), int32 tokens, float32
        parameters (int32 top-k) of each row, 0 = the default for all.  Not waited for."""
        p = native.BatchSampling(temperature_ptr or None, top_k_ptr or None, top_p_ptr or None,
                                 min_p_ptr or None, random_ptr or None)
        if native.lib().llambda_hip_batch_sampler_sample_device(
                self._h, logits_ptr or None, self.vocab if count is None else count, rows,
                ctypes.byref(p), tokens_ptr or None, stream or None) != 0:
            raise SamplingError(native.last_error())

    def sample(self, logits, *, random_value, temperature=None, top_k=None, top_p=None,
               min_p=None) -> np.ndarray:
        """Tokens (int64) of host logits [rows][count]; a parameter is one number or one per row."""
        a = np.ascontiguousarray(logits, dtype=np.float32)
        if a.ndim != 2:
            raise SamplingError(f"logits have {a.ndim} dimensions, not 2")
        rows = a.shape[0]
        keep = []

        def each(v):
            if v is None:
                return None
            keep.append(v)
            return v.ctypes.data

        def optional(v, dtype=np.float32):
            return each(None if v is None else _per_row(v, rows, dtype))

        p = native.BatchSampling(optional(temperature), optional(top_k, np.int32), optional(top_p), optional(min_p),
                                 each(_random_per_row(random_value, rows)))
        out = np.empty(rows, dtype=np.int64)
        if native.lib().llambda_hip_batch_sampler_sample(self._h, a.ctypes.data, a.shape[1], rows,
                                                         ctypes.byref(p), out.ctypes.data) != 0:
            raise SamplingError(native.last_error())
        return out


@dataclass
class TokenScores:
    """Of each row: natural logarithms of the given tokens' probabilities, the entropy, and the most likely tokens
    with their log probabilities (-1, -inf where there are no more)."""
    log_probs: np.ndarray       # float32 [rows][givens]
    entropy: np.ndarray         # float32 [rows]
    top_tokens: np.ndarray      # int32 [rows][top]
    top_log_probs: np.ndarray   # float32 [rows][top]


class HipTokenScorer:
    """Log probabilities of given tokens, entropy and top alternatives of rows of logits
    (llambda_hip_token_scorer_*)."""

    def __init__(self, vocab: int, max_rows: int, max_top: int = 0):
        self._h = None
        for name, value in (("vocab", vocab), ("max_rows", max_rows), ("max_top", max_top)):
            if value < 0:
                raise SamplingError(f"{name} {value} is negative")
        handle = ctypes.c_void_p()
        if native.lib().llambda_hip_token_scorer_create(vocab, max_rows, max_top, ctypes.byref(handle)) != 0:
            raise SamplingError(native.last_error())
        self._h = handle
        self.vocab = vocab
        self.max_rows = max_rows
        self.max_top = max_top

    def close(self) -> None:
        if getattr(self, "_h", None):
            native.lib().llambda_hip_token_scorer_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass

    def score_device(self, logits_ptr: int, rows: int, *, given_ptr: int = 0, given: int = 0, top: int = 0,
                     log_probs_ptr: int = 0, entropy_ptr: int = 0, top_tokens_ptr: int = 0,
                     top_log_probs_ptr: int = 0, count: Optional[int] = None, stride: int = 0,
                     stream: int = 0) -> None:
        """Device pointers: logits [rows][count] (the vocabulary by default), stride elements from row to row (0:
        dense), int32 given tokens [rows][given]; results as in TokenScores, 0 = not wanted.  Not waited for."""
        out = native.TokenScores(log_probs_ptr or None, entropy_ptr or None, top_tokens_ptr or None,
                                 top_log_probs_ptr or None)
        if native.lib().llambda_hip_token_scorer_score_device(
                self._h, logits_ptr or None, stride, self.vocab if count is None else count, rows,
                given_ptr or None, given, top, ctypes.byref(out), stream or None) != 0:
            raise SamplingError(native.last_error())

    def score(self, logits, given=None, top: int = 0) -> TokenScores:
        """Scores of host logits [rows][count]; given: tokens of each row, [rows] or [rows][givens]."""
        a = np.ascontiguousarray(logits, dtype=np.float32)
        if a.ndim != 2:
            raise SamplingError(f"logits have {a.ndim} dimensions, not 2")
        if top < 0:
            raise SamplingError(f"top {top} is negative")
        rows = a.shape[0]
        g = np.empty((rows, 0), dtype=np.int32)
        if given is not None:
            v = np.asarray(given)
            if v.dtype.kind not in "iu":
                raise SamplingError(f"given tokens must be whole numbers, got {v.dtype}")
            if v.shape[:1] != (rows,) or v.ndim > 2:
                raise SamplingError(f"given tokens of shape {v.shape} for {rows} rows")
            if v.size and (int(v.min()) < 0 or int(v.max()) >= a.shape[1]):
                raise SamplingError(f"given tokens are not all in 0..{a.shape[1] - 1}")
            g = np.ascontiguousarray(v.reshape(rows, v.size // rows if rows else 0), dtype=np.int32)
        r = TokenScores(np.empty(g.shape, np.float32), np.empty(rows, np.float32),
                        np.empty((rows, top), np.int32), np.empty((rows, top), np.float32))
        out = native.TokenScores(r.log_probs.ctypes.data, r.entropy.ctypes.data, r.top_tokens.ctypes.data,
                                 r.top_log_probs.ctypes.data)
        if native.lib().llambda_hip_token_scorer_score(self._h, a.ctypes.data, a.shape[1], rows, g.ctypes.data,
                                                       g.shape[1], top, ctypes.byref(out)) != 0:
            raise SamplingError(native.last_error())
        return r
