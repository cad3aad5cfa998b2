"""Mamba-2 mixer sessions on the HIP backend.

A ``SsmLayer`` holds the tensors that a recurrent layer of the reference's
Nemotron-H step function reads between ``ssm_in`` and ``ssm_out``
(llambda.lisp:5768-5825, 6020-6128); ``HipSsmSession`` uploads them once, holds
the states of a pool of sequences, and runs the convolution, the scan and the
gated norm on the device: prompts of several lengths, or one token of each
sequence.  Rows are those of the projection sessions around it: ``ssm_in``'s
output [z | x | B | C | dt], ``ssm_out``'s input.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Tuple

import numpy as np

from . import ggml, native
from .hip_backend import HipBackendError, _check


@dataclass
class SsmLayer:
    heads: int
    head_dim: int
    groups: int
    state: int
    conv_width: int
    conv_weight: np.ndarray               # F32 [channels][conv_width]  ssm_conv1d.weight
    dt_bias: np.ndarray                   # F32 [heads]                 ssm_dt.bias
    a: np.ndarray                         # F32 [heads]                 ssm_a (negative)
    d: np.ndarray                         # F32 [heads]                 ssm_d
    norm: np.ndarray                      # F32 [heads * head_dim]      ssm_norm.weight
    conv_bias: Optional[np.ndarray] = None  # F32 [channels]            ssm_conv1d.bias
    norm_epsilon: float = 1e-5

    @property
    def inner(self) -> int:
        return self.heads * self.head_dim

    @property
    def channels(self) -> int:
        """Channels of the convolution: x | B | C."""
        return self.inner + 2 * self.groups * self.state

    @property
    def row(self) -> int:
        """Elements of an input row: z | x | B | C | dt."""
        return self.inner + self.channels + self.heads


class HipSsmSession:
    """`slots` sequences' states, in device memory of the session's own (zeroed) or the caller's
    (conv_states_ptr [slots][conv_width - 1][channels], ssm_states_ptr
    [slots][heads][head_dim][state]); max_tokens and max_sequences bound a call."""

    def __init__(self, layer: SsmLayer, *, slots: int = 1, max_tokens: int = 4096,
                 max_sequences: int = 1, conv_states_ptr: int = 0, ssm_states_ptr: int = 0):
        self.pointer = None
        self.layer = layer
        self.slots = slots
        keep = []

        def arr(a, n, what):
            if a is None:
                return None
            a = np.ascontiguousarray(a, dtype=np.float32)
            if a.size != n:
                raise HipBackendError(f"HIP SSM {what} has {a.size} elements, not {n}.")
            keep.append(a)
            return a.ctypes.data

        d = native.SsmDesc()
        d.heads, d.head_dim, d.groups = layer.heads, layer.head_dim, layer.groups
        d.state, d.conv_width = layer.state, layer.conv_width
        d.conv_weight = arr(layer.conv_weight, layer.channels * layer.conv_width, "conv_weight")
        d.conv_bias = arr(layer.conv_bias, layer.channels, "conv_bias")
        d.dt_bias = arr(layer.dt_bias, layer.heads, "dt_bias")
        d.a = arr(layer.a, layer.heads, "a")
        d.d = arr(layer.d, layer.heads, "d")
        d.norm = arr(layer.norm, layer.inner, "norm")
        d.norm_epsilon = layer.norm_epsilon
        d.slots, d.max_tokens, d.max_sequences = slots, max_tokens, max_sequences
        d.conv_states = conv_states_ptr or None
        d.ssm_states = ssm_states_ptr or None
        handle = ctypes.c_void_p()
        _check(native.lib().llambda_hip_ssm_session_create(ctypes.byref(d), ctypes.byref(handle)),
               "HIP SSM session creation")
        self.pointer = handle.value

    def close(self) -> None:
        if self.pointer:
            native.lib().llambda_hip_ssm_session_destroy(self.pointer)
            self.pointer = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass

    def _live(self):
        if not self.pointer:
            raise HipBackendError("HIP SSM session is closed.")
        return self.pointer

    @property
    def input_element_count(self) -> int:
        return native.lib().llambda_hip_ssm_session_input_element_count(self.pointer)

    @property
    def output_element_count(self) -> int:
        return native.lib().llambda_hip_ssm_session_output_element_count(self.pointer)

    def run(self, x: np.ndarray, slot: int = 0) -> np.ndarray:
        """Rows x [tokens][row] of the sequence in `slot`, which continues from there."""
        x = np.ascontiguousarray(x, dtype=np.float32).reshape(-1, self.layer.row)
        y = np.empty((x.shape[0], self.layer.inner), dtype=np.float32)
        _check(native.lib().llambda_hip_ssm_session_run(
            self._live(), slot, x.ctypes.data, x.size, y.ctypes.data, y.size, x.shape[0]), "HIP SSM run")
        return y

    def run_device(self, x_ptr: int, y_ptr: int, tokens: int, offsets_ptr: int, sequences: int,
                   from_ptr: int = 0, to_ptr: int = 0, stream: int = 0) -> None:
        """Sequence i's rows [offsets[i], offsets[i + 1]); int32 lists on the device, 0 = slot i."""
        _check(native.lib().llambda_hip_ssm_session_run_device(
            self._live(), x_ptr or None, y_ptr or None, tokens, offsets_ptr or None, sequences,
            from_ptr or None, to_ptr or None, stream or None), "HIP SSM device run")

    def step_device(self, x_ptr: int, y_ptr: int, sequences: int, from_ptr: int = 0, to_ptr: int = 0,
                    stream: int = 0) -> None:
        """One token of each sequence."""
        _check(native.lib().llambda_hip_ssm_session_step_device(
            self._live(), x_ptr or None, y_ptr or None, sequences, from_ptr or None, to_ptr or None,
            stream or None), "HIP SSM device step")

    def sync(self, stream: int = 0) -> None:
        """Wait for `stream`; raises if the device refused sequences of a call."""
        _check(native.lib().llambda_hip_ssm_session_sync(self._live(), stream or None), "HIP SSM sync")

    def reset(self, slot: int) -> None:
        _check(native.lib().llambda_hip_ssm_session_reset(self._live(), slot), "HIP SSM reset")

    def _state_shapes(self):
        L = self.layer
        return (L.conv_width - 1, L.channels), (L.heads, L.head_dim, L.state)

    def write_state(self, slot: int, conv: np.ndarray, ssm: np.ndarray) -> None:
        shapes = self._state_shapes()
        conv = np.ascontiguousarray(conv, dtype=np.float32)
        ssm = np.ascontiguousarray(ssm, dtype=np.float32)
        if conv.shape != shapes[0] or ssm.shape != shapes[1]:
            raise HipBackendError(f"HIP SSM state has shapes {conv.shape}, {ssm.shape}, not {shapes}.")
        _check(native.lib().llambda_hip_ssm_session_write_state(
            self._live(), slot, conv.ctypes.data, ssm.ctypes.data, 0), "HIP SSM state write")

    def write_state_device(self, slot: int, conv_ptr: int, ssm_ptr: int) -> None:
        _check(native.lib().llambda_hip_ssm_session_write_state(
            self._live(), slot, conv_ptr or None, ssm_ptr or None, 1), "HIP SSM state write")

    def read_state(self, slot: int) -> Tuple[np.ndarray, np.ndarray]:
        """(conv [conv_width - 1][channels], ssm [heads][head_dim][state]) of `slot`."""
        conv, ssm = (np.empty(s, dtype=np.float32) for s in self._state_shapes())
        _check(native.lib().llambda_hip_ssm_session_read_state(
            self._live(), slot, conv.ctypes.data, ssm.ctypes.data), "HIP SSM state read")
        return conv, ssm


def ssm_layer_from_model(model, layer_index: int, *, heads: int, groups: int,
                         norm_epsilon: float = 1e-5) -> SsmLayer:
    """The tensors blk.N.ssm_* of layer `layer_index`, from a projection.ProjectionModel
    (heads: nemotron_h_moe.ssm.time_step_rank, groups: .ssm.group_count)."""
    def vector(name, required=True):
        t = model.tensor_info(f"blk.{layer_index}.{name}", required=required)
        if t is None:
            return None
        if t.type_tag != ggml.F32:
            raise HipBackendError(f"blk.{layer_index}.{name} must be F32")
        return np.ascontiguousarray(t.data).view(np.float32).reshape(-1)

    norm = vector("ssm_norm.weight")
    conv = model.tensor_info(f"blk.{layer_index}.ssm_conv1d.weight", required=True)
    width, channels = conv.columns, conv.rows
    if norm.size % heads or (channels - norm.size) % (2 * groups):
        raise HipBackendError(f"blk.{layer_index}: {channels} convolution channels and {norm.size} inner channels "
                              f"do not fit {heads} heads in {groups} groups")
    return SsmLayer(heads=heads, head_dim=norm.size // heads, groups=groups,
                    state=(channels - norm.size) // (2 * groups), conv_width=width,
                    conv_weight=vector("ssm_conv1d.weight").reshape(channels, width),
                    conv_bias=vector("ssm_conv1d.bias", required=False),
                    dt_bias=vector("ssm_dt.bias"), a=vector("ssm_a"), d=vector("ssm_d"), norm=norm,
                    norm_epsilon=norm_epsilon)


def synthetic_ssm(rng: np.random.Generator, *, heads=64, head_dim=64, groups=8, state=128,
                  conv_width=4, conv_bias=True) -> SsmLayer:
    """A layer with steps of 0.001 to 0.1 (log-uniform) and A in [-16, -1], as such layers start from."""
    channels = heads * head_dim + 2 * groups * state
    step = np.exp(rng.uniform(np.log(1e-3), np.log(1e-1), size=heads))
    f = np.float32
    return SsmLayer(heads=heads, head_dim=head_dim, groups=groups, state=state, conv_width=conv_width,
                    conv_weight=(rng.normal(size=(channels, conv_width)) * 0.5).astype(f),
                    conv_bias=(rng.normal(size=channels) * 0.1).astype(f) if conv_bias else None,
                    dt_bias=(step + np.log(-np.expm1(-step))).astype(f),
                    a=-rng.uniform(1, 16, size=heads).astype(f),
                    d=(1 + 0.1 * rng.normal(size=heads)).astype(f),
                    norm=(1 + 0.1 * rng.normal(size=heads * head_dim)).astype(f))
