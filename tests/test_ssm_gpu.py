"""Mamba-2 mixer sessions (llambda_hip_ssm_session_*) against the recurrence
in 64 bits (ssm_reference.py, which derives the bounds)."""
import ctypes

import numpy as np
import pytest

import ssm_reference
from llambda_amd import native
from llambda_amd.hip_backend import HipBackendError
from llambda_amd.ssm import HipSsmSession, synthetic_ssm
from ssm_reference import U

pytestmark = pytest.mark.gpu

LAYOUTS = {
    "hybrid": dict(heads=64, head_dim=64, groups=8, state=128, conv_width=4),
    "one_group": dict(heads=6, head_dim=80, groups=1, state=64, conv_width=3),
    "wide": dict(heads=4, head_dim=128, groups=2, state=256, conv_width=4),
    "narrow": dict(heads=8, head_dim=32, groups=2, state=16, conv_width=2),
    "thin": dict(heads=3, head_dim=16, groups=3, state=32, conv_width=4),
    "odd": dict(heads=5, head_dim=48, groups=1, state=128, conv_width=4, conv_bias=False),
    "broad_norm": dict(heads=48, head_dim=96, groups=1, state=16, conv_width=4),
}


class Case:
    """A session over tensors on the device, and the reference's answer to the same call."""

    def __init__(self, layout, lengths, seed, old=None, new=None, slots=None, extra_rows=0, layer=None):
        import torch
        self.torch = torch
        rng = np.random.default_rng(seed)
        self.layer = layer or synthetic_ssm(rng, **LAYOUTS[layout])
        L = self.layer
        self.lengths, n = lengths, len(lengths)
        self.tokens = sum(lengths) + extra_rows
        self.x = rng.normal(size=(self.tokens, L.row)).astype(np.float32)
        self.old = np.arange(n) if old is None else np.asarray(old)
        self.new = np.arange(n) if new is None else np.asarray(new)
        self.slots = slots or int(max(self.old.max(), self.new.max(), 0)) + 1
        self.conv = rng.normal(size=(self.slots, L.conv_width - 1, L.channels)).astype(np.float32)
        self.ssm = rng.normal(size=(self.slots, L.heads, L.head_dim, L.state)).astype(np.float32)
        self.offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)

    def device(self, max_tokens=None):
        torch = self.torch
        t = torch.from_numpy
        self.dx, self.dconv, self.dssm = t(self.x).cuda(), t(self.conv).cuda(), t(self.ssm).cuda()
        self.doff = t(self.offsets).cuda()
        self.dold = t(self.old.astype(np.int32)).cuda()
        self.dnew = t(self.new.astype(np.int32)).cuda()
        self.dy = torch.full((self.tokens, self.layer.inner), 7.25, device="cuda")
        self.session = HipSsmSession(self.layer, slots=self.slots, max_tokens=max_tokens or self.tokens,
                                     max_sequences=len(self.lengths), conv_states_ptr=self.dconv.data_ptr(),
                                     ssm_states_ptr=self.dssm.data_ptr())
        torch.cuda.synchronize()
        return self

    def run(self, stream=0, lists=True):
        s, n = self.session, len(self.lengths)
        old, new = (self.dold.data_ptr(), self.dnew.data_ptr()) if lists else (0, 0)
        s.run_device(self.dx.data_ptr(), self.dy.data_ptr(), self.tokens, self.doff.data_ptr(), n, old, new, stream)

    def step(self, stream=0, lists=True):
        old, new = (self.dold.data_ptr(), self.dnew.data_ptr()) if lists else (0, 0)
        self.session.step_device(self.dx.data_ptr(), self.dy.data_ptr(), len(self.lengths), old, new, stream)

    def reference(self):
        """Per sequence what ssm_reference.sequence returns."""
        L, out = self.layer, []
        for i, old in enumerate(self.old):
            conv = self.conv[old] if old >= 0 else np.zeros((L.conv_width - 1, L.channels), np.float32)
            ssm = self.ssm[old] if old >= 0 else np.zeros((L.heads, L.head_dim, L.state), np.float32)
            out.append(ssm_reference.sequence(L, self.x[self.offsets[i]:self.offsets[i + 1]], conv, ssm))
        return out

    def check(self, refused=()):
        y, conv, ssm = (a.cpu().numpy() for a in (self.dy, self.dconv, self.dssm))
        want_conv, written = self.conv.copy(), set()
        for i, (out, taps, state, bound, state_bound) in enumerate(self.reference()):
            rows = slice(self.offsets[i], self.offsets[i + 1])
            if i in refused:
                assert np.all(y[rows] == 7.25), f"sequence {i}: rows of a refused sequence"
                continue
            far = np.abs(y[rows] - out) - bound
            assert not far.size or far.max() <= 0, (
                f"sequence {i} of {self.lengths[i]}: row {far.max(1).argmax()} is {far.max():.3g} outside")
            if self.new[i] < 0:
                continue
            written.add(int(self.new[i]))
            want_conv[self.new[i]] = taps
            far = np.abs(ssm[self.new[i]] - state) - state_bound
            assert far.max() <= 0, f"sequence {i}: state {far.max():.3g} outside"
        assert np.array_equal(conv, want_conv)
        for k in range(self.slots):
            if k not in written:
                assert np.array_equal(ssm[k], self.ssm[k]), f"slot {k} changed"
        assert np.all(y[self.offsets[-1]:] == 7.25), "rows behind the last sequence"


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("lengths", [[1], [2, 31, 32, 33], [0, 65, 0, 1, 5], [129, 300]], ids=str)
def test_prompts(hip, layout, lengths):
    n = len(lengths)
    rng = np.random.default_rng(n)
    old = rng.permutation(n)
    old[::2] = -1
    new = n + rng.permutation(n)
    c = Case(layout, lengths, 11, old, new, slots=2 * n, extra_rows=3).device()
    c.run()
    c.session.sync()
    c.check()


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("lengths", [[1] * 9, [40, 260]], ids=str)
@pytest.mark.parametrize("fresh", [False, True])
def test_errors_together(hip, layout, lengths, fresh):
    """All outputs and all states together differ by single precision's roundings, not by a product's of fewer bits."""
    n = len(lengths)
    c = Case(layout, lengths, 37, np.full(n, -1) if fresh else np.arange(n), n + np.arange(n), slots=2 * n).device()
    if max(lengths) > 1:
        c.run()
    else:
        c.step()
    c.session.sync()
    want = c.reference()
    y, ssm = c.dy.cpu().numpy().astype(np.float64), c.dssm.cpu().numpy().astype(np.float64)
    off = ssm_reference.together(y, np.concatenate([w[0] for w in want]))
    state_off = ssm_reference.together(ssm[n:], np.stack([w[2] for w in want]))
    print(f"{layout} {lengths}: outputs {off:.2e}, states {state_off:.2e}")
    assert off <= ssm_reference.TOGETHER and state_off <= ssm_reference.TOGETHER


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("n", [1, 7])
def test_steps(hip, layout, n):
    rng = np.random.default_rng(n)
    c = Case(layout, [1] * n, 12, rng.permutation(n), n + rng.permutation(n), slots=2 * n).device()
    c.step()
    c.session.sync()
    c.check()


@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_steps_of_many_sequences(hip, layout):
    """Enough for the larger parts of a state (more than 512 of 8192 elements)."""
    n = {"hybrid": 11, "one_group": 100, "wide": 37, "narrow": 71, "thin": 180, "odd": 109, "broad_norm": 13}[layout]
    rng = np.random.default_rng(n)
    old = rng.permutation(n)
    old[::5] = -1
    c = Case(layout, [1] * n, 12, old, n + rng.permutation(n), slots=2 * n).device()
    c.step()
    c.session.sync()
    c.check()


def test_steps_in_place_new_and_dropped(hip):
    c = Case("hybrid", [1] * 5, 13, [3, -1, 2, 6, -1], [3, 0, 2, -1, -1], slots=7).device()
    c.step()
    c.session.sync()
    c.check()


def test_prompts_in_place_new_and_dropped(hip):
    c = Case("one_group", [200, 3, 0, 40, 17], 14, [3, -1, 2, 6, -1], [3, 0, 2, -1, -1], slots=7).device()
    c.run()
    c.session.sync()
    c.check()


def test_without_lists_sequence_i_is_slot_i(hip):
    c = Case("narrow", [4, 150, 1], 15, slots=4).device()
    c.run(lists=False)
    c.session.sync()
    c.check()
    c = Case("narrow", [1, 1, 1], 16, slots=4).device()
    c.step(lists=False)
    c.session.sync()
    c.check()


def test_one_state_read_by_several(hip):
    """A prefix's state continued in several ways."""
    c = Case("thin", [40, 200, 3], 17, [0, 0, 0], [1, 2, 3], slots=4).device()
    c.run()
    c.session.sync()
    c.check()


def test_long_sequence_of_many_segments(hip):
    c = Case("narrow", [5003, 64], 18, [0, 1], [0, 2], slots=3).device()
    c.run()
    c.session.sync()
    c.check()


def test_decays_of_long_segments(hip):
    """A state that only decays, by about 2^-100 over each of two segments of 64 chunks (512 narrow heads are
    128 workgroups to a segment).  Steps of 32 have a softplus that is exact, so the decay is 2^(32 a log2 e)
    a token.  Over the second segment each chunk multiplies by an exponential (off by 2^-23 of itself, and by
    2^-25 ln 2 for its argument of less than 2) and rounds: 3.4 2^-24 a chunk.  Over the first there is one,
    of a sum that is rounded once: 2^-25 of 128, times ln 2, and 3 2^-24."""
    import torch
    heads, tokens = 512, 4096
    rng = np.random.default_rng(36)
    layer = synthetic_ssm(rng, heads=heads, head_dim=16, groups=1, state=16, conv_bias=False)
    layer.dt_bias[:] = 32
    layer.a = (-rng.uniform(80, 100, size=heads) * np.log(2) / (32 * 2048)).astype(np.float32)
    conv = torch.zeros(1, 3, layer.channels, device="cuda")
    start = (rng.uniform(1, 2, size=(1, heads, 16, 16)) * 2.0 ** 120).astype(np.float32)
    ssm = torch.from_numpy(start).cuda()
    x, y = torch.zeros(tokens, layer.row, device="cuda"), torch.empty(tokens, layer.inner, device="cuda")
    offsets = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    session = HipSsmSession(layer, max_tokens=tokens, conv_states_ptr=conv.data_ptr(), ssm_states_ptr=ssm.data_ptr())
    torch.cuda.synchronize()
    session.run_device(x.data_ptr(), y.data_ptr(), tokens, offsets.data_ptr(), 1)
    session.sync()
    want = start.astype(np.float64) * np.exp(tokens * 32 * layer.a.astype(np.float64))[None, :, None, None]
    off = np.abs(ssm.cpu().numpy() / want - 1).max()
    assert off <= 64 * 3.4 * U + 128 * U / 2 * np.log(2) + 3 * U
    assert not y.cpu().numpy().any() and not conv.cpu().numpy().any()


def test_misaligned_rows_and_buffers(hip):
    """Rows of an odd length from a pointer that is only 4-byte aligned."""
    import torch
    c = Case("thin", [50, 9], 19).device()
    flat = torch.empty(c.dx.numel() + 1, device="cuda")
    flat[1:] = c.dx.reshape(-1)
    out = torch.full((c.dy.numel() + 1,), 7.25, device="cuda")
    torch.cuda.synchronize()
    c.session.run_device(flat.data_ptr() + 4, out.data_ptr() + 4, c.tokens, c.doff.data_ptr(), 2)
    c.session.sync()
    c.dy = out[1:].reshape(c.dy.shape)
    c.check()


def test_strong_decays_and_large_steps(hip):
    """Decays that leave nothing beside decays that keep all: exponents far beyond single precision's range."""
    rng = np.random.default_rng(20)
    layer = synthetic_ssm(rng, **LAYOUTS["narrow"])
    layer.a[:] = [-1e4, -16, -1e-6, 0, -50, -1, -3e3, -8]
    c = Case("narrow", [97, 260], 21, layer=layer)
    c.x[:, -layer.heads:] *= 4
    c.x[::13, -layer.heads:] = 60
    c.device().run()
    c.session.sync()
    c.check()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_non_finite_rows_reach_no_earlier_token_and_no_other_sequence(hip, value):
    import torch
    c = Case("narrow", [70, 90, 20], 22)
    L = c.layer
    clean = c.reference()
    at, ch = 41, 5
    c.x[c.offsets[1] + at, L.inner + ch] = value  # an x channel of head 0 in the second sequence
    c.device().run()
    c.session.sync()
    y = c.dy.cpu().numpy()
    for i in (0, 2):
        out, _, _, bound, _ = clean[i]
        assert np.all(np.abs(y[c.offsets[i]:c.offsets[i + 1]] - out) <= bound)
    out, _, _, bound, _ = clean[1]
    rows = y[c.offsets[1]:c.offsets[2]]
    assert np.all(np.abs(rows[:at] - out[:at]) <= bound[:at])
    width = L.inner // L.groups
    assert np.all(~np.isfinite(rows[at:, ch])) and np.all(~np.isfinite(rows[at:, :width]))
    other = slice(width, None)  # the other group's channels do not know
    assert np.all(np.abs(rows[:, other] - out[:, other]) <= bound[:, other])
    # B of one token: its group's states from there on
    c = Case("narrow", [70, 90, 20], 22)
    c.x[c.offsets[1] + at, L.inner + L.inner + 3] = value
    c.device().run()
    c.session.sync()
    rows = c.dy.cpu().numpy()[c.offsets[1]:c.offsets[2]]
    assert np.all(np.abs(rows[:at] - out[:at]) <= bound[:at])
    assert not np.isfinite(rows[at + 1:, :width]).any()
    assert np.all(np.abs(rows[:, other] - out[:, other]) <= bound[:, other])
    torch.cuda.synchronize()


def test_refused_on_the_device(hip):
    import torch
    # slot 2 is written twice; slot 0 is written by 3 and read by 4; slot 9 does not exist
    c = Case("one_group", [40, 5, 130, 7, 8, 2], 23, [3, 4, 1, -1, 0, 5], [2, 6, 2, 0, 7, 5], slots=8).device()
    c.dold[5] = 9
    torch.cuda.synchronize()
    c.run()
    with pytest.raises(HipBackendError, match="outside the pool.*written by one sequence"):
        c.session.sync()
    c.session.sync()  # reported once
    c.check(refused=(0, 2, 3, 5))
    c = Case("one_group", [1] * 6, 24, [3, 4, 1, -1, 0, 5], [2, 6, 2, 0, 7, 5], slots=8).device()
    c.dnew[5] = -2
    torch.cuda.synchronize()
    c.step()
    with pytest.raises(HipBackendError, match="outside the pool.*written by one sequence"):
        c.session.sync()
    c.check(refused=(0, 2, 3, 5))


def test_refusals_of_several_calls_are_reported_together(hip):
    """Of calls on several streams since the last report; then none is left."""
    import torch
    c = Case("thin", [5, 3, 4], 41, slots=3).device()
    streams = [torch.cuda.Stream() for _ in range(2)]
    bad = torch.tensor([0, 5, 3, 12], dtype=torch.int32, device="cuda")
    c.dold[1] = 9
    torch.cuda.synchronize()
    for _ in range(2):
        c.session.run_device(c.dx.data_ptr(), c.dy.data_ptr(), c.tokens, bad.data_ptr(), 3, c.dnew.data_ptr(),
                             c.dnew.data_ptr(), streams[0].cuda_stream)
        c.run(streams[1].cuda_stream)
        torch.cuda.synchronize()
        with pytest.raises(HipBackendError, match="offsets do not ascend.*outside the pool"):
            c.session.sync(streams[0].cuda_stream)
        for s in streams:
            c.session.sync(s.cuda_stream)


@pytest.mark.parametrize("offsets", [[0, 5, 3, 12], [0, 5, 12, 13], [-1, 5, 6, 12], [0, 12, 0, 12]])
def test_offsets_that_do_not_ascend(hip, offsets):
    import torch
    c = Case("thin", [5, 3, 4], 25).device()
    c.doff.copy_(torch.tensor(offsets, dtype=torch.int32))
    torch.cuda.synchronize()
    c.run()
    with pytest.raises(HipBackendError, match="offsets do not ascend"):
        c.session.sync()
    assert bool((c.dy == 7.25).all()) and np.array_equal(c.dssm.cpu().numpy(), c.ssm)
    assert np.array_equal(c.dconv.cpu().numpy(), c.conv)
    # the session goes on
    c.doff.copy_(torch.from_numpy(c.offsets))
    torch.cuda.synchronize()
    c.run()
    c.session.sync()
    c.check()


def test_captured_calls_replay(hip):
    """A prompt and a step in one graph, replayed between eager calls of another session."""
    import torch
    c = Case("hybrid", [70, 1, 33], 26, [0, 1, 2], [3, 4, 5], slots=6).device()
    e = Case("hybrid", [70, 1, 33], 27, [0, 1, 2], [3, 4, 5], slots=6).device()
    d = Case("hybrid", [1] * 9, 28, np.arange(9), 9 + np.arange(9), slots=18).device()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        c.run(stream.cuda_stream)
        d.step(stream.cuda_stream)
    rng = np.random.default_rng(29)
    for _ in range(4):
        for k in (c, d):
            k.x = rng.normal(size=k.x.shape).astype(np.float32)
            k.dx.copy_(torch.from_numpy(k.x))
            k.dy.fill_(7.25)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        e.run()
        torch.cuda.synchronize()
        for k in (c, d, e):
            k.session.sync()
            k.check()
            k.dssm.copy_(torch.from_numpy(k.ssm))
            k.dconv.copy_(torch.from_numpy(k.conv))


def test_calls_on_several_streams_share_the_workspace(hip):
    """Each call waits for the one before, whatever its stream."""
    import torch
    c = Case("narrow", [900, 700], 30, [0, 1], [2, 3], slots=4).device()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.full_like(c.dy, 7.25) for _ in range(6)]
    torch.cuda.synchronize()
    for k, out in enumerate(outs):
        c.session.run_device(c.dx.data_ptr(), out.data_ptr(), c.tokens, c.doff.data_ptr(), 2, c.dold.data_ptr(),
                             c.dnew.data_ptr(), streams[k % 3].cuda_stream)
    torch.cuda.synchronize()
    c.session.sync()
    c.dy = outs[0]
    c.check()
    for out in outs[1:]:
        assert torch.equal(out, outs[0])


@pytest.mark.parametrize("rows", [1, 2])
def test_host_runs_wait_for_device_calls_in_flight(hip, rows):
    """Prompts of a slot on a stream of the caller's, at once followed by a host run of the same slot."""
    import torch
    c = Case("hybrid", [2000], 34).device()
    more = np.random.default_rng(35).normal(size=(rows, c.layer.row)).astype(np.float32)
    stream = torch.cuda.Stream()

    def outcome(wait):
        c.dconv.copy_(torch.from_numpy(c.conv))
        c.dssm.copy_(torch.from_numpy(c.ssm))
        torch.cuda.synchronize()
        for _ in range(8):
            c.run(stream.cuda_stream)
        if wait:
            torch.cuda.synchronize()
        y = c.session.run(more)
        torch.cuda.synchronize()
        c.session.sync()
        return [y, *c.session.read_state(0)]

    for a, b in zip(outcome(True), outcome(False)):
        assert np.array_equal(a, b)


def test_host_runs_and_states(hip):
    rng = np.random.default_rng(31)
    layer = synthetic_ssm(rng, **LAYOUTS["one_group"])
    x = rng.normal(size=(45, layer.row)).astype(np.float32)
    s = HipSsmSession(layer, slots=3, max_tokens=64)
    assert (s.input_element_count, s.output_element_count) == (layer.row, layer.inner)
    conv = np.zeros((layer.conv_width - 1, layer.channels), np.float32)
    ssm = np.zeros((layer.heads, layer.head_dim, layer.state), np.float32)
    out, taps, state, bound, state_bound = ssm_reference.sequence(layer, x, conv, ssm)
    y = np.concatenate([s.run(x[:30], slot=1), s.run(x[30:31], slot=1), s.run(x[31:], slot=1)])
    assert np.all(np.abs(y - out) <= bound)
    got_conv, got_ssm = s.read_state(1)
    assert np.array_equal(got_conv, taps) and np.all(np.abs(got_ssm - state) <= state_bound)
    for k in (0, 2):
        assert not any(a.any() for a in s.read_state(k))
    s.write_state(2, got_conv, got_ssm)
    assert np.array_equal(s.run(x[:9], slot=2), s.run(x[:9], slot=1))
    s.reset(1)
    assert np.all(np.abs(s.run(x, slot=1) - out) <= bound)
    with pytest.raises(HipBackendError, match="slot 3 is not in 0..2"):
        s.run(x, slot=3)
    with pytest.raises(HipBackendError, match="65 tokens are not in 1..64"):
        s.run(np.zeros((65, layer.row), np.float32))
    s.close()
    with pytest.raises(HipBackendError, match="closed"):
        s.run(x)


def test_refused_on_the_host(hip):
    c = Case("thin", [5, 3], 32, slots=2).device()
    s, x, y, o = c.session, c.dx.data_ptr(), c.dy.data_ptr(), c.doff.data_ptr()
    for args, text in [((0, y, 8, o, 2), "null input"), ((x, 0, 8, o, 2), "null input"),
                       ((x, y, 8, 0, 2), "null offsets"), ((x, y, 9, o, 2), "9 tokens"),
                       ((x, y, 0, o, 2), "0 tokens"), ((x, y, 8, o, 3), "3 sequences"),
                       ((x, y, 8, o, 0), "0 sequences"), ((x + 2, y, 8, o, 2), "aligned"),
                       ((x, x + 4, 8, o, 2), "overlap")]:
        with pytest.raises(HipBackendError, match=text):
            s.run_device(*args)
    with pytest.raises(HipBackendError, match="3 sequences"):
        s.step_device(x, y, 3)
    few = HipSsmSession(c.layer, slots=1, max_tokens=8, max_sequences=2)
    with pytest.raises(HipBackendError, match="without a slot list"):
        few.step_device(x, y, 2)
    L = native.lib()
    assert L.llambda_hip_ssm_session_run_device(None, x, y, 8, o, 2, None, None, None) == -1
    assert L.llambda_hip_ssm_session_read_state(s.pointer, 0, None, None) == -1
    assert L.llambda_hip_ssm_session_sync(None, None) == -1
    assert L.llambda_hip_ssm_session_create(None, ctypes.byref(ctypes.c_void_p())) == -1


def test_more_workgroups_than_a_launch_has(hip):
    """Refused before anything is enqueued: 65535 sequences of 131 heads, one head to a workgroup of 512 threads,
    are more than 2^32 threads.  The slots take part of them."""
    import torch
    layer = synthetic_ssm(np.random.default_rng(38), heads=131, head_dim=16, groups=1, state=16)
    session = HipSsmSession(layer, slots=8, max_tokens=65535, max_sequences=65535)
    x = torch.zeros(65535, layer.row, device="cuda")
    y = torch.full((65535, layer.inner), 7.25, device="cuda")
    few = torch.arange(9, dtype=torch.int32, device="cuda")
    many = torch.full((65536,), -1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with pytest.raises(HipBackendError, match="65535 tokens of 65535 sequences are too many"):
        # (nothing is read: the rows and the offsets are not those of such a call)
        session.run_device(x.data_ptr(), y.data_ptr(), 65535, many.data_ptr(), 65535, many.data_ptr(), many.data_ptr())
    session.sync()
    assert bool((y == 7.25).all())
    session.run_device(x.data_ptr(), y.data_ptr(), 8, few.data_ptr(), 8)  # the session goes on
    session.sync()
    assert bool((y[8:] == 7.25).all()) and bool((y[:8] != 7.25).all())


@pytest.mark.parametrize("layout", ["hybrid", "wide", "narrow"])
@pytest.mark.parametrize("x,b,c,state", [(1e-12, 1, 1, 1), (1e6, 1e-6, 1e3, 1e-9), (1e-18, 1e-10, 1e25, 1e-15),
                                         (1e8, 1e4, 1e-10, 1e15), (1, 1e-30, 1e20, 1)], ids=str)
def test_magnitudes(hip, layout, x, b, c, state):
    """Operands are held at powers of two that follow their largest values: of x from chunk to chunk (here by
    up to 10^12 either way), of B and C from token to token, of the state with its inputs."""
    rng = np.random.default_rng(21)
    layer = synthetic_ssm(rng, **LAYOUTS[layout])
    part = np.repeat([x, b, c], [layer.inner, layer.groups * layer.state, layer.groups * layer.state])
    layer.conv_weight = (layer.conv_weight * part[:, None]).astype(np.float32)
    if layer.conv_bias is not None:
        layer.conv_bias = (layer.conv_bias * part).astype(np.float32)
    case = Case(layout, [150, 300], 22, layer=layer)
    case.ssm *= np.float32(state)
    row = 0
    while row < case.tokens:
        case.x[row:row + 40, layer.inner:2 * layer.inner] *= np.float32(10.0 ** rng.integers(-6, 7))
        row += 40
    case.device()
    case.run()
    case.session.sync()
    case.check()


@pytest.mark.parametrize("layout", ["narrow", "odd", "wide"])
def test_last_rows_near_the_end_of_single_precision(hip, layout):
    """Taps of 0.5 of a last row of 2.5e38 are finite; those of the row repeated, as the chunk is filled up, are not."""
    rng = np.random.default_rng(39)
    layer = synthetic_ssm(rng, **LAYOUTS[layout])
    layer.conv_weight[:layer.inner] = 0.9 if layer.conv_width == 2 else 0.5
    layer.d[:] = 0.5
    case = Case(layout, [33, 64, 150, 1], 40, layer=layer)
    for end in case.offsets[1:]:
        case.x[end - 1, layer.inner:layer.inner + 40] = 2.5e38
        case.x[end - 1, :layer.inner] = 1e-30  # (the gate, so that the row's norm is of ordinary numbers)
    case.device().run()
    case.session.sync()
    case.check()


@pytest.mark.parametrize("run", [True, False])
def test_outputs_whose_squares_leave_single_precision(hip, run):
    rng = np.random.default_rng(23)
    layer = synthetic_ssm(rng, **LAYOUTS["one_group"])
    layer.d = (layer.d * 1e25).astype(np.float32)
    case = Case("one_group", [1, 1, 1], 24, layer=layer).device()
    if run:
        case.run()
    else:
        case.step()
    case.session.sync()
    case.check()


@pytest.mark.parametrize("state", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("conv_width", [2, 3, 4])
def test_every_state_and_number_of_taps(hip, state, conv_width):
    layer = synthetic_ssm(np.random.default_rng(42), heads=6, head_dim=48, groups=2, state=state, conv_width=conv_width)
    for lengths, old in (([1, 33, 130], [0, -1, 2]), ([1, 1, 1], [2, -1, 0])):
        c = Case(None, lengths, 43, old, [3, 4, 5], slots=6, layer=layer).device()
        c.run()
        c.session.sync()
        c.check()
    c.dconv.copy_(c.torch.from_numpy(c.conv))
    c.dssm.copy_(c.torch.from_numpy(c.ssm))
    c.dy.fill_(7.25)
    c.step()
    c.session.sync()
    c.check()


@pytest.mark.parametrize("heads,head_dim,groups", [(20, 128, 1), (96, 128, 3), (128, 128, 1), (512, 16, 256), (4, 16, 4)])
def test_norm_widths(hip, heads, head_dim, groups):
    """Groups of 2560, 4096, 16384 (the most), 32 and 16 channels."""
    layer = synthetic_ssm(np.random.default_rng(44), heads=heads, head_dim=head_dim, groups=groups, state=16)
    c = Case(None, [1, 3, 40], 45, [0, -1, 2], [3, 4, 5], slots=6, extra_rows=2, layer=layer).device()
    c.run()
    c.session.sync()
    c.check()
    c = Case(None, [1, 1, 1], 46, [0, -1, 2], [3, 4, 5], slots=6, layer=layer).device()
    c.step()
    c.session.sync()
    c.check()


def test_rows_before_the_first_sequence(hip):
    c = Case("narrow", [50, 0, 7], 47, slots=3, extra_rows=5)
    c.offsets += 5
    c.device().run()
    c.session.sync()
    assert bool((c.dy[:5] == 7.25).all())
    c.check()


@pytest.mark.parametrize("given", ["old", "new"])
def test_one_slot_list(hip, given):
    """The list that is not given is slot i."""
    old, new = ([3, -1, 4], None) if given == "old" else (None, [3, -1, 4])
    for lengths in ([40, 2, 1], [1, 1, 1]):
        c = Case("narrow", lengths, 48, old, new, slots=5).device()
        lists = (c.dold.data_ptr(), 0) if given == "old" else (0, c.dnew.data_ptr())
        if max(lengths) > 1:
            c.session.run_device(c.dx.data_ptr(), c.dy.data_ptr(), c.tokens, c.doff.data_ptr(), 3, *lists)
        else:
            c.session.step_device(c.dx.data_ptr(), c.dy.data_ptr(), 3, *lists)
        c.session.sync()
        c.check()
