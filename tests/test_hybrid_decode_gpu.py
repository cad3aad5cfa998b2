"""A hybrid model's operators together, as a server runs them: packed prompts
through projection, mixer, projection, routed experts and output head, a token
drawn for each sequence, then further tokens by one captured graph, replayed.
Every stage is compared with its definition in 64 bits on the input that the
device gave it."""
import numpy as np
import pytest

import oracle
import ssm_reference
from llambda_amd import ggml, synthetic
from llambda_amd.hip_backend import make_hip_session_packed
from llambda_amd.moe import HipMoeSession, HipRouter, Routing, synthetic_nemotron_h
from llambda_amd.sampling import HipBatchSampler
from llambda_amd.ssm import HipSsmSession, synthetic_ssm
from test_batch_sampling_gpu import reference as sampling_reference
from test_router_gpu import _experts, reference as routing_reference

pytestmark = pytest.mark.gpu

HIDDEN, VOCAB, LENGTHS = 512, 1000, [5, 40, 1, 70]


class Model:
    def __init__(self, rng):
        self.ssm = synthetic_ssm(rng, heads=8, head_dim=32, groups=2, state=16)
        self.moe = synthetic_nemotron_h(rng, hidden=HIDDEN, experts=16, top_k=4, ffn=96, shared_ffn=160)
        self.routing = Routing(16, 4, score="sigmoid", bias=(rng.normal(size=16) * 0.3).astype(np.float32),
                               groups=4, top_groups=2, group_rank=2, weights_scale=1.75)
        self.embedding = rng.normal(size=(VOCAB, HIDDEN)).astype(np.float32)
        self.packed = {}
        for name, rows, columns in [("ssm_in", self.ssm.row, HIDDEN), ("ssm_out", HIDDEN, self.ssm.inner),
                                    ("output", VOCAB, HIDDEN)]:
            self.packed[name] = (synthetic.packed(ggml.Q4_K, rng, rows, columns), rows, columns)
        self.sessions = {n: make_hip_session_packed(w, ggml.Q4_K, r, c) for n, (w, r, c) in self.packed.items()}

    def projection(self, name, x, y):
        w, rows, columns = self.packed[name]
        w = oracle.dequantize(ggml.Q4_K, w, rows * columns).reshape(rows, columns).astype(np.float64)
        x = x.astype(np.float64)
        assert np.all(np.abs(y - x @ w.T) <= 1e-4 * (np.abs(x) @ np.abs(w).T)), name

    def experts(self, x, y):
        logits = x.astype(np.float64) @ self.moe.router.astype(np.float64).T
        idx, w = routing_reference(self.routing, logits.astype(np.float32))
        experts, sizes, shared = _experts(self.moe, x)
        want, size = shared[0].copy(), shared[1].copy()
        for t in range(len(x)):
            want[t] += (w[t, :, None] * experts[t, idx[t]]).sum(0)
            size[t] += (w[t, :, None] * sizes[t, idx[t]]).sum(0)
        assert np.all(np.abs(y - want) <= 1e-4 * size)


class Buffers:
    def __init__(self, torch, model, tokens, sequences):
        def make(*shape):
            return torch.zeros(*shape, device="cuda")
        self.hidden, self.rows = make(tokens, HIDDEN), make(tokens, model.ssm.row)
        self.mixed, self.mixer_out = make(tokens, model.ssm.inner), make(tokens, HIDDEN)
        self.added, self.expert_out = make(sequences, HIDDEN), make(sequences, HIDDEN)
        self.last, self.logits = make(sequences, HIDDEN), make(sequences, VOCAB)

    def host(self):
        return {k: v.cpu().numpy() for k, v in vars(self).items()}


def test_prompts_then_replayed_steps(hip):
    import torch
    rng = np.random.default_rng(17)
    model = Model(rng)
    n, tokens = len(LENGTHS), sum(LENGTHS)
    slots = [4, 0, 3, 1]  # slot 2 stays another's
    mixer = HipSsmSession(model.ssm, slots=5, max_tokens=tokens, max_sequences=n)
    moe = HipMoeSession(model.moe)
    router = HipRouter(model.routing)
    moe.set_router(router)
    sampler = HipBatchSampler(VOCAB, n)
    embedding = torch.from_numpy(model.embedding).cuda()
    prompt = torch.from_numpy(rng.integers(0, VOCAB, size=tokens).astype(np.int32)).cuda()
    offsets = torch.from_numpy(np.concatenate([[0], np.cumsum(LENGTHS)]).astype(np.int32)).cuda()
    new = torch.tensor(slots, dtype=torch.int32, device="cuda")
    fresh = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    ends = (offsets[1:] - 1).long()
    parameters = dict(t=np.array([2000, 0, 500, 9000], np.float32), k=np.array([0, 0, 50, 7], np.int32),
                      p=np.array([0.95, 1, 0.8, 1], np.float32), m=np.array([0.01, 0, 0, 0.1], np.float32))
    device = {k: torch.from_numpy(v).cuda() for k, v in parameters.items()}
    random = torch.zeros(n, device="cuda")
    drawn = torch.zeros(n, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    s = stream.cuda_stream

    def forward(b, ids, count, mix, rows_of):
        b.hidden.copy_(embedding.index_select(0, ids.long()))
        model.sessions["ssm_in"].run_device(b.hidden.data_ptr(), b.rows.data_ptr(), count, s)
        mix(b)
        model.sessions["ssm_out"].run_device(b.mixed.data_ptr(), b.mixer_out.data_ptr(), count, s)
        b.added.copy_(rows_of(b.hidden) + rows_of(b.mixer_out))
        moe.run_device(b.added.data_ptr(), b.expert_out.data_ptr(), n, s)
        b.last.copy_(b.added + b.expert_out)
        model.sessions["output"].run_device(b.last.data_ptr(), b.logits.data_ptr(), n, s)
        sampler.sample_device(b.logits.data_ptr(), n, drawn.data_ptr(), random.data_ptr(),
                              temperature_ptr=device["t"].data_ptr(), top_k_ptr=device["k"].data_ptr(),
                              top_p_ptr=device["p"].data_ptr(), min_p_ptr=device["m"].data_ptr(), stream=s)

    def check(b, ids, lengths, before, u):
        """The stages of a finished forward; the mixer's from the states `before`."""
        h = b.host()
        assert np.array_equal(h["hidden"], model.embedding[ids])
        model.projection("ssm_in", h["hidden"], h["rows"])
        at = 0
        for i, length in enumerate(lengths):
            y, conv, ssm, bound, ssm_bound = ssm_reference.sequence(
                model.ssm, h["rows"][at:at + length], *before[i])
            assert np.all(np.abs(h["mixed"][at:at + length] - y) <= bound)
            got = mixer.read_state(slots[i])
            assert np.array_equal(got[0], conv)
            assert np.all(np.abs(got[1] - ssm) <= ssm_bound)
            at += length
        model.projection("ssm_out", h["mixed"], h["mixer_out"])
        last = np.cumsum(lengths) - 1
        assert np.array_equal(h["added"], h["hidden"][last] + h["mixer_out"][last])
        model.experts(h["added"], h["expert_out"])
        assert np.array_equal(h["last"], h["added"] + h["expert_out"])
        model.projection("output", h["last"], h["logits"])
        want = [sampling_reference(row, u[i], *(parameters[k][i] for k in "tkpm"))
                for i, row in enumerate(h["logits"])]
        assert drawn.cpu().numpy().tolist() == want and min(want) >= 0

    zero = (np.zeros((model.ssm.conv_width - 1, model.ssm.channels), np.float32),
            np.zeros((model.ssm.heads, model.ssm.head_dim, model.ssm.state), np.float32))
    other = tuple(rng.normal(size=v.shape).astype(np.float32) for v in zero)
    mixer.write_state(2, *other)

    u = rng.random(n).astype(np.float32) * np.float32(0.999999)
    random.copy_(torch.from_numpy(u))
    torch.cuda.synchronize()
    first = Buffers(torch, model, tokens, n)
    with torch.cuda.stream(stream):
        forward(first, prompt, tokens,
                lambda b: mixer.run_device(b.rows.data_ptr(), b.mixed.data_ptr(), tokens, offsets.data_ptr(), n,
                                           fresh.data_ptr(), new.data_ptr(), s),
                lambda v: v.index_select(0, ends))
    mixer.sync(s)
    moe.sync(s)
    check(first, prompt.cpu().numpy(), LENGTHS, [zero] * n, u)

    # one more token of each sequence: the draw feeds the next replay
    b = Buffers(torch, model, n, n)
    torch.cuda.synchronize()

    def step():
        forward(b, drawn, n,
                lambda b: mixer.step_device(b.rows.data_ptr(), b.mixed.data_ptr(), n, new.data_ptr(),
                                            new.data_ptr(), s), lambda v: v)

    before = [mixer.read_state(slot) for slot in slots]
    ids = drawn.cpu().numpy().copy()
    with torch.cuda.stream(stream):
        step()  # eager once: torch's own workspaces exist when the graph is captured
    mixer.sync(s)
    check(b, ids, [1] * n, before, u)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        step()
    for replay in range(3):
        u = rng.random(n).astype(np.float32) * np.float32(0.999999)
        random.copy_(torch.from_numpy(u))
        before = [mixer.read_state(slot) for slot in slots]
        ids = drawn.cpu().numpy().copy()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        mixer.sync()
        check(b, ids, [1] * n, before, u)
    for got, want in zip(mixer.read_state(2), other):
        assert np.array_equal(got, want)
