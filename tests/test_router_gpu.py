"""Routing to experts (llambda_hip_router_*, and MoE layers gated by a router)
against the definition in 64 bits.  Indices are equal; a weight is a quotient
formed in 64 bits and rounded once to single precision, so it is off by at
most 2^-24 of its value, and by 2^-23 counting the two sides' exponentials."""
import numpy as np
import pytest

import oracle
from llambda_amd import native, synthetic
from llambda_amd.hip_backend import HipBackendError
from llambda_amd.moe import (HipMoeSession, HipRouter, Routing, synthetic_nemotron_h,
                             synthetic_qwen3next)

pytestmark = pytest.mark.gpu

FLT_MAX = np.finfo(np.float32).max


def reference(r: Routing, logits):
    """(indices, weights) [tokens][top_k] in 64 bits."""
    idx = np.full((len(logits), r.top_k), -1, np.int64)
    w = np.zeros((len(logits), r.top_k))
    bias = np.zeros(r.experts) if r.bias is None else r.bias.astype(np.float64)
    size = r.experts // r.groups
    for t, row in enumerate(logits):
        open_ = row > -FLT_MAX  # false for NaN
        l = np.where(open_, row, -np.inf).astype(np.float64)
        with np.errstate(all="ignore"):
            if r.score == "softmax":
                top = l.max()
                s = np.where(l == top, 1.0, np.exp(l - top))
                s = np.where(open_, s, 0.0)
                s = s / s.sum()
            else:
                s = np.where(open_, 1 / (1 + np.exp(-l)), 0.0)
        choice = s + bias
        open_ = open_ & ~np.isnan(choice)
        if r.groups > 1:
            rank = []
            for g in range(r.groups):
                part = slice(g * size, (g + 1) * size)
                best = np.sort(choice[part][open_[part]])[::-1][:r.group_rank]
                rank.append(best.sum() if best.size else -np.inf)
            rank = np.array(rank)
            best = [g for g in np.argsort(-rank, kind="stable")[:r.top_groups] if rank[g] > -np.inf]
            open_ = open_ & np.isin(np.arange(r.experts) // size, best)
        # without a bias the order is the logits', also where the scores round to the same number
        by = choice if r.bias is not None or r.groups > 1 else l
        order = [e for e in np.argsort(np.where(open_, -by, np.inf), kind="stable") if open_[e]][:r.top_k]
        idx[t, :len(order)] = order
        w[t, :len(order)] = s[order]
        total = w[t].sum()
        if r.weights_norm and total > 0:
            w[t] /= total
        w[t] *= float(np.float32(r.weights_scale))
    return idx, w


def check(r, logits, got=None):
    idx, w = got or HipRouter(r).run(logits)
    want_idx, want_w = reference(r, logits)
    assert np.array_equal(idx, want_idx)
    assert np.all(np.abs(w - want_w) <= 2.0 ** -23 * np.abs(want_w))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("experts,top_k", [(1, 1), (5, 5), (64, 1), (65, 7), (128, 6), (200, 64), (512, 10),
                                           (1000, 33), (1024, 8)])
def test_top_k(hip, score, bias, experts, top_k):
    rng = np.random.default_rng(experts)
    logits = (rng.normal(size=(13, experts)) * 2).astype(np.float32)
    b = (rng.normal(size=experts) * 0.2).astype(np.float32) if bias else None
    for norm, scale in ((True, 2.5), (False, 1.0)):
        check(Routing(experts, top_k, score=score, bias=b, weights_norm=norm, weights_scale=scale), logits)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(256, 8, 4, 8), (96, 3, 2, 5), (64, 64, 9, 9),
                                                             (1024, 4, 1, 20), (60, 5, 5, 6), (17, 17, 3, 2)])
@pytest.mark.parametrize("group_rank", [1, 2])
def test_groups(hip, score, bias, experts, groups, top_groups, top_k, group_rank):
    rng = np.random.default_rng(experts + groups)
    logits = (rng.normal(size=(9, experts)) * 2).astype(np.float32)
    b = (rng.normal(size=experts) * 0.2).astype(np.float32) if bias else None
    check(Routing(experts, top_k, score=score, bias=b, groups=groups, top_groups=top_groups,
                  group_rank=group_rank), logits)


@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_equal_and_infinite_logits(hip, groups, bias, score):
    rng = np.random.default_rng(5)
    E = 128
    logits = (rng.normal(size=(12, E)) * 2).astype(np.float32)
    logits[0] = 1.5                              # all equal: the lowest indices
    logits[1] = np.round(logits[1])              # many equal
    logits[2, ::2] = -FLT_MAX                    # masked by the type's lowest value
    logits[3, 1:] = -np.inf                      # one expert left
    logits[4] = np.nan                           # none
    logits[5, 10:20] = np.nan
    logits[6] = -FLT_MAX
    logits[7, 40:80] = -np.inf
    logits[8] = -0.0
    logits[8, 7] = 0.0
    logits[9] = -30 + np.arange(E) / 64          # far from the others' range
    logits[10, 33] = np.inf
    logits[11, 64:] = np.nan
    b = np.repeat((rng.normal(size=E // 8) * 0.2).astype(np.float32), 8) if bias else None
    check(Routing(E, 6, score=score, bias=b, groups=groups, top_groups=max(1, groups // 2), group_rank=2), logits)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_that_round_to_the_same_number(hip, score):
    """Without a bias and groups they rank by their logits, else they are equals."""
    rng = np.random.default_rng(13)
    logits = rng.normal(size=(3, 64)).astype(np.float32)
    logits[0, [5, 9, 40, 41]] = [40, 50, 60, 45]     # sigmoids of 1
    logits[1] = -2000 - rng.permutation(64)          # softmax scores of 0 beside the highest's 1
    logits[1, 33] = 0
    logits[2] = rng.permutation(64) - 900            # sigmoids of 0
    plain, zeros = Routing(64, 4, score=score), Routing(64, 4, score=score, bias=np.zeros(64, np.float32))
    for r in (plain, zeros, Routing(64, 4, score=score, groups=4, top_groups=4)):
        check(r, logits)
    row = 0 if score == "sigmoid" else 1
    by_logit = np.argsort(-logits[row], kind="stable")[:4]
    assert HipRouter(plain).run(logits)[0][row].tolist() == by_logit.tolist()
    first = [5, 9, 40, 41] if score == "sigmoid" else [33, 0, 1, 2]
    assert HipRouter(zeros).run(logits)[0][row].tolist() == first


def test_biases_that_are_not_finite(hip):
    rng = np.random.default_rng(6)
    logits = rng.normal(size=(4, 96)).astype(np.float32)
    bias = np.zeros(96, np.float32)
    bias[[3, 50]] = np.nan   # never chosen
    bias[70] = np.inf        # always
    bias[80] = -np.inf       # last
    check(Routing(96, 5, score="sigmoid", bias=bias), logits)


@pytest.mark.parametrize("experts,groups", [(96, 8), (1024, 16)])
def test_infinite_biases_in_groups(hip, experts, groups):
    """A group that holds +inf and -inf is as one that holds +inf; no more groups open than top_groups."""
    rng = np.random.default_rng(15)
    size = experts // groups
    logits = rng.normal(size=(5, experts)).astype(np.float32)
    bias = np.full(experts, -np.inf, np.float32)
    bias[2 * size:] = 0
    bias[size + 3] = np.inf  # the second group: one of +inf, the others of -inf
    r = Routing(experts, 6, score="sigmoid", bias=bias, groups=groups, top_groups=2, group_rank=2)
    idx, w = HipRouter(r).run(logits)
    s = 1 / (1 + np.exp(-logits.astype(np.float64)))
    for t in range(len(logits)):
        rank = np.sort(s[t].reshape(groups, size), axis=1)[:, -2:].sum(1)
        g = 2 + int(rank[2:].argmax())
        best = g * size + np.argsort(-s[t, g * size:(g + 1) * size], kind="stable")[:5]
        want = [size + 3, *best]
        assert idx[t].tolist() == want
        share = s[t, want] / s[t, want].sum()
        assert np.all(np.abs(w[t] - share) <= 2.0 ** -23 * share)


def test_scores_that_underflow(hip):
    """Weights whose sum is zero stay as they are (zeros)."""
    logits = np.full((2, 64), -1e30, np.float32)
    logits[1, 5] = 0
    check(Routing(64, 3, score="sigmoid"), logits)
    check(Routing(64, 3, score="softmax", weights_norm=False), logits)


def test_device_runs_on_streams_and_in_a_graph(hip):
    import torch
    rng = np.random.default_rng(7)
    r = Routing(256, 8, score="sigmoid", bias=(rng.normal(size=256) * 0.1).astype(np.float32), groups=8,
                top_groups=4, group_rank=2)
    router = HipRouter(r)
    tokens = 301
    x = torch.zeros(tokens * 256 + 1, device="cuda")[1:]  # 4-byte aligned
    idx = torch.empty((tokens, 8), dtype=torch.int32, device="cuda")
    w = torch.empty((tokens, 8), device="cuda")
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        router.run_device(x.data_ptr(), idx.data_ptr(), w.data_ptr(), tokens, stream.cuda_stream)
    for k in range(3):
        logits = rng.normal(size=(tokens, 256)).astype(np.float32)
        x.copy_(torch.from_numpy(logits.reshape(-1)))
        torch.cuda.synchronize()
        if k == 1:
            router.run_device(x.data_ptr(), idx.data_ptr(), w.data_ptr(), tokens)
        else:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        check(r, logits, (idx.cpu().numpy().astype(np.int64), w.cpu().numpy()))


def _experts(layer, x):
    """[tokens][experts][hidden] outputs of every expert and the shared one's, in 64 bits, with the sums of
    the absolute products."""
    from llambda_amd.moe import QWEN3NEXT
    H, E, F, Fs = layer.hidden, layer.expert_count, layer.expert_ffn, layer.shared_ffn

    def dense(p, rows, cols):
        return oracle.dequantize(p[0], p[1], rows * cols).reshape(rows, cols).astype(np.float64)

    def ffn(gate, up, down):
        u = up @ x.T.astype(np.float64)
        if gate is not None:
            g = gate @ x.T.astype(np.float64)
            u = u * g / (1 + np.exp(-g))
        else:
            u = np.maximum(u, 0) ** 2
        return (down @ u).T, (np.abs(down) @ np.abs(u)).T

    swiglu = layer.variant == QWEN3NEXT
    up, down = dense(layer.up, E * F, H), dense(layer.down, E * H, F)
    gate = dense(layer.gate, E * F, H) if swiglu else None
    out = [ffn(gate[e * F:(e + 1) * F] if swiglu else None, up[e * F:(e + 1) * F], down[e * H:(e + 1) * H])
           for e in range(E)]
    shared = ffn(dense(layer.shared_gate, Fs, H) if swiglu else None, dense(layer.shared_up, Fs, H),
                 dense(layer.shared_down, H, Fs))
    if swiglu:
        s = 1 / (1 + np.exp(-(x.astype(np.float64) @ layer.shared_gate_inp.astype(np.float64))))
        shared = tuple(v * s[:, None] for v in shared)
    return np.stack([o[0] for o in out], 1), np.stack([o[1] for o in out], 1), shared


@pytest.mark.parametrize("tokens", [1, 2, 37, 300])
@pytest.mark.parametrize("variant", ["qwen3next", "nemotron"])
def test_moe_layer_with_a_router(hip, variant, tokens):
    """The layer's experts and weights are the router's for the logits that it returns, its outputs the
    experts' weighted sums; without the router it is as before."""
    rng = np.random.default_rng(8)
    if variant == "qwen3next":
        layer = synthetic_qwen3next(rng, hidden=512, experts=16, top_k=4, ffn=256, shared_ffn=256)
    else:
        layer = synthetic_nemotron_h(rng, hidden=256, experts=16, top_k=4, ffn=96, shared_ffn=160)
    x = synthetic.activations(rng, tokens, layer.hidden)
    session = HipMoeSession(layer)
    before = session.run(x, with_routing=True)
    r = Routing(16, 4, score="sigmoid", bias=(rng.normal(size=16) * 0.3).astype(np.float32), groups=4,
                top_groups=2, group_rank=2, weights_norm=True, weights_scale=1.75)
    router = HipRouter(r)
    session.set_router(router)
    router.close()  # the session keeps what it needs
    y, idx, w, logits = session.run(x, with_routing=True)
    check(r, logits, (idx, w))
    plain = x.astype(np.float64) @ layer.router.astype(np.float64).T
    assert np.abs(logits - plain).max() <= 1e-4 * np.abs(plain).max()
    experts, sizes, shared = _experts(layer, x)
    want, size = shared[0].copy(), shared[1].copy()
    for t in range(tokens):
        want[t] += (w[t, :, None] * experts[t, idx[t]]).sum(0)
        size[t] += (w[t, :, None] * sizes[t, idx[t]]).sum(0)
    assert np.all(np.abs(y - want) <= 1e-4 * size)
    session.set_router(None)
    for a, b in zip(before, session.run(x, with_routing=True)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("experts,top_k", [(64, 8), (128, 6), (200, 16), (512, 10), (1000, 64)])
@pytest.mark.parametrize("kind", ["qwen3next", "no shared", "nemotron", "latent"])
def test_moe_layers_of_many_experts_with_a_router(hip, kind, experts, top_k):
    rng = np.random.default_rng(18)
    if kind in ("qwen3next", "no shared"):
        layer = synthetic_qwen3next(rng, hidden=256, experts=experts, top_k=top_k, ffn=256,
                                    shared_ffn=0 if kind == "no shared" else 256)
    else:
        layer = synthetic_nemotron_h(rng, hidden=256, experts=experts, top_k=top_k, ffn=32, shared_ffn=64,
                                     **(dict(latent_in=64, latent_out=64) if kind == "latent" else {}))
    session = HipMoeSession(layer)
    for routing in (Routing(experts, top_k, weights_norm=False, weights_scale=3),
                    Routing(experts, top_k, score="sigmoid", bias=(rng.normal(size=experts) * 0.3).astype(np.float32),
                            groups=8, top_groups=5, group_rank=2)):
        router = HipRouter(routing)
        session.set_router(router)
        for tokens in (1, 3, 70):
            x = synthetic.activations(rng, tokens, layer.hidden)
            y, idx, w, logits = session.run(x, with_routing=True)
            check(routing, logits, (idx, w))
            assert np.isfinite(y).all()
            alone = router.run(logits)
            assert np.array_equal(alone[0], idx) and np.array_equal(alone[1], w)


def test_moe_layer_with_the_reference_gating_as_a_router(hip):
    """Qwen3Next's gating is a sigmoid router without bias and groups."""
    rng = np.random.default_rng(9)
    layer = synthetic_qwen3next(rng, hidden=512, experts=32, top_k=4, ffn=256, shared_ffn=256)
    session = HipMoeSession(layer)
    for tokens in (1, 50):
        x = synthetic.activations(rng, tokens, 512)
        session.set_router(None)
        y, idx, w, _ = session.run(x, with_routing=True)
        session.set_router(HipRouter(Routing(32, 4, score="sigmoid")))
        y2, idx2, w2, _ = session.run(x, with_routing=True)
        assert np.array_equal(idx, idx2)
        # the reference rounds the sigmoids, their sum and the quotients to single: 2^-24 each of at most
        # k + 2 values in a row, and the outputs move by as much of the weighted sums
        assert np.all(np.abs(w - w2) <= 7 * 2.0 ** -24 * np.abs(w))
        assert np.abs(y - y2).max() <= 16 * 2.0 ** -24 * np.abs(y).max() * 4


def test_captured_gating_outlives_a_change_of_router(hip):
    """A graph keeps the router that it was captured with."""
    import torch
    rng = np.random.default_rng(12)
    layer = synthetic_qwen3next(rng, hidden=512, experts=16, top_k=4, ffn=256, shared_ffn=256)
    session = HipMoeSession(layer)
    biases = [(rng.normal(size=16) * 2).astype(np.float32) for _ in range(4)]
    x = torch.from_numpy(synthetic.activations(rng, 3, 512)).cuda()
    y = torch.zeros(3, 512, device="cuda")
    want = []
    for b in biases:
        session.set_router(HipRouter(Routing(16, 4, bias=b)))
        want.append(session.run(x.cpu().numpy()))
    assert len({w.tobytes() for w in want}) == len(want)
    stream = torch.cuda.Stream()
    graphs = []
    for b in biases[:2]:
        session.set_router(HipRouter(Routing(16, 4, bias=b)))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
            session.run_device(x.data_ptr(), y.data_ptr(), 3, stream.cuda_stream)
        graphs.append(graph)
    for b in biases[2:] + [None]:
        session.set_router(None if b is None else HipRouter(Routing(16, 4, bias=b)))
        for graph, w in zip(graphs, want):
            graph.replay()
            torch.cuda.synchronize()
            assert np.array_equal(y.cpu().numpy(), w)


def test_moe_layer_errors_with_a_router(hip):
    from llambda_amd.moe import MoeLayerInputError
    rng = np.random.default_rng(10)
    layer = synthetic_qwen3next(rng, hidden=512, experts=8, top_k=4, ffn=256, shared_ffn=256)
    layer.router[:] = -1.0
    layer.router[5] = 0.0
    session = HipMoeSession(layer)
    session.set_router(HipRouter(Routing(8, 4, score="sigmoid")))
    x = np.full((2, 512), 1e36, np.float32)  # logits of -inf but one
    with pytest.raises(MoeLayerInputError, match="fewer than top-k"):
        session.run(x)
    with pytest.raises(HipBackendError, match="a router of 3 of 8 experts on a layer of 4 of 8"):
        session.set_router(HipRouter(Routing(8, 3)))
    assert native.lib().llambda_hip_moe_session_set_router(None, None) == -1


def test_refusals(hip):
    import torch
    router = HipRouter(Routing(8, 2))
    x = torch.zeros(8, device="cuda")
    for args, text in [((0, x.data_ptr(), x.data_ptr(), 1), "null"), ((x.data_ptr(), 0, x.data_ptr(), 1), "null"),
                       ((x.data_ptr(), x.data_ptr(), 0, 1), "null"),
                       ((x.data_ptr(), x.data_ptr(), x.data_ptr(), 0), "bad batch"),
                       ((x.data_ptr() + 1, x.data_ptr(), x.data_ptr(), 1), "aligned")]:
        with pytest.raises(HipBackendError, match=text):
            router.run_device(*args)
    router.close()
    with pytest.raises(HipBackendError, match="closed"):
        router.run(np.zeros((1, 8), np.float32))
