"""Log probabilities, entropy and top alternatives on the device against their definition in 64 bits.

Bounds, with d = x - max and weights p: an exponential's relative error is that of d and of its product with log2 e
(1.5 |d| 2^-23) and of the exponential (2^-22); its sums are in 64 bits, those of e d over a lane's 32 logits in
single precision (34 2^-24).  A result is rounded once."""
import numpy as np
import pytest

from llambda_amd.sampling import HipTokenScorer, SamplingError
from test_batch_sampling_gpu import head_like

pytestmark = pytest.mark.gpu


def reference(row, top):
    """(log probabilities, entropy, top tokens, bounds of the log sum and of the entropy), None if there are none."""
    x = row.astype(np.float64)
    if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any():
        return None
    d = x - x.max()
    e = np.exp(d)
    s = e.sum()
    lp = d - np.log(s)
    p = e / s
    f = np.where(p > 0, d, 0)
    rel = 1.5 * np.abs(f) * 2.0 ** -23 + 2.0 ** -22
    log_bound = (p * rel).sum()
    spread = (p * np.abs(f)).sum()
    h = np.log(s) + spread
    h_bound = log_bound * (1 + spread) + (p * np.abs(f) * (rel + 34 * 2.0 ** -24)).sum() + abs(h) * 2.0 ** -24
    order = np.argsort(-x, kind="stable")[:top]
    return lp, h, order[x[order] > -np.inf], log_bound, h_bound


def check(scorer, x, given=None, top=0):
    got = scorer.score(x, given, top)
    given = np.empty((len(x), 0), int) if given is None else np.asarray(given).reshape(len(x), -1)
    for i, row in enumerate(x):
        want = reference(row, top)
        if want is None:
            assert np.all(np.isnan(got.log_probs[i])) and np.isnan(got.entropy[i])
            assert np.all(got.top_tokens[i] == -1) and np.all(np.isnan(got.top_log_probs[i]))
            continue
        lp, h, order, log_bound, h_bound = want
        assert abs(got.entropy[i] - h) <= h_bound, (i, got.entropy[i], h, h_bound)
        n = len(order)
        assert got.top_tokens[i].tolist() == order.tolist() + [-1] * (top - n)
        assert np.all(got.top_log_probs[i, n:] == -np.inf)
        for g, w in ((got.log_probs[i], lp[given[i]]), (got.top_log_probs[i, :n], lp[order])):
            both = np.isfinite(w)
            assert np.array_equal(g[~both], w[~both])
            assert np.all(np.abs(g[both] - w[both]) <= log_bound + np.abs(w[both]) * 2.0 ** -24)


@pytest.fixture(scope="module")
def scorer(hip):
    s = HipTokenScorer(262144, 40, 64)
    yield s
    s.close()


@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 2), (2, 63), (5, 255), (1, 2048), (3, 2049), (2, 4095), (7, 5001),
                                         (2, 32000), (3, 128256), (2, 128257), (1, 262144), (40, 1000)])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
def test_rows_like_a_head(scorer, rows, vocab, top):
    rng = np.random.default_rng(1)
    x = head_like(rng, rows, vocab)
    check(scorer, x, rng.integers(0, vocab, size=(rows, 3)), top)


@pytest.mark.parametrize("top", [1, 3, 20, 64])
def test_equal_and_ordered_logits(scorer, top):
    """Ties go to the lowest index, wherever they lie; neighbours hold the largest."""
    rng = np.random.default_rng(2)
    n = 10000
    rows = [np.zeros(n), np.full(n, -3.5), np.arange(n) * 0.001, -np.arange(n) * 0.001,
            rng.integers(0, 3, size=n), rng.integers(0, 200, size=n) * 0.125, np.where(np.arange(n) % 7 == 0, 0.0, -0.0),
            np.where(np.arange(n) == 5000, 30.0, 0.0), np.where(np.arange(n) < 100, 2.0, 1.0)]
    check(scorer, np.array(rows, dtype=np.float32), np.full((len(rows), 1), 5000), top)


@pytest.mark.parametrize("top", [1, 5, 64])
def test_masked_logits(scorer, top):
    """-inf and the type's lowest value; rows without a distribution stand alone."""
    rng = np.random.default_rng(3)
    n = 5000
    x = head_like(rng, 9, n)
    low = np.finfo(np.float32).min
    x[0, 2048:] = -np.inf
    x[1, :] = -np.inf
    x[1, 4321] = 1.5
    x[2, :] = -np.inf
    x[3, 17] = np.nan
    x[4, 4999] = np.inf
    x[5, rng.random(n) < 0.999] = -np.inf
    x[6, :] = low
    x[6, 70:74] = 0
    x[7, rng.random(n) < 0.5] = low
    x[8, :] = low
    given = rng.integers(0, n, size=(9, 4))
    given[:, 0] = 4321
    check(scorer, x, given, top)


def test_certain_and_large(scorer):
    """A token that is nearly certain: what is left shows; logits far from zero; wide rows."""
    n = 4000
    x = np.zeros((5, n), dtype=np.float32)
    x[0, 3] = 26.0        # the others' weight is 2e-8 of it
    x[1, 7], x[1, 8] = 20.0, 2.0
    x[2] = np.linspace(-1000, 1000, n)
    x[3] = np.linspace(30000, 30010, n)
    x[4] = np.linspace(-3e38, 3e38, n)
    check_rows = [[3, 4], [7, 8], [n - 1, 0], [n - 1, n // 2], [n - 1, n - 2]]
    got = scorer.score(x, check_rows, 5)
    for i, row in enumerate(x):
        lp, h, order, log_bound, h_bound = reference(row, 5)
        assert got.top_tokens[i].tolist() == order.tolist()
        w = lp[check_rows[i]]
        assert np.all(np.abs(got.log_probs[i] - w) <= log_bound + np.abs(w) * 2.0 ** -24)
        assert abs(got.entropy[i] - h) <= h_bound
    # the sum keeps what is next to 1
    want = reference(x[0], 1)[0][3]
    assert want < 0 and abs(got.log_probs[0, 0] - want) <= 1e-5 * -want


def test_device_rows_strides_and_results_left_out(hip):
    import torch
    rng = np.random.default_rng(4)
    rows, vocab, stride = 6, 3001, 3100
    x = np.zeros((rows, stride), dtype=np.float32)
    x[:, :vocab] = head_like(rng, rows, vocab)
    x[:, vocab:] = np.nan
    d = torch.from_numpy(x).cuda()
    given = torch.tensor([[1, -1, 3000], [0, 3001, 5]] * 3, dtype=torch.int32, device="cuda")
    lp = torch.zeros((rows, 3), device="cuda")
    entropy = torch.zeros(rows, device="cuda")
    tokens = torch.zeros((rows, 7), dtype=torch.int32, device="cuda")
    scorer = HipTokenScorer(4000, rows, 10)
    torch.cuda.synchronize()
    scorer.score_device(d.data_ptr(), rows, given_ptr=given.data_ptr(), given=3, top=7, count=vocab, stride=stride,
                        log_probs_ptr=lp.data_ptr(), top_tokens_ptr=tokens.data_ptr())
    scorer.score_device(d.data_ptr(), rows, count=vocab, stride=stride, entropy_ptr=entropy.data_ptr())
    torch.cuda.synchronize()
    for i in range(rows):
        want = reference(x[i, :vocab], 7)
        assert tokens[i].tolist() == want[2].tolist()
        assert abs(float(entropy[i]) - want[1]) <= want[4]
        for g, t in zip(lp[i].tolist(), given[i].tolist()):
            if 0 <= t < vocab:
                assert abs(g - want[0][t]) <= want[3] + abs(want[0][t]) * 2.0 ** -24
            else:
                assert np.isnan(g)


def test_calls_that_are_refused(hip):
    import torch
    d = torch.zeros((2, 100), device="cuda")
    out = torch.zeros(200, device="cuda")
    scorer = HipTokenScorer(100, 2, 5)
    p, o = d.data_ptr(), out.data_ptr()
    torch.cuda.synchronize()
    for args, more, message in [
            ((0, 2), dict(entropy_ptr=o), "null argument"), ((p, 0), dict(entropy_ptr=o), "0 rows"),
            ((p, 3), dict(entropy_ptr=o), "3 rows"), ((p, 2), dict(count=101, entropy_ptr=o), "101 logits do not fit"),
            ((p, 2), dict(count=0, entropy_ptr=o), "0 logits do not fit"),
            ((p, 2), dict(stride=99, entropy_ptr=o), "at a stride of 99"), ((p, 2), dict(top=6, top_tokens_ptr=o), "6 top"),
            ((p, 2), dict(top=5), "null top tokens"), ((p, 2), dict(given=1, given_ptr=o), "null given tokens or"),
            ((p, 2), dict(given=1, log_probs_ptr=o), "null given tokens or"),
            ((p, 2), dict(given=5000, given_ptr=o, log_probs_ptr=o), "5000 given tokens"),
            ((p + 2, 2), dict(entropy_ptr=o), "4-byte aligned")]:
        with pytest.raises(SamplingError, match=message):
            scorer.score_device(*args, **more)
    torch.cuda.synchronize()
    assert not out.any()


def test_captured_and_on_two_streams(hip):
    import torch
    rng = np.random.default_rng(5)
    rows, vocab = 9, 20000
    scorer = HipTokenScorer(vocab, rows, 8)
    d = torch.zeros((rows, vocab), device="cuda")
    given = torch.zeros((rows, 1), dtype=torch.int32, device="cuda")
    results = [[torch.zeros((rows, 1), device="cuda"), torch.zeros(rows, device="cuda"),
                torch.zeros((rows, 8), dtype=torch.int32, device="cuda"), torch.zeros((rows, 8), device="cuda")]
               for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in range(2)]

    def call(r, stream):
        scorer.score_device(d.data_ptr(), rows, given_ptr=given.data_ptr(), given=1, top=8, log_probs_ptr=r[0].data_ptr(),
                            entropy_ptr=r[1].data_ptr(), top_tokens_ptr=r[2].data_ptr(), top_log_probs_ptr=r[3].data_ptr(),
                            stream=stream.cuda_stream)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    call(results[0], streams[0])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=streams[0], capture_error_mode="relaxed"):
        call(results[0], streams[0])
    for _ in range(3):
        x = head_like(rng, rows, vocab)
        g = rng.integers(0, vocab, size=(rows, 1)).astype(np.int32)
        d.copy_(torch.from_numpy(x))
        given.copy_(torch.from_numpy(g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        call(results[1], streams[0])
        call(results[2], streams[1])
        torch.cuda.synchronize()
        host = scorer.score(x, g, 8)
        for r in results:
            for t, h in zip(r, (host.log_probs, host.entropy, host.top_tokens, host.top_log_probs)):
                assert np.array_equal(t.cpu().numpy(), h)
        check(scorer, x, g, 8)
