"""Sampling of a batch (llambda_hip_batch_sampler_*) against its definition in
64 bits.  The weights are good to 2e-9 and summed exactly in steps of 2^-44, so
the tokens are equal unless a random number lies within about 2e-9 of a
boundary."""
import numpy as np
import pytest

from llambda_amd.sampling import HipBatchSampler, SamplingError

pytestmark = pytest.mark.gpu

FLT_MAX = np.finfo(np.float32).max


def reference(row, u, t=1.0, k=0, p=1.0, m=0.0):
    u, t, p, m = (float(np.float32(v)) for v in (u, t, p, m))
    n = row.size
    if (not 0 <= t < np.inf or not 0 < p <= 1 or not 0 <= m <= 1 or not 0 <= u < 1 or k < 0
            or np.isnan(row).any() or not (row > -np.inf).any()):
        return -1
    if t == 0:
        k, t = 1, 1.0
    order = np.argsort(-row, kind="stable")
    v = row[order].astype(np.float64)
    with np.errstate(invalid="ignore"):
        w = np.where(v == v[0], 1.0, np.exp(v / t - v[0] / t))
    if 0 < k < n:
        w[k:] = 0
    if p < 1:
        c = np.cumsum(w)
        w = np.where(np.concatenate([[0], c[:-1]]) < p * c[-1], w, 0)
    w = np.where(w >= m, w, 0)
    full = np.zeros(n)
    full[order] = w
    c = np.cumsum(full)
    return int((c <= u * c[-1]).sum())


def head_like(rng, rows, n):
    x = rng.normal(size=(rows, n)) * 3
    for r in x:
        r[rng.integers(0, n, size=20)] += 6
    return x.astype(np.float32)


def check(sampler, x, u, t=1.0, k=0, p=1.0, m=0.0):
    rows = len(x)
    each = [np.broadcast_to(np.asarray(v), (rows,)) for v in (u, t, k, p, m)]
    got = sampler.sample(x, random_value=u, temperature=t, top_k=k, top_p=p, min_p=m)
    want = [reference(r, *(v[i] for v in each)) for i, r in enumerate(x)]
    assert got.tolist() == want


@pytest.fixture(scope="module")
def sampler(hip):
    s = HipBatchSampler(262144, 64)
    yield s
    s.close()


FILTERS = [dict(), dict(k=1), dict(k=40), dict(k=500), dict(k=5000), dict(p=0.9), dict(p=0.02), dict(p=0.9999),
           dict(m=0.05), dict(m=1e-6), dict(m=1.0), dict(k=40, p=0.9, m=0.05), dict(k=3000, p=0.8, m=0.01),
           dict(p=0.7, m=0.2), dict(p=0.5, m=1e-7), dict(k=200, p=0.5)]


@pytest.mark.parametrize("filters", FILTERS, ids=str)
@pytest.mark.parametrize("n", [1, 2, 255, 256, 257, 1000, 32001, 128256])
def test_rows(sampler, filters, n):
    rng = np.random.default_rng(n)
    rows = 7 if n > 20000 else 40
    x = head_like(rng, rows, n)
    check(sampler, x, rng.random(rows).astype(np.float32) * np.float32(0.999999),
          t=rng.choice([0.25, 0.7, 1.0, 2.0], size=rows).astype(np.float32), **filters)


def test_each_row_its_own_parameters(sampler):
    rng = np.random.default_rng(3)
    n, rows = 50000, 64
    x = head_like(rng, rows, n)
    check(sampler, x, rng.random(rows).astype(np.float32) * np.float32(0.999999),
          t=rng.choice([0.0, 0.5, 1.0, 3.0], size=rows), k=rng.choice([0, 1, 20, 400, 100000], size=rows),
          p=rng.choice([0.3, 0.9, 1.0], size=rows), m=rng.choice([0.0, 0.0, 0.1, 0.5], size=rows))


@pytest.mark.parametrize("filters", FILTERS, ids=str)
def test_equal_logits(sampler, filters):
    """Ties go to the lower index, in lists and where they outgrow one."""
    rng = np.random.default_rng(4)
    n = 30011
    x = np.zeros((6, n), np.float32)
    x[1] = rng.integers(0, 3, size=n)
    x[2, ::7] = 5
    x[3] = np.round(rng.normal(size=n) * 3)
    x[4] = np.where(rng.random(n) < 0.5, 0.0, -0.0)
    x[5, 20000:] = 1
    check(sampler, x, [0.0, 0.3, 0.9999, 0.5, 0.77, 0.25], t=[1, 1, 0.5, 2, 1, 1], **filters)


@pytest.mark.parametrize("filters", FILTERS, ids=str)
def test_masked_and_infinite_logits(sampler, filters):
    rng = np.random.default_rng(5)
    n = 5000
    x = head_like(rng, 9, n)
    x[0, 17:] = -np.inf
    x[1, :] = -np.inf
    x[1, 4321] = -3
    x[2, ::2] = -FLT_MAX
    x[3] = -FLT_MAX
    x[4, [100, 2000]] = np.inf
    x[5, :4990] = -np.inf
    x[6] *= 1e30
    x[7] *= 1e-30
    x[8, 1000:] = -1e30
    check(sampler, x, rng.random(9).astype(np.float32) * np.float32(0.999999), **filters)


@pytest.mark.parametrize("u", [0.0, 1 - 2.0 ** -24])
@pytest.mark.parametrize("filters", FILTERS, ids=str)
def test_ends_of_the_random_range(sampler, filters, u):
    check(sampler, head_like(np.random.default_rng(6), 5, 9999), [u] * 5, **filters)


@pytest.mark.parametrize("t", [1e-38, 1e-3, 1e3, 1e38])
def test_extreme_temperatures(sampler, t):
    x = head_like(np.random.default_rng(7), 4, 9999)
    for filters in FILTERS:
        check(sampler, x, [0.1, 0.5, 0.9, 0.99], t=t, **filters)


def test_longest_rows(sampler):
    rng = np.random.default_rng(8)
    x = head_like(rng, 4, 262144)
    for filters in (dict(), dict(k=1024), dict(p=0.95), dict(k=40, p=0.95, m=0.05)):
        check(sampler, x, [0.2, 0.4, 0.6, 0.8], **filters)


def test_rows_without_a_token_and_bad_parameters_on_the_device(hip):
    """The device form marks them with -1 and serves the others."""
    import torch
    rng = np.random.default_rng(9)
    n, rows = 1001, 12
    x = head_like(rng, rows, n)
    x[0, 500] = np.nan
    x[1] = -np.inf
    u = np.full(rows, 0.5, np.float32)
    t, k = np.ones(rows, np.float32), np.full(rows, 40, np.int32)
    p, m = np.full(rows, 0.9, np.float32), np.full(rows, 0.05, np.float32)
    u[2], u[3], t[4], t[5], k[6], p[7], p[8], m[9], m[10] = 1.0, np.nan, -1, np.inf, -1, 0, 1.5, -0.1, np.nan
    s = HipBatchSampler(n, rows)
    d = [torch.from_numpy(a).cuda() for a in (x, u, t, k, p, m)]
    tokens = torch.full((rows + 1,), 77, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    s.sample_device(d[0].data_ptr(), rows, tokens.data_ptr(), d[1].data_ptr(), temperature_ptr=d[2].data_ptr(),
                    top_k_ptr=d[3].data_ptr(), top_p_ptr=d[4].data_ptr(), min_p_ptr=d[5].data_ptr())
    torch.cuda.synchronize()
    want = [reference(x[i], u[i], t[i], int(k[i]), p[i], m[i]) for i in range(rows)]
    assert want[:11] == [-1] * 11 and want[11] >= 0
    assert tokens.tolist() == want + [77]


def test_defaults_shorter_rows_streams_and_a_graph(hip):
    import torch
    rng = np.random.default_rng(10)
    n, rows = 40001, 6
    s = HipBatchSampler(65536, 8)
    flat = torch.zeros(rows * n + 1, device="cuda")
    x, u = flat[1:], torch.zeros(rows, device="cuda")  # 4-byte aligned
    a, b = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
    p = torch.full((rows,), 0.9, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=streams[0], capture_error_mode="relaxed"):
        s.sample_device(x.data_ptr(), rows, a.data_ptr(), u.data_ptr(), count=n, stream=streams[0].cuda_stream)
    for _ in range(4):
        logits = head_like(rng, rows, n)
        r = rng.random(rows).astype(np.float32) * np.float32(0.999999)
        x.copy_(torch.from_numpy(logits.reshape(-1)))
        u.copy_(torch.from_numpy(r))
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        torch.cuda.synchronize()
        for k in range(3):  # eager calls on two streams share the workspace in order
            s.sample_device(x.data_ptr(), rows, b.data_ptr(), u.data_ptr(), top_p_ptr=p.data_ptr(), count=n,
                            stream=streams[k % 2].cuda_stream)
        torch.cuda.synchronize()
        assert a.tolist() == [reference(logits[i], r[i]) for i in range(rows)]
        assert b.tolist() == [reference(logits[i], r[i], p=0.9) for i in range(rows)]


@pytest.mark.parametrize("n", [3, 700])
def test_many_rows(hip, n):
    rng = np.random.default_rng(n)
    rows = 2500
    s = HipBatchSampler(n, rows)
    check(s, head_like(rng, rows, n), rng.random(rows).astype(np.float32) * np.float32(0.999999),
          t=rng.choice([0.0, 0.7, 1.0, 2.0], size=rows).astype(np.float32),
          k=rng.choice([0, 1, 2, 3, 40], size=rows), p=rng.choice([1.0, 0.9, 0.3], size=rows).astype(np.float32),
          m=rng.choice([0.0, 0.1], size=rows).astype(np.float32))


@pytest.mark.parametrize("n", [2, 20000])
def test_replays_between_eager_calls_with_every_filter(hip, n):
    """A captured call and eager ones of the same sampler, in turn."""
    import torch
    rng = np.random.default_rng(14)
    rows = 8
    s = HipBatchSampler(32768, rows)
    filters = dict(t=rng.choice([0.5, 1.0, 1.5], size=rows).astype(np.float32),
                   k=np.array([0, 0, 1, 5, 40, 300, 3000, 0], np.int32),
                   p=np.array([1, 0.9, 1, 0.9, 0.95, 0.8, 0.9, 0.05], np.float32),
                   m=np.array([0, 0, 0, 0.1, 0, 0.01, 0, 0], np.float32))
    d = {k: torch.from_numpy(v).cuda() for k, v in filters.items()}
    x, u = torch.zeros(rows, n, device="cuda"), torch.zeros(rows, device="cuda")
    a, b = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
    stream = torch.cuda.Stream()

    def call(out, at):
        s.sample_device(x.data_ptr(), rows, out.data_ptr(), u.data_ptr(), temperature_ptr=d["t"].data_ptr(),
                        top_k_ptr=d["k"].data_ptr(), top_p_ptr=d["p"].data_ptr(), min_p_ptr=d["m"].data_ptr(),
                        count=n, stream=at)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        call(a, stream.cuda_stream)
    for _ in range(4):
        logits = head_like(rng, rows, n)
        r = rng.random(rows).astype(np.float32) * np.float32(0.999999)
        x.copy_(torch.from_numpy(logits))
        u.copy_(torch.from_numpy(r))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        call(b, 0)
        torch.cuda.synchronize()
        want = [reference(logits[i], r[i], *(filters[k][i] for k in "tkpm")) for i in range(rows)]
        assert a.tolist() == want and b.tolist() == want


def test_random_numbers_of_more_digits(sampler):
    """Numbers just below 1 are no error on the host, and a top-k beyond 32 bits keeps all."""
    x = head_like(np.random.default_rng(16), 2, 700)
    got = sampler.sample(x, random_value=1 - 2.0 ** -50, top_k=2 ** 33 + 1)
    assert got.tolist() == [reference(r, 1 - 2.0 ** -24) for r in x]


def test_refusals(sampler):
    x = np.zeros((2, 100), np.float32)
    for kw, text in [(dict(random_value=1.0), "RANDOM-VALUE"), (dict(random_value=[0.5, -0.1]), "Row 1: RANDOM-VALUE"),
                     (dict(random_value=0.5, top_k=-1), "TOP-K"), (dict(random_value=0.5, top_p=0), "TOP-P"),
                     (dict(random_value=0.5, min_p=1.1), "MIN-P"), (dict(random_value=0.5, temperature=-1), "TEMPERATURE"),
                     (dict(random_value=0.5, temperature=np.inf), "TEMPERATURE")]:
        with pytest.raises(SamplingError, match=text):
            sampler.sample(x, **kw)
    x[1, 3] = np.nan
    with pytest.raises(SamplingError, match="Row 1: a NaN logit"):
        sampler.sample(x, random_value=0.5)
    with pytest.raises(SamplingError, match="65 rows"):
        sampler.sample(np.zeros((65, 100), np.float32), random_value=0.5)
    with pytest.raises(SamplingError, match="do not fit"):
        sampler.sample(np.zeros((1, 262145), np.float32), random_value=0.5)
    with pytest.raises(SamplingError, match="null argument"):
        sampler.sample_device(0, 1, 0, 0)
    with pytest.raises(SamplingError, match="dimensions"):
        sampler.sample(np.zeros(100, np.float32), random_value=0.5)


@pytest.mark.parametrize("n", [3, 5])
def test_the_most_rows(hip, n):
    rng = np.random.default_rng(17)
    rows = 65535
    s = HipBatchSampler(n, rows)
    x = (rng.normal(size=(rows, n)) * 2).astype(np.float32)
    u = rng.random(rows).astype(np.float32) * np.float32(0.999999)
    got = s.sample(x, random_value=u, top_k=2, top_p=0.9)
    at = rng.integers(0, rows, size=300).tolist() + [0, rows - 1]
    assert [int(got[i]) for i in at] == [reference(x[i], u[i], k=2, p=0.9) for i in at]
    assert got.min() >= 0 and got.max() < n
