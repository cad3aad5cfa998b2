"""What holds for every way that a call takes through the device: calls that plan for themselves, calls of few rows behind a
plan, calls whose rows share keys; and workspaces that different calls use in turn."""
import numpy as np
import pytest

from llambda_amd.hip_backend import HipBackendError
from test_attention_gpu import KINDS, Problem, random_tree

pytestmark = pytest.mark.gpu

WAYS = {
    "alone": ([20, 1, 40, 5], [16, 30, 0, 64]),
    "few": ([1, 2, 3] * 50, [40, 0, 170] * 50),
    "many": ([300, 120, 1, 90, 400], [16, 30, 64, 0, 6000]),  # the last one's tiles lie in several shares
}


def refuse(p, message, skip, session=None):
    """The call leaves the sequences `skip` as they are, does the others, and is reported once."""
    import torch
    torch.cuda.synchronize()
    session = session or p.open()
    p.y.fill_(77)
    torch.cuda.synchronize()
    p.call(session)
    with pytest.raises(HipBackendError, match=message):
        session.sync()
    p.check(skip=skip)
    session.sync()
    return session


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("kinds, head_dim", [(("f32", "f16"), 64), (("bf16", "bf16"), 128), (("f32", "f32"), 256)],
                         ids=["f32-f16", "bf16-bf16", "f32-f32"])
def test_refused_sequences(hip, way, kinds, head_dim):
    lengths, cached = WAYS[way]
    rng = np.random.default_rng(60)
    last = len(lengths) - 1

    def problem():
        return Problem(rng, lengths, cached, heads=8, kv_heads=2, head_dim=head_dim, kinds=kinds)

    for i, entry, page in [(last, 0, -1), (last, 0, 2 ** 31 - 1), (2, 0, -2 ** 31), (0, 1, "pages"), (last, "end", -5)]:
        p = problem()
        entry = (lengths[i] + cached[i] - 1) // p.page if entry == "end" else entry
        p.d_table[i, entry] = p.pages if page == "pages" else page
        session = refuse(p, "a page lies outside", [i])
        # the same session with the page in place
        p.d_table[i, entry] = int(p.table[i, entry])
        p.y.fill_(77)
        p.call(session)
        session.sync()
        p.check()
    for i, context in [(1, -1), (last, 2 ** 31 - 3), (0, -2 ** 31), (last, "one too many")]:
        p = problem()
        p.context[i] = p.width * p.page - lengths[i] + 1 if context == "one too many" else context
        refuse(p, "do not fit the session's context", [i])
    for at, offset in [(2, -1), (1, sum(lengths) + 1), (last, 0), (0, -2 ** 31), (last + 1, 2 ** 31 - 1)]:
        p = problem()
        p.offsets[at] = offset
        refuse(p, "offsets do not ascend", list(range(len(lengths))))
    p = problem()  # two at once, and a call with nothing to refuse
    p.d_table[0, 0] = p.pages
    p.context[last] = -7
    session = refuse(p, "context.*outside the pool", [0, last])
    p.d_table[0, 0] = int(p.table[0, 0])
    p.context[last] = cached[last]
    p.y.fill_(77)
    p.call(session)
    session.sync()
    p.check()


@pytest.mark.parametrize("way", WAYS)
def test_every_sequence_is_refused(hip, way):
    lengths, cached = WAYS[way]
    rng = np.random.default_rng(61)
    p = Problem(rng, lengths, cached, heads=8, kv_heads=2)
    p.d_table[:, 0] = -1
    session = refuse(p, "a page lies outside", list(range(len(lengths))))
    p.d_table[:, 0] = p.d_table.new_tensor(p.table[:, 0])
    p.context.fill_(-1)
    refuse(p, "do not fit the session's context", list(range(len(lengths))), session)
    p.context.copy_(p.context.new_tensor(cached))
    p.call(session)
    session.sync()
    p.check()


@pytest.mark.parametrize("way", WAYS)
def test_refused_trees(hip, way):
    import torch
    rng = np.random.default_rng(62)
    lengths = {"alone": [20, 1, 40, 5], "few": [10] * 40, "many": [61, 256, 1, 90]}[way]
    cached = [int(rng.integers(0, 900)) for _ in lengths]
    more = dict(heads=8, kv_heads=2)
    for i, node, parent in [(0, 3, 3), (0, 0, 0), (len(lengths) - 1, 4, -2), (len(lengths) - 1, 2, 2 ** 31 - 1),
                            (0, 5, -2 ** 31)]:
        p = Problem(rng, lengths, cached, trees=[random_tree(rng, n) for n in lengths], **more)
        p.parents[sum(lengths[:i]) + node] = parent
        refuse(p, "a parent that is no earlier node", [i])
    lengths, cached = ([200, 257, 40], [5, 5, 300]) if way == "many" else ([3, 257] + [9] * 60, [5] * 62)
    p = Problem(rng, lengths, cached, trees=[random_tree(rng, n) for n in lengths], **more)
    refuse(p, "too many nodes", [1])


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("heads, kv_heads, head_dim", [(8, 2, 64), (4, 1, 128), (7, 7, 80), (8, 2, 256)])
def test_trees_of_few_rows_behind_a_plan(hip, kinds, heads, kv_heads, head_dim):
    """Ancestors from the workspace, rows that wavefronts share."""
    rng = np.random.default_rng(63)
    lengths = [10] * 30 + [16, 1, 0, 33, 2]
    cached = [int(v) for v in rng.integers(0, 700, size=len(lengths))]
    p = Problem(rng, lengths, cached, heads=heads, kv_heads=kv_heads, head_dim=head_dim, kinds=kinds,
                trees=[random_tree(rng, n) for n in lengths], spare=3)
    session = p.open()
    p.call(session)
    session.sync()
    p.check()


class Pair:
    """Two problems in the layers of one session's pages."""

    def __init__(self, rng, a, b, **more):
        import torch
        page = more.setdefault("page", 16)
        need = [sum(-(-(n + c) // page) for n, c in zip(*x)) for x in (a, b)]
        self.both = [Problem(rng, *x, layers=2, layer=i, extra_pages=max(need) - need[i] + 2, **more)
                     for i, x in enumerate((a, b))]
        p, q = self.both
        width = max(p.width, q.width)
        for x in self.both:
            table = np.full((len(x.lengths), width), -7, dtype=np.int32)
            table[:, :x.width] = x.table
            x.table, x.d_table, x.width = table, torch.from_numpy(table).cuda(), width
        for name in ("keys", "values"):
            both = getattr(p, name).copy()
            both[1] = getattr(q, name)[1]
            pool = getattr(p, "d_" + name)
            pool.copy_(torch.from_numpy(both).to(pool.dtype))
            setattr(q, "d_" + name, pool)
            setattr(p, name, both)
            setattr(q, name, both.copy())
        self.session = p.open(max_tokens=max(p.tokens, q.tokens), max_sequences=max(len(p.lengths), len(q.lengths)))
        torch.cuda.synchronize()

    def check(self):
        import torch
        torch.cuda.synchronize()
        p, q = self.both
        for name in ("keys", "values"):
            got = getattr(p, "d_" + name).float().cpu().numpy()
            getattr(p, name)[1], getattr(q, name)[0] = got[1], got[0]
        p.check()
        q.check()


PAIRS = {
    "prompts and steps in parts": (([300, 1, 150], [3000, 5, 0]), ([1] * 9, [9000, 4, 0, 500, 64, 31, 2000, 1, 7])),
    "prompts and many steps": (([700, 30, 90], [0, 5, 60]), ([1] * 300, [300] * 100 + [40] * 200)),
    "steps alone and many steps": (([1, 1], [6000, 70]), ([1] * 280, [200] * 280)),
    "two prompts": (([500, 20], [2000, 0]), ([90, 800], [30, 0])),
}


@pytest.mark.parametrize("name", PAIRS)
@pytest.mark.parametrize("kinds", [("f32", "f16"), ("bf16", "bf16")], ids="-".join)
def test_different_calls_on_two_streams(hip, name, kinds):
    """The calls of a session wait for each other, whatever their streams: their workspace is one."""
    import torch
    rng = np.random.default_rng(64)
    pair = Pair(rng, *PAIRS[name], heads=8, kv_heads=2, head_dim=64, kinds=kinds)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(3):
        for x in pair.both:
            x.y.fill_(77)
        torch.cuda.synchronize()
        for k in range(12):
            pair.both[k % 2].call(pair.session, stream=streams[(k + turn) % 3].cuda_stream)
        pair.session.sync(streams[0].cuda_stream)
        pair.check()


@pytest.mark.parametrize("name", PAIRS)
def test_a_call_between_leaves_no_trace(hip, name):
    """The same bits before and after another kind of call of the same session; and from a graph, whose replays the other's
    eager calls lie between."""
    import torch
    rng = np.random.default_rng(65)
    pair = Pair(rng, *PAIRS[name], heads=8, kv_heads=2, head_dim=128)
    p, q = pair.both
    session, stream = pair.session, torch.cuda.Stream()
    first = []
    for x in (p, q):
        x.call(session, stream=stream.cuda_stream)
        session.sync(stream.cuda_stream)
        first.append(x.y.clone())
    pair.check()

    def again(x, call):
        x.y.fill_(77)
        torch.cuda.synchronize()
        call()
        session.sync(stream.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(x.y, first[x.layer])

    for x in (p, q, p):
        again(x, lambda: x.call(session, stream=stream.cuda_stream))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        p.call(session, stream=stream.cuda_stream)

    def replay():
        with torch.cuda.stream(stream):
            graph.replay()

    for _ in range(3):
        again(p, replay)
        again(q, lambda: q.call(session, stream=stream.cuda_stream))
    pair.check()


def test_different_scores_on_two_streams(hip):
    """Calls of one scorer with logits, counts, tops and results of their own."""
    import torch
    from llambda_amd.sampling import HipTokenScorer
    from test_batch_sampling_gpu import head_like
    rng = np.random.default_rng(66)
    scorer = HipTokenScorer(40000, 60, 20)
    calls = []
    for rows, vocab, top in [(60, 40000, 1), (3, 5001, 20), (40, 30000, 7)]:
        x = head_like(rng, rows, vocab)
        given = rng.integers(0, vocab, size=(rows, 2)).astype(np.int32)
        want = scorer.score(x, given, top)
        empty = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
        out = [empty(rows, 2), empty(rows), empty(rows, top, t=torch.int32), empty(rows, top)]
        calls.append((torch.from_numpy(x).cuda(), torch.from_numpy(given).cuda(), out, want, top))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(4):
        for *_, out, _, _ in calls:
            for t in out:
                t.fill_(-5)
        torch.cuda.synchronize()
        for k in range(18):
            x, given, out, _, top = calls[k % 3]
            scorer.score_device(x.data_ptr(), len(x), given_ptr=given.data_ptr(), given=2, top=top, count=x.shape[1],
                                log_probs_ptr=out[0].data_ptr(), entropy_ptr=out[1].data_ptr(),
                                top_tokens_ptr=out[2].data_ptr(), top_log_probs_ptr=out[3].data_ptr(),
                                stream=streams[(k + turn) % 2].cuda_stream)
        torch.cuda.synchronize()
        for _, _, out, want, _ in calls:
            for t, w in zip(out, (want.log_probs, want.entropy, want.top_tokens, want.top_log_probs)):
                assert np.array_equal(t.cpu().numpy(), w)
