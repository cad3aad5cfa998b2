"""Attention over a paged cache on the device against attention in 64 bits, and what it must leave alone."""
import numpy as np
import pytest

import attention_reference as ref
from llambda_amd.attention import AttentionLayout, HipAttentionSession
from llambda_amd.hip_backend import HipBackendError

pytestmark = pytest.mark.gpu

KINDS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


def torch_type(kind):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]


class Problem:
    """Sequences with cached tokens and new rows: host arrays in float32 (exactly what the types hold), a pool of
    pages in no order, and the same on the device."""

    def __init__(self, rng, lengths, cached, *, heads=8, kv_heads=2, head_dim=64, kinds=("f32", "f16"), page=16,
                 packed=False, spare=0, fill=None, trees=None, layers=1, layer=0, q_scale=2.0, extra_pages=3):
        import torch
        self.lengths, self.cached, self.kinds, self.trees = list(lengths), list(cached), kinds, trees
        self.heads, self.kv, self.dim, self.page, self.layer = heads, kv_heads, head_dim, page, layer
        n, tokens = len(lengths), sum(lengths) + spare
        self.tokens = tokens
        row, cell = kinds

        def make(*shape):
            return ref.rounded(rng.normal(size=shape).astype(np.float32), row)

        self.q = make(tokens, heads, head_dim) * np.float32(q_scale)
        self.k, self.v = make(tokens, kv_heads, head_dim), make(tokens, kv_heads, head_dim)
        need = [-(-(a + b) // page) for a, b in zip(lengths, cached)]
        width = max(max(need), 1) + 1
        pages = sum(need) + extra_pages
        order = rng.permutation(pages)
        self.table = np.full((n, width), -7, dtype=np.int32)  # entries behind a sequence's pages are not read
        at = 0
        for i in range(n):
            self.table[i, :need[i]] = order[at:at + need[i]]
            at += need[i]
        shape = (layers, pages, kv_heads, page, head_dim)
        self.keys = ref.rounded(rng.normal(size=shape).astype(np.float32), cell)
        self.values = ref.rounded(rng.normal(size=shape).astype(np.float32), cell)
        if fill is not None:  # everything but the cached tokens
            for pool in (self.keys, self.values):
                keep = np.full(shape, np.float32(fill), dtype=np.float32)
                for i in range(n):
                    for j in range(cached[i]):
                        w = (layer, self.table[i, j // page], slice(None), j % page)
                        keep[w] = pool[w]
                pool[...] = keep
        self.session = HipAttentionSession
        rt, ct = torch_type(row), torch_type(cell)
        self.d_keys = torch.from_numpy(self.keys).to(ct).cuda()
        self.d_values = torch.from_numpy(self.values).to(ct).cuda()
        if packed:
            self.rows = torch.empty((tokens, (2 * heads + 2 * kv_heads) * head_dim), dtype=rt, device="cuda")
            cuts = np.cumsum([0, heads, kv_heads, kv_heads, heads]) * head_dim
            self.d = [self.rows[:, a:b] for a, b in zip(cuts[:-1], cuts[1:])]
        else:
            self.d = [torch.empty((tokens, h * head_dim), dtype=rt, device="cuda") for h in (heads, kv_heads, kv_heads, heads)]
        for t, a in zip(self.d, (self.q, self.k, self.v)):
            t.copy_(torch.from_numpy(a.reshape(tokens, -1)).to(rt))
        self.y = self.d[3]
        self.y.fill_(77)
        self.offsets = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")
        self.context = torch.tensor(cached, dtype=torch.int32, device="cuda")
        self.d_table = torch.from_numpy(self.table).cuda()
        self.parents = None
        if trees is not None:
            self.parents = torch.tensor(np.concatenate([np.asarray(t, dtype=np.int32) for t in trees]
                                                       + [np.zeros(spare, np.int32)]), dtype=torch.int32, device="cuda")
        self.layers, self.pages, self.width, self.scale = layers, pages, width, 1 / np.sqrt(head_dim)
        torch.cuda.synchronize()

    def open(self, **more):
        layout = AttentionLayout(self.heads, self.kv, self.dim, row_type=self.kinds[0], cache_type=self.kinds[1])
        options = dict(pages=self.pages, page_tokens=self.page, max_context=self.width * self.page,
                       max_tokens=max(self.tokens, 1), max_sequences=len(self.lengths), layers=self.layers,
                       key_pages_ptr=self.d_keys.data_ptr(), value_pages_ptr=self.d_values.data_ptr())
        return HipAttentionSession(layout, **{**options, **more})

    def call(self, session, step=False, stream=0):
        q, k, v, y = self.d
        session.run_device(q.data_ptr(), k.data_ptr(), v.data_ptr(), y.data_ptr(), self.tokens, self.context.data_ptr(),
                           self.d_table.data_ptr(), len(self.lengths), offsets_ptr=0 if step else self.offsets.data_ptr(),
                           parents_ptr=0 if self.parents is None else self.parents.data_ptr(), layer=self.layer,
                           q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0), output_stride=y.stride(0),
                           stream=stream)

    def places(self, i):
        at = np.arange(self.cached[i] + self.lengths[i])
        return self.table[i, at // self.page], at % self.page

    def check(self, skip=(), finite=True):
        import torch
        torch.cuda.synchronize()
        row, cell = self.kinds
        keys, values = self.keys.copy(), self.values.copy()
        y = self.y.float().cpu().numpy().reshape(self.tokens, self.heads, self.dim)
        begin, worst = 0, 0.0
        for i, (n, c) in enumerate(zip(self.lengths, self.cached)):
            mine = slice(begin, begin + n)
            begin += n
            if i in skip:
                assert np.all(y[mine] == 77), f"rows of refused sequence {i} changed"
                continue
            if not n:
                continue
            page, at = self.places(i)
            for pool, new in ((keys, self.k), (values, self.v)):
                pool[self.layer, page[c:], :, at[c:]] = ref.rounded(new[mine], cell)
            visible = ref.sees(n, c, None if self.trees is None else self.trees[i])
            k, v = (pool[self.layer, page, :, at] for pool in (keys, values))
            want, bound = ref.attention(self.q[mine], k, v, visible, np.float32(self.scale), row, cell)
            if finite:
                assert np.all(np.isfinite(want))
            off = np.abs(y[mine] - want)
            ok = (off <= bound) | (~np.isfinite(want) & ~np.isfinite(y[mine]))
            worst = max(worst, float((off / bound)[np.isfinite(want)].max(initial=0)))
            assert np.all(ok), (f"sequence {i} ({n} rows behind {c}): {np.count_nonzero(~ok)} outputs off, first "
                                f"{np.argwhere(~ok)[0]}, by {off[~ok][0]:.3e}, allowed {bound[~ok][0]:.3e}")
        assert np.all(y[begin:] == 77), "rows of no sequence changed"
        for name, got, want in (("keys", self.d_keys, keys), ("values", self.d_values, values)):
            got = got.float().cpu().numpy()
            assert np.array_equal(got, want, equal_nan=True), f"{name} differ"
        print(f"worst {worst:.3f} of the bound", flush=True)


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("heads, kv_heads, head_dim, page", [
    (8, 2, 64, 16), (4, 4, 128, 32), (14, 2, 128, 64), (3, 1, 256, 16), (8, 1, 16, 128), (6, 2, 80, 16), (4, 1, 208, 64)])
def test_prompts(hip, kinds, heads, kv_heads, head_dim, page):
    """Packed sequences: one row, odd lengths, none, cached tokens that end inside pages and tiles; rows behind."""
    rng = np.random.default_rng(1)
    p = Problem(rng, [33, 1, 0, 150, 64, 17], [0, 70, 5, 31, 64, 1], heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, page=page, kinds=kinds, spare=3)
    session = p.open()
    p.call(session)
    session.sync()
    p.check()


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("heads, kv_heads, head_dim", [(8, 2, 128), (7, 1, 64), (2, 2, 256), (40, 1, 32), (24, 3, 96)])
def test_steps(hip, kinds, heads, kv_heads, head_dim):
    rng = np.random.default_rng(2)
    cached = [0, 1, 15, 16, 31, 63, 64, 65, 127, 300, 1000, 2111]
    p = Problem(rng, [1] * len(cached), cached, heads=heads, kv_heads=kv_heads, head_dim=head_dim, kinds=kinds)
    session = p.open()
    p.call(session, step=True)
    session.sync()
    p.check()


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
def test_long_contexts_in_parts(hip, kinds):
    """Positions shared out over the device: steps behind 20000 tokens, more pages than a workgroup lists at a
    time, and a prompt behind 9000."""
    rng = np.random.default_rng(3)
    p = Problem(rng, [1, 1], [20000, 77], heads=4, kv_heads=2, head_dim=64, kinds=kinds)
    session = p.open()
    p.call(session, step=True)
    session.sync()
    p.check()
    p = Problem(rng, [70, 3], [9000, 4], heads=4, kv_heads=1, head_dim=128, kinds=kinds, page=32)
    session = p.open()
    p.call(session)
    session.sync()
    p.check()


def random_tree(rng, n):
    return [int(rng.integers(max(-1, j - 4), j)) if rng.random() < 0.7 else int(rng.integers(-1, j)) if j else -1
            for j in range(n)]


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("heads, kv_heads, head_dim", [(4, 2, 64), (8, 1, 128), (16, 2, 256)])
def test_trees(hip, kinds, heads, kv_heads, head_dim):
    """A chain, a star, random trees, one node, the most nodes; no cached tokens, and ends inside tiles."""
    rng = np.random.default_rng(4)
    trees = [[-1, 0, 1, 2, 3], [-1] * 40, random_tree(rng, 61), [-1], random_tree(rng, 256), [], random_tree(rng, 33)]
    p = Problem(rng, [len(t) for t in trees], [0, 45, 1000, 64, 31, 9, 1], heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, kinds=kinds, trees=trees, spare=2)
    session = p.open()
    p.call(session)
    session.sync()
    p.check()


@pytest.mark.parametrize("heads, kv_heads", [(4, 2), (2, 2)])
def test_small_trees_take_the_kernel_of_steps(hip, heads, kv_heads):
    rng = np.random.default_rng(5)
    trees = [random_tree(rng, n) for n in (7, 1, 13, 5)]
    p = Problem(rng, [len(t) for t in trees], [200, 0, 31, 640], heads=heads, kv_heads=kv_heads, trees=trees, head_dim=128)
    session = p.open()
    p.call(session)
    session.sync()
    p.check()


def test_columns_of_one_buffer(hip):
    rng = np.random.default_rng(6)
    for kinds in (("f32", "f16"), ("bf16", "bf16")):
        p = Problem(rng, [40, 9], [3, 0], kinds=kinds, packed=True, head_dim=80)
        session = p.open()
        p.call(session)
        session.sync()
        p.check()


def test_layers_have_pages_of_their_own(hip):
    rng = np.random.default_rng(7)
    p = Problem(rng, [40, 9], [3, 20], layers=3, layer=1)
    session = p.open()
    p.call(session)
    session.sync()
    p.check()


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("step", [False, True])
def test_pages_hold_no_numbers_behind_the_tokens(hip, kinds, fill, step):
    rng = np.random.default_rng(8)
    lengths = [1, 1, 1] if step else [40, 1, 70]
    p = Problem(rng, lengths, [3, 64, 130], kinds=kinds, fill=fill, head_dim=64, page=64)
    session = p.open()
    p.call(session, step=step)
    session.sync()
    p.check()


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("rows", [9, 150])
def test_tokens_that_are_no_numbers_reach_only_rows_that_see_them(hip, kinds, bad, rows):
    """A later token's key and value, and a tree node's, are infinite or NaN in some elements."""
    rng = np.random.default_rng(9)
    trees = [random_tree(rng, rows)]
    for tree in (None, trees):
        p = Problem(rng, [rows], [21], kinds=kinds, head_dim=64, heads=4, kv_heads=2, trees=tree)
        p.v[5, 0, 3] = bad
        p.v[5, 1, 40] = -bad
        p.k[7, 1, 10] = bad
        import torch
        for t, a in zip(p.d[1:3], (p.k, p.v)):
            t.copy_(torch.from_numpy(a.reshape(p.tokens, -1)).to(t.dtype))
        torch.cuda.synchronize()
        session = p.open()
        p.call(session)
        session.sync()
        torch.cuda.synchronize()
        y = p.y.float().cpu().numpy().reshape(rows, 4, 64)
        seen = ref.sees(rows, 21, None if tree is None else tree[0])[:, 21:]
        # heads 0, 1 read kv head 0; a value spoils its element, a key the whole row of its heads
        spoiled = np.zeros(y.shape, dtype=bool)
        spoiled[:, :2, 3] |= seen[:, 5, None]
        spoiled[:, 2:, 40] |= seen[:, 5, None]
        whole = seen[:, 7]
        assert np.all(np.isfinite(y[:, :2][~spoiled[:, :2]]))
        assert np.all(~np.isfinite(y[:, :2][spoiled[:, :2]]))
        assert np.all(np.isfinite(y[~whole][:, 2:][~spoiled[~whole][:, 2:]]))
        # the finite ones are right: the same problem without the bad token's elements
        p.v[5, 0, 3] = p.v[5, 1, 40] = 0
        p.k[7, 1, 10] = 0
        page, at = p.places(0)
        for pool, new in ((p.keys, p.k), (p.values, p.v)):
            pool[0, page[21:], :, at[21:]] = ref.rounded(new, kinds[1])
        want, bound = ref.attention(p.q, *(pool[0, page, :, at] for pool in (p.keys, p.values)),
                                    ref.sees(rows, 21, None if tree is None else tree[0]), np.float32(p.scale), *kinds)
        good = ~spoiled
        good[whole, 2:] = False
        assert np.all(np.abs(y - want)[good] <= bound[good])


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("q_scale", [1e-30, 1e-3, 60.0, 1e4])
def test_magnitudes(hip, kinds, q_scale):
    """Scores from nothing to one key taking all; f16 rows end at 65504."""
    rng = np.random.default_rng(10)
    if kinds[0] == "f16":
        q_scale = min(max(q_scale, 1e-3), 1e4)
    p = Problem(rng, [50, 1, 40], [100, 200, 0], kinds=kinds, q_scale=1.0, head_dim=128, heads=4, kv_heads=1)
    p.q = ref.rounded(p.q * np.float32(q_scale), kinds[0])
    import torch
    p.d[0].copy_(torch.from_numpy(p.q.reshape(p.tokens, -1)).to(p.d[0].dtype))
    torch.cuda.synchronize()
    session = p.open()
    p.call(session)
    session.sync()
    p.check()


def test_rows_of_very_different_elements(hip):
    """Queries whose elements span the range, keys and values at f16's ends, equal scores of many keys."""
    rng = np.random.default_rng(11)
    p = Problem(rng, [30, 200], [70, 0], kinds=("f32", "f16"), head_dim=64, heads=4, kv_heads=2)
    p.q *= np.exp(rng.uniform(-12, 0, size=p.q.shape)).astype(np.float32)
    p.q[5] = 0
    p.k *= np.float32(2.0 ** -3)
    p.v *= np.exp(rng.uniform(-8, 9, size=p.v.shape)).astype(np.float32)
    import torch
    for t, a in zip(p.d, (p.q, p.k, p.v)):
        t.copy_(torch.from_numpy(a.reshape(p.tokens, -1)))
    torch.cuda.synchronize()
    session = p.open()
    p.call(session)
    session.sync()
    p.check()


def test_refused_sequences_are_left_as_they_are(hip):
    import torch
    rng = np.random.default_rng(12)

    def problem(**more):
        return Problem(rng, [20, 1, 40, 5], [16, 30, 0, 64], **more)

    def broken(p, message, skip):
        session = p.open()
        p.call(session)
        with pytest.raises(HipBackendError, match=message):
            session.sync()
        for i in skip:
            if p.cached[i] < 0 or p.cached[i] > 1000:
                p.cached[i] = 0
        p.check(skip=skip)
        session.sync()  # reported once

    p = problem()
    p.d_table[2, 1] = p.pages
    broken(p, "a page lies outside", [2])
    p = problem()
    p.d_table[0, 0] = -1  # a page of cached tokens
    broken(p, "a page lies outside", [0])
    p = problem()
    p.context[1] = -1
    broken(p, "do not fit the session's context", [1])
    p = problem()
    p.context[3] = 2 ** 31 - 3
    broken(p, "do not fit the session's context", [3])
    p = problem()
    p.offsets[2] = 5  # descends
    torch.cuda.synchronize()
    broken(p, "offsets do not ascend", [0, 1, 2, 3])
    p = problem()
    p.offsets[4] = 10 ** 6
    broken(p, "offsets do not ascend", [0, 1, 2, 3])
    trees = [random_tree(rng, n) for n in (20, 1, 40, 5)]
    trees[2][7] = 7
    p = problem(trees=[t if i != 2 else [-1] * 40 for i, t in enumerate(trees)])
    p.parents[28] = 7
    broken(p, "a parent that is no earlier node", [2])
    trees = [random_tree(rng, 3), [-1] * 257]
    p = Problem(rng, [3, 257], [5, 5], trees=trees)
    broken(p, "too many nodes", [1])


def test_calls_that_are_refused(hip):
    rng = np.random.default_rng(13)
    p = Problem(rng, [20, 4], [16, 3])
    session = p.open()
    q, k, v, y = (t.data_ptr() for t in p.d)
    c, t, o = p.context.data_ptr(), p.d_table.data_ptr(), p.offsets.data_ptr()

    def refused(message, *args, **more):
        with pytest.raises(HipBackendError, match=message):
            session.run_device(*args, **more)

    refused("null q", 0, k, v, y, 24, c, t, 2, offsets_ptr=o)
    refused("null output", q, k, v, 0, 24, c, t, 2, offsets_ptr=o)
    refused("null context or table", q, k, v, y, 24, 0, t, 2, offsets_ptr=o)
    refused("0 tokens are not in", q, k, v, y, 0, c, t, 2, offsets_ptr=o)
    refused("25 tokens are not in", q, k, v, y, 25, c, t, 2, offsets_ptr=o)
    refused("3 sequences are not in", q, k, v, y, 24, c, t, 3, offsets_ptr=o)
    refused("24 tokens of 2 sequences without offsets", q, k, v, y, 24, c, t, 2)
    refused("layer 1 is not in", q, k, v, y, 24, c, t, 2, offsets_ptr=o, layer=1)
    refused("stride 100 of q", q, k, v, y, 24, c, t, 2, offsets_ptr=o, q_stride=100)
    refused("rows of k must be 16-byte aligned", q, k, v, y, 24, c, t, 2, offsets_ptr=o, k_stride=130)
    refused("rows of v must be 16-byte aligned", q, k, v + 4, y, 24, c, t, 2, offsets_ptr=o)
    refused("q and output overlap", q, k, v, q, 24, c, t, 2, offsets_ptr=o)
    refused("v and output overlap", q, k, y + 16, y, 24, c, t, 2, offsets_ptr=o)
    refused("table rows of 1 entries", q, k, v, y, 24, c, t, 2, offsets_ptr=o, table_stride=1)
    refused("lists must be 4-byte aligned", q, k, v, y, 24, c + 2, t, 2, offsets_ptr=o)
    for args, message in [((c, t, 0, c, 2, 4), "null argument"), ((c, t, c, c, 0, 4), "0 sequences"),
                          ((c, t, c, c, 2, 0), "paths of 0 entries"), ((c, t, c + 1, c, 2, 4), "4-byte aligned")]:
        with pytest.raises(HipBackendError, match=message):
            session.accept_device(*args)
    table = p.table[0]
    with pytest.raises(HipBackendError, match="is not in 0.."):
        session.read([0, 99], 0, 32)
    with pytest.raises(HipBackendError, match="does not hold 33 tokens"):
        session.read([0, 1], 0, 33)
    with pytest.raises(HipBackendError, match="rows of q, k and v"):
        session.run(p.q[:3], p.k[:2], p.v[:3], table)
    with pytest.raises(HipBackendError, match="no earlier node"):
        session.run(p.q[:2], p.k[:2], p.v[:2], table, parents=[0, -1])
    session.sync()
    p.check(skip=[0, 1])
    session.close()
    with pytest.raises(HipBackendError, match="closed"):
        session.sync()


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
def test_host_rows(hip, kinds):
    """Rows, pages and trees from host memory: a prompt, further tokens one by one, then a tree."""
    rng = np.random.default_rng(14)
    row, cell = kinds
    layout = AttentionLayout(4, 2, 48, row_type=row, cache_type=cell, scale=0.2)
    session = HipAttentionSession(layout, pages=12, page_tokens=16, max_context=100, max_tokens=60, layers=2)
    table = [3, 9, 0, 5, 11, 1, 7]
    kept = rng.normal(size=(2, 20, 2, 48)).astype(np.float32)
    session.write(table, 0, *(ref.stored(a, cell) for a in kept), layer=1)
    k, v = (ref.rounded(a, cell) for a in kept)
    for n, tree in [(40, None), (1, None), (1, None), (9, random_tree(rng, 9))]:
        q, nk, nv = (ref.rounded(rng.normal(size=(n, h, 48)).astype(np.float32), row) for h in (4, 2, 2))
        y = ref.loaded(session.run(*(ref.stored(a, row) for a in (q, nk, nv)), table, len(k), parents=tree, layer=1), row)
        k, v = np.concatenate([k, ref.rounded(nk, cell)]), np.concatenate([v, ref.rounded(nv, cell)])
        want, bound = ref.attention(q, k, v, ref.sees(n, len(k) - n, tree), np.float32(0.2), row, cell)
        assert np.all(np.abs(y - want) <= bound)
    got = session.read(table, 0, len(k), layer=1)
    for a, b in zip(got, (k, v)):
        assert np.array_equal(ref.loaded(a, cell), b)
    for a in session.read(table, 0, 100, layer=0):
        assert not np.any(a)


@pytest.mark.parametrize("kinds", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")], ids="-".join)
def test_accepted_paths(hip, kinds):
    import torch
    rng = np.random.default_rng(15)
    trees = [random_tree(rng, 61) for _ in range(4)] + [random_tree(rng, 5)]
    paths = np.zeros((5, 64), dtype=np.int32)
    counts = []
    for i, (node, tree) in enumerate(zip((60, 31, -1, 0, 4), trees)):
        path = []
        while node >= 0:
            path.append(node)
            node = tree[node]
        counts.append(len(path))
        paths[i, :len(path)] = path[::-1]
    counts[3], paths[3, :3] = 3, [5, 5, 6]  # does not ascend: left as it is
    p = Problem(rng, [len(t) for t in trees], [0, 45, 100, 64, 31], kinds=kinds, trees=trees, layers=2, layer=1)
    session = p.open()
    p.call(session)
    session.sync()
    p.check()
    keys, values = p.d_keys.clone(), p.d_values.clone()
    d_paths, d_counts = torch.from_numpy(paths).cuda(), torch.tensor(counts, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    session.accept_device(p.context.data_ptr(), p.d_table.data_ptr(), d_paths.data_ptr(), d_counts.data_ptr(), 5, 64)
    with pytest.raises(HipBackendError, match="an accepted path does not ascend"):
        session.sync()
    for before, after in ((keys, p.d_keys), (values, p.d_values)):
        want = before.clone()
        for i in (0, 1, 2, 4):
            for j in range(counts[i]):
                a, b = p.cached[i] + int(paths[i, j]), p.cached[i] + j
                want[:, p.table[i, b // 16], :, b % 16] = before[:, p.table[i, a // 16], :, a % 16]
        assert torch.equal(after, want)
    # places and pages out of range, too many nodes
    for change, message in [(dict(context=p.width * 16 - 1), "do not fit"), (dict(page=-1), "a page lies outside"),
                            (dict(count=65), "does not ascend"), (dict(path=256), "does not ascend")]:
        context, table, count, path = p.context.clone(), p.d_table.clone(), d_counts.clone(), d_paths.clone()
        count[3] = 0
        context[0] = change.get("context", 0)
        table[0, 0] = change.get("page", int(p.table[0, 0]))
        count[0] = change.get("count", 1)
        path[0, 0] = change.get("path", 3)
        count[1:] = 0
        before = p.d_keys.clone()
        torch.cuda.synchronize()
        session.accept_device(context.data_ptr(), table.data_ptr(), path.data_ptr(), count.data_ptr(), 5, 64)
        with pytest.raises(HipBackendError, match=message):
            session.sync()
        assert torch.equal(before, p.d_keys)


def test_captured_calls_replay(hip):
    """A step and a tree with its accepted path in one graph, replayed with new inputs beside eager work."""
    import torch
    rng = np.random.default_rng(16)
    steps = Problem(rng, [1] * 5, [40, 700, 0, 64, 3000], heads=8, kv_heads=2, head_dim=128)
    trees = [random_tree(rng, 20) for _ in range(3)]
    tree = Problem(rng, [20] * 3, [500, 0, 90], heads=4, kv_heads=2, trees=trees)
    a, b = steps.open(), tree.open()
    paths = torch.tensor([[0], [0], [0]], dtype=torch.int32, device="cuda")
    counts = torch.zeros(3, dtype=torch.int32, device="cuda")  # nothing moves: the check stays simple
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()

    def work():
        steps.call(a, step=True, stream=stream.cuda_stream)
        tree.call(b, stream=stream.cuda_stream)
        b.accept_device(tree.context.data_ptr(), tree.d_table.data_ptr(), paths.data_ptr(), counts.data_ptr(), 3, 1,
                        stream=stream.cuda_stream)

    work()
    a.sync(stream.cuda_stream)
    b.sync(stream.cuda_stream)
    steps.check()
    tree.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        work()
    for replay in range(3):
        for p in (steps, tree):
            p.q = rng.normal(size=p.q.shape).astype(np.float32)
            p.k = rng.normal(size=p.k.shape).astype(np.float32)
            for t, x in zip(p.d, (p.q, p.k)):
                t.copy_(torch.from_numpy(x.reshape(p.tokens, -1)))
            p.y.fill_(77)
            p.keys[...] = p.d_keys.float().cpu().numpy()
            p.values[...] = p.d_values.float().cpu().numpy()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        a.sync()
        b.sync()
        steps.check()
        tree.check()
        steps.y.fill_(77)
        steps.call(a, step=True)  # an eager call between replays
        a.sync()
        steps.check()


def test_calls_on_two_streams_share_the_workspace(hip):
    import torch
    rng = np.random.default_rng(17)
    p = Problem(rng, [1] * 6, [900, 10, 2500, 64, 0, 333], heads=8, kv_heads=2)
    session = p.open(max_tokens=200)
    others = [Problem(rng, [30, 100, 7], [50, 0, 3], heads=8, kv_heads=2) for _ in range(2)]
    # the others' pages lie in the same session's pools only by their own sessions
    sessions = [o.open() for o in others]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s in streams:
            p.call(session, step=True, stream=s.cuda_stream)
        for o, x, s in zip(others, sessions, streams):
            o.call(x, stream=s.cuda_stream)
    torch.cuda.synchronize()
    session.sync()
    for x in sessions:
        x.sync()
    for q in (p, *others):
        q.check()


def test_rows_do_not_depend_on_what_ran_before(hip):
    """The same call twice, with another in between that leaves other things in the workspace: the same bits."""
    import torch
    rng = np.random.default_rng(18)
    p = Problem(rng, [1] * 4, [5000, 10, 2500, 64], heads=8, kv_heads=2, head_dim=128)
    session = p.open(max_tokens=600)
    p.call(session, step=True)
    session.sync()
    first = p.y.clone()
    q = Problem(rng, [150, 1, 200, 9], [0, 10, 60, 64], heads=8, kv_heads=2, head_dim=128)
    other = HipAttentionSession(AttentionLayout(8, 2, 128), pages=q.pages, page_tokens=16, max_context=q.width * 16,
                                max_tokens=600, max_sequences=4, key_pages_ptr=q.d_keys.data_ptr(),
                                value_pages_ptr=q.d_values.data_ptr())
    q.call(other)
    other.sync()
    q.check()
    p.y.fill_(77)
    p.call(session, step=True)
    session.sync()
    assert torch.equal(p.y, first)
    p.check()


def test_pages_beyond_32_bits(hip):
    """A pool of 5 GB whose last pages are used."""
    import torch
    rng = np.random.default_rng(19)
    pages, page, kv, dim = 20000, 128, 8, 128
    keys, values = (torch.zeros((pages, kv, page, dim), dtype=torch.float16, device="cuda") for _ in range(2))
    table = np.array([[pages - 1, 3, pages - 2]], dtype=np.int32)
    cached = rng.normal(size=(2, 300, kv, dim)).astype(np.float16)
    for pool, a in zip((keys, values), cached):
        for j in range(300):
            pool[int(table[0, j // page]), :, j % page] = torch.from_numpy(a[j]).cuda()
    session = HipAttentionSession(AttentionLayout(16, kv, dim), pages=pages, page_tokens=page, max_context=3 * page,
                                  max_tokens=40, key_pages_ptr=keys.data_ptr(), value_pages_ptr=values.data_ptr())
    q, k, v = (rng.normal(size=(40, h, dim)).astype(np.float32) for h in (16, kv, kv))
    torch.cuda.synchronize()
    y = session.run(q, k, v, table[0], 300)
    k, v = (np.concatenate([a.astype(np.float32), ref.rounded(b, "f16")]) for a, b in zip(cached, (k, v)))
    want, bound = ref.attention(q, k, v, ref.sees(40, 300), np.float32(1 / np.sqrt(dim)), "f32", "f16")
    assert np.all(np.abs(y - want) <= bound)
    got = session.read(table[0], 0, 340)
    assert np.array_equal(got[0].astype(np.float32), k) and np.array_equal(got[1].astype(np.float32), v)


def test_many_sequences(hip):
    """More sequences than a plan's workgroup has threads, some empty."""
    rng = np.random.default_rng(20)
    lengths = rng.integers(0, 4, size=700).tolist()
    cached = rng.integers(0, 50, size=700).tolist()
    p = Problem(rng, lengths, cached, heads=2, kv_heads=1, head_dim=32)
    session = p.open()
    p.call(session)
    session.sync()
    p.check()
    p = Problem(rng, [1] * 700, cached, heads=2, kv_heads=1, head_dim=32)
    session = p.open()
    p.call(session, step=True)
    session.sync()
    p.check()


def test_pages_shared_by_sequences(hip):
    """A prefix that several sequences read."""
    rng = np.random.default_rng(21)
    p = Problem(rng, [1, 1, 1], [40, 40, 35], heads=4, kv_heads=2)
    p.table[1, :2] = p.table[0, :2]
    p.table[2, :2] = p.table[0, :2]
    p.d_table[:, :2] = p.d_table[0, :2]
    session = p.open()
    p.call(session, step=True)
    session.sync()
    p.check()


@pytest.mark.parametrize("kinds", [("f32", "f16"), ("f32", "f32"), ("bf16", "bf16")], ids="-".join)
def test_many_tiles_to_a_share(hip, kinds):
    """Shares of many tiles, whose ends lie near those of tiles, in tiles shorter than that is near, and behind them."""
    rng = np.random.default_rng(22)
    few = dict(heads=8, kv_heads=8, head_dim=16, kinds=kinds)
    for lengths, cached, more in [
            ([1] * 256, [300] * 256, few),
            ([1] * 256, rng.integers(0, 900, size=256).tolist(), few),
            ([1] * 200, rng.integers(0, 60, size=200).tolist(), dict(few, heads=64, kv_heads=64)),
            (rng.integers(0, 3, size=120).tolist(), rng.integers(0, 700, size=120).tolist(),
             dict(few, heads=80, kv_heads=2)),
            # too many for a workgroup's own plan, one of them long
            ([1] * 400, [30000] + [9] * 300 + [600] * 99, dict(few, heads=16, kv_heads=16))]:
        p = Problem(rng, lengths, cached, **more)
        session = p.open()
        p.call(session, step=max(lengths) == 1)
        session.sync()
        p.check()
        p.y.fill_(77)
        p.call(session)  # with offsets, the same
        session.sync()
        p.check()


@pytest.mark.parametrize("kinds", [("f32", "f16"), ("f32", "f32"), ("bf16", "bf16")], ids="-".join)
@pytest.mark.parametrize("lengths, cached, heads, kv_heads", [
    ([300] + [200] * 11 + [90, 257, 1, 512], [6000] + [0] * 15, 32, 32),  # a long one: in shares
    ([200] * 12 + [130, 257, 0, 512, 700], [0] * 17, 64, 64),              # each tile a share
    ([64] * 40 + [2, 0, 130], [0] * 20 + [33] * 23, 128, 32),
    ([170] * 3 + [1200], [0, 90, 1000, 64], 4, 1)])
def test_prompts_of_many_heads(hip, kinds, lengths, cached, heads, kv_heads):
    rng = np.random.default_rng(23)
    p = Problem(rng, lengths, cached, heads=heads, kv_heads=kv_heads, head_dim=16, kinds=kinds)
    session = p.open()
    p.call(session)
    session.sync()
    p.check()


@pytest.mark.parametrize("heads, kv_heads", [(1024, 1), (300, 300), (1024, 1024), (1, 1)])
def test_ends_of_the_ranges(hip, heads, kv_heads):
    """One head and the most; sequences that fill the context; a context that ends inside a page."""
    rng = np.random.default_rng(24)
    for lengths, cached, step in [([1, 1, 1], [0, 85, 36], True), ([3, 0, 1], [83, 0, 85], False)]:
        p = Problem(rng, lengths, cached, heads=heads, kv_heads=kv_heads, head_dim=16)
        p.table = p.table[:, :6].copy()
        p.d_table = p.d_table[:, :6].contiguous()
        p.width = 6
        import torch
        torch.cuda.synchronize()
        session = p.open(max_context=86, max_tokens=p.tokens)
        p.call(session, step=step)
        session.sync()
        p.check()


def test_two_threads_and_one_session(hip):
    """Host calls of several threads on sequences of their own, and scores beside them."""
    from concurrent.futures import ThreadPoolExecutor
    from llambda_amd.sampling import HipTokenScorer
    layout = AttentionLayout(4, 2, 32)
    session = HipAttentionSession(layout, pages=40, page_tokens=16, max_context=150, max_tokens=60)
    scorer = HipTokenScorer(3001, 4, 4)

    def one(i):
        rng = np.random.default_rng(100 + i)
        table = list(range(10 * i, 10 * i + 10))
        k, v = (np.empty((0, 2, 32), np.float32) for _ in range(2))
        for n in (40, 1, 60, 1, 1):
            q, nk, nv = (rng.normal(size=(n, h, 32)).astype(np.float32) for h in (4, 2, 2))
            y = session.run(q, nk, nv, table, len(k))
            k, v = np.concatenate([k, ref.rounded(nk, "f16")]), np.concatenate([v, ref.rounded(nv, "f16")])
            want, bound = ref.attention(q, k, v, ref.sees(n, len(k) - n), np.float32(1 / np.sqrt(32)), "f32", "f16")
            assert np.all(np.abs(y - want) <= bound)
            x = rng.normal(size=(2, 3001)).astype(np.float32)
            top = scorer.score(x, top=1).top_tokens[:, 0]
            assert np.array_equal(top, x.argmax(1))
        return True

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(one, range(4)))


def test_calls_of_too_many_launches_are_refused(hip):
    import torch
    n, kv = 65535, 256
    row = torch.zeros(n * kv * 16, dtype=torch.float32, device="cuda")
    lists = torch.zeros(n, dtype=torch.int32, device="cuda")
    session = HipAttentionSession(AttentionLayout(kv, kv, 16), pages=1, page_tokens=16, max_context=16, max_tokens=n,
                                  max_sequences=n)
    y = torch.full_like(row, 77)
    torch.cuda.synchronize()
    with pytest.raises(HipBackendError, match="65535 tokens of 65535 sequences are too many for one call"):
        session.run_device(row.data_ptr(), row.data_ptr(), row.data_ptr(), y.data_ptr(), n, lists.data_ptr(),
                           lists.data_ptr(), n)
    session.sync()
    assert torch.all(y == 77)


@pytest.mark.parametrize("kinds", [("f32", "f16"), ("bf16", "bf16")], ids="-".join)
def test_a_million_tokens_in_one_page(hip, kinds):
    rng = np.random.default_rng(25)
    for lengths, cached in [([1], [2 ** 20 - 1]), ([100], [10 ** 6])]:
        p = Problem(rng, lengths, cached, heads=1, kv_heads=1, head_dim=16, kinds=kinds, page=2 ** 20, extra_pages=0)
        session = p.open()
        p.call(session)
        session.sync()
        p.check()


@pytest.mark.parametrize("kinds", [("f32", "f16"), ("bf16", "bf16")], ids="-".join)
@pytest.mark.parametrize("spare", [3, 700])
def test_calls_without_a_row(hip, kinds, spare):
    """Rows that belong to no sequence only, and one sequence among many empty ones."""
    rng = np.random.default_rng(26)
    for lengths in ([0, 0], [0] * 300 + [2] + [0] * 30):
        p = Problem(rng, lengths, [5] * len(lengths), kinds=kinds, spare=spare)
        session = p.open()
        p.call(session)
        session.sync()
        p.check()


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("rows", [9, 150])
def test_queries_that_are_no_numbers_spoil_their_own_rows(hip, kinds, bad, rows):
    import torch
    rng = np.random.default_rng(27)
    p = Problem(rng, [rows], [70], kinds=kinds, heads=4, kv_heads=2)
    p.q[3, 1, 5] = bad
    p.d[0].copy_(torch.from_numpy(p.q.reshape(rows, -1)).to(p.d[0].dtype))
    torch.cuda.synchronize()
    session = p.open()
    p.call(session)
    session.sync()
    torch.cuda.synchronize()
    y = p.y.float().cpu().numpy().reshape(rows, 4, 64)
    assert not np.any(np.isfinite(y[3, 1]))
    p.q[3, 1, 5] = 0
    page, at = p.places(0)
    for pool, new in ((p.keys, p.k), (p.values, p.v)):
        pool[0, page[70:], :, at[70:]] = ref.rounded(new, kinds[1])
    want, bound = ref.attention(p.q, *(pool[0, page, :, at] for pool in (p.keys, p.values)), ref.sees(rows, 70),
                                np.float32(p.scale), *kinds)
    good = np.ones((rows, 4), dtype=bool)
    good[3, 1] = False
    assert np.all((np.abs(y - want) <= bound)[good])


def test_a_page_read_twice_by_a_sequence(hip):
    rng = np.random.default_rng(28)
    p = Problem(rng, [1, 30], [70, 64], heads=4, kv_heads=2)
    for i in range(2):
        p.table[i, 1] = p.table[i, 0]
        p.d_table[i, 1] = p.d_table[i, 0]
    import torch
    torch.cuda.synchronize()
    session = p.open()
    p.call(session)
    session.sync()
    p.check()
