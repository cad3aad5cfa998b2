"""Keys that hold infinities: a score of -inf has no weight, whatever the types and the heads' width; one of +inf, or one
that is no number, leaves its row without a distribution."""
import numpy as np
import pytest

import attention_reference as ref
from test_attention_gpu import KINDS, Problem, random_tree

pytestmark = pytest.mark.gpu


def put(p, bad):
    """Infinities in keys: bad lists (sequence, position, kv head, element, value), at cached positions and new ones."""
    import torch
    starts = np.concatenate([[0], np.cumsum(p.lengths)])
    for i, at, h, d, value in bad:
        if at < p.cached[i]:
            p.keys[p.layer, p.table[i, at // p.page], h, at % p.page, d] = value
        else:
            p.k[starts[i] + at - p.cached[i], h, d] = value
    p.d_keys.copy_(torch.from_numpy(p.keys).to(p.d_keys.dtype))
    p.d[1].copy_(torch.from_numpy(p.k.reshape(p.tokens, -1)).to(p.d[1].dtype))
    torch.cuda.synchronize()


def check(p):
    """Against 64 bits over the keys whose score is not -inf.  Returns how many rows have a result and how many none."""
    import torch
    torch.cuda.synchronize()
    row, cell = p.kinds
    y = p.y.float().cpu().numpy().reshape(p.tokens, p.heads, p.dim)
    group, begin, finite, none = p.heads // p.kv, 0, 0, 0
    for i, (n, c) in enumerate(zip(p.lengths, p.cached)):
        mine = slice(begin, begin + n)
        begin += n
        page, at = p.places(i)
        keys, values = (pool[p.layer, page, :, at].copy() for pool in (p.keys, p.values))
        keys[c:], values[c:] = ref.rounded(p.k[mine], cell), ref.rounded(p.v[mine], cell)
        sees = ref.sees(n, c, None if p.trees is None else p.trees[i])
        for h in range(p.heads):
            with np.errstate(invalid="ignore"):
                s = np.einsum("rd,kd->rk", p.q[mine, h].astype(np.float64), keys[:, h // group].astype(np.float64))
            empty = (sees & ~(s < np.inf)).any(1) | ~(sees & (s > -np.inf)).any(1)  # no softmax, or none left
            tame = np.where(np.isfinite(keys[:, h // group:h // group + 1]), keys[:, h // group:h // group + 1], 0)
            want, bound = ref.attention(p.q[mine, h:h + 1], tame, values[:, h // group:h // group + 1],
                                        sees & (s > -np.inf), np.float32(p.scale), row, cell)
            got = y[mine, h]
            assert not np.any(np.isfinite(got[empty])), f"sequence {i}, head {h}"
            off = np.abs(got - want[:, 0])[~empty]
            assert np.all(off <= bound[~empty, 0]), (f"sequence {i}, head {h}: rows "
                                                     f"{np.flatnonzero(~empty)[~(off <= bound[~empty, 0]).all(1)]}")
            none += int(empty.sum())
            finite += int((~empty & (sees & (s == -np.inf)).any(1)).sum())
    return finite, none


def run(p, step=False):
    session = p.open()
    p.call(session, step=step)
    session.sync()
    finite, none = check(p)
    assert finite and none, "the keys were to leave rows of both kinds"


WIDTHS = [16, 48, 64, 80, 112, 128, 208, 256]


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("head_dim", WIDTHS)
@pytest.mark.parametrize("shape", ["steps", "prompts", "many"])
def test_infinite_keys(hip, kinds, head_dim, shape):
    """In a key's first elements, its last and between; one element of a key and several; cached keys and new ones."""
    rng = np.random.default_rng(40)
    if shape == "steps":
        lengths, cached = [1] * 8, [40, 33, 64, 500, 1100, 20, 90, 31]
    elif shape == "prompts":
        lengths, cached = [150, 90], [70, 33]
    else:  # more sequences than plan for themselves
        lengths, cached = [1, 2] * 150, [40, 33] * 150
    p = Problem(rng, lengths, cached, heads=8, kv_heads=2, head_dim=head_dim, kinds=kinds)
    inf = np.float32(np.inf)
    bad = [(0, 5, 0, 1, inf), (0, 39, 1, head_dim - 1, -inf), (1, 7, 0, 7, -inf), (1, 32, 1, head_dim // 2, inf),
           (1, 32, 1, 3, inf), (1, 33, 0, 0, inf)]
    if shape == "prompts":
        bad += [(0, 100, 1, 2, inf), (0, 180, 0, head_dim - 2, -inf)]
    put(p, bad)
    run(p, step=shape == "steps")


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("head_dim", [64, 80, 256])
def test_infinite_keys_of_long_contexts(hip, kinds, head_dim):
    """Positions in parts that are joined, rows that share keys and rows that do not."""
    rng = np.random.default_rng(41)
    inf = np.float32(np.inf)
    p = Problem(rng, [1, 1], [9000, 77], heads=8, kv_heads=2, head_dim=head_dim, kinds=kinds)
    put(p, [(0, 17, 0, 1, inf), (0, 8000, 1, 4, inf), (1, 30, 0, head_dim - 1, -inf)])
    run(p, step=True)
    p = Problem(rng, [300, 3], [5000, 4], heads=8, kv_heads=2, head_dim=head_dim, kinds=kinds)
    put(p, [(0, 17, 0, 1, inf), (0, 4999, 1, 4, inf), (0, 5100, 1, 0, -inf)])
    run(p)


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("nodes", [20, 200])
def test_infinite_keys_of_trees(hip, kinds, nodes):
    rng = np.random.default_rng(42)
    inf = np.float32(np.inf)
    p = Problem(rng, [nodes, 5], [70, 0], heads=8, kv_heads=2, head_dim=80, kinds=kinds,
                trees=[random_tree(rng, nodes), random_tree(rng, 5)])
    put(p, [(0, 3, 0, 2, inf), (0, 70, 1, 79, -inf), (0, 75, 1, 40, inf), (1, 0, 0, 5, inf)])
    run(p)


@pytest.mark.parametrize("kinds", [("f32", "f16")], ids="-".join)
def test_keys_beyond_the_caches_range(hip, kinds):
    """Rows in single precision whose keys become infinities in the cache."""
    rng = np.random.default_rng(43)
    p = Problem(rng, [90], [20], heads=8, kv_heads=2, head_dim=64, kinds=kinds)
    put(p, [(0, 25, 0, 9, np.float32(1e5)), (0, 60, 1, 33, np.float32(-3e30))])
    run(p)


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
def test_every_score_is_infinite(hip, kinds):
    """A row that has no weight left has no result, wherever its keys are; zeros times infinities are no numbers."""
    import torch
    rng = np.random.default_rng(44)
    p = Problem(rng, [40, 1], [3, 700], heads=4, kv_heads=2, head_dim=48, kinds=kinds)
    p.keys[..., 5] = np.inf
    p.k[..., 5] = np.inf
    p.q[:, 0, 5] = -np.abs(p.q[:, 0, 5])
    p.q[:, 1, 5] = 0
    p.d[0].copy_(torch.from_numpy(p.q.reshape(p.tokens, -1)).to(p.d[0].dtype))
    put(p, [])
    session = p.open()
    p.call(session)
    session.sync()
    torch.cuda.synchronize()
    assert not np.any(np.isfinite(p.y.float().cpu().numpy()))
