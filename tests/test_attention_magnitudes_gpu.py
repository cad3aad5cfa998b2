"""Scores far beyond what exponents hold: the largest takes all, equal ones share.  Queries and keys are small whole numbers
times powers of two, so that scores are exact in single precision and the answer is known."""
import numpy as np
import pytest

import attention_reference as ref
from test_attention_gpu import KINDS, Problem, random_tree

pytestmark = pytest.mark.gpu


def whole(rng, shape, power):
    return np.ldexp(rng.integers(-8, 9, size=shape).astype(np.float32), power)


def problem(rng, lengths, cached, power, **more):
    """Scores are whole multiples of 2^power, below 2^(power + 15)."""
    p = Problem(rng, lengths, cached, **more)
    for_q = power // 2 if p.kinds[1] == "f16" else power - power // 3
    p.q[...] = whole(rng, p.q.shape, for_q)
    p.k[...] = whole(rng, p.k.shape, power - for_q)
    p.keys[...] = whole(rng, p.keys.shape, power - for_q)
    p.keys[..., 1::2, :] = p.keys[..., ::2, :]  # cached keys in pairs, whose scores are equal
    return p


def check(p, step=False):
    import torch
    for t, a in ((p.d[0], p.q), (p.d[1], p.k), (p.d_keys, p.keys)):
        t.copy_(torch.from_numpy(a.reshape(t.shape)).to(t.dtype))
    torch.cuda.synchronize()
    session = p.open()
    p.call(session, step=step)
    session.sync()
    torch.cuda.synchronize()
    row, cell = p.kinds
    y = p.y.float().cpu().numpy().reshape(p.tokens, p.heads, p.dim).astype(np.float64)
    group, begin, u, shared = p.heads // p.kv, 0, 2.0 ** -24, 0
    for i, (n, c) in enumerate(zip(p.lengths, p.cached)):
        mine = slice(begin, begin + n)
        begin += n
        page, at = p.places(i)
        keys, values = (pool[p.layer, page, :, at].copy() for pool in (p.keys, p.values))
        keys[c:], values[c:] = p.k[mine], ref.rounded(p.v[mine], cell)
        sees = ref.sees(n, c, None if p.trees is None else p.trees[i])
        for h in range(p.heads):
            s = np.where(sees, p.q[mine, h].astype(np.float64) @ keys[:, h // group].astype(np.float64).T, -np.inf)
            first = s == s.max(1, keepdims=True)
            # the others have less than exp(-200) of a weight
            assert np.all((s.max(1, keepdims=True) - s)[~first] * p.scale > 200)
            shared += int((first.sum(1) > 1).sum())
            weight = first / first.sum(1, keepdims=True)
            v = values[:, h // group].astype(np.float64)
            want, reach = weight @ v, weight @ np.abs(v)
            # the bound of attention_reference with exact scores
            bound = (16 + sees.sum(1, keepdims=True) / 8 + 64) * u * reach + 2.0 ** -33 * (sees @ np.abs(v))
            if row != "f32":
                bound += 1.001 * ref.EPS[row] / 2 * (reach + np.abs(want)) + 2.0 ** -24
            off = np.abs(y[mine, h] - want)
            assert np.all(off <= bound), f"sequence {i}, head {h}: rows {np.flatnonzero(~(off <= bound).all(1))[:5]}"
    assert shared, "some rows were to have several largest scores"


def powers(kinds):
    """Largest scores from 2^25 to the end of the type."""
    return (14, 20, 24) if "f16" in kinds else (14, 20, 30, 60, 110)


CASES = [(k, n) for k in KINDS for n in powers(k)]
NAMES = ["-".join(k) + f"-{n}" for k, n in CASES]


@pytest.mark.parametrize("kinds, power", CASES, ids=NAMES)
@pytest.mark.parametrize("head_dim", [64, 80, 128, 256])
def test_steps_and_prompts(hip, kinds, power, head_dim):
    rng = np.random.default_rng(50)
    more = dict(heads=8, kv_heads=2, head_dim=head_dim, kinds=kinds)
    check(problem(rng, [1] * 6, [40, 0, 64, 500, 1100, 31], power, **more), step=True)
    check(problem(rng, [150, 90], [70, 33], power, **more))
    check(problem(rng, [1, 2] * 150, [40, 33] * 150, power, **more))


@pytest.mark.parametrize("kinds, power", CASES, ids=NAMES)
def test_parts_and_trees(hip, kinds, power):
    rng = np.random.default_rng(51)
    more = dict(heads=8, kv_heads=2, head_dim=64, kinds=kinds)
    check(problem(rng, [1, 1], [9000, 77], power, **more), step=True)
    check(problem(rng, [300, 3], [5000, 4], power, **more))
    check(problem(rng, [20, 5], [70, 0], power, trees=[random_tree(rng, 20), random_tree(rng, 5)], **more))
    check(problem(rng, [200], [70], power, trees=[random_tree(rng, 200)], **more))


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("rows", [9, 150])
def test_scores_rise_from_far_below(hip, kinds, rows):
    """The first keys' scores lie at -2^35 and near, the last ones' at zero: what the first left must leave no trace."""
    rng = np.random.default_rng(52)
    p = problem(rng, [rows], [1000], 20, heads=8, kv_heads=2, head_dim=64, kinds=kinds)
    p.q[...] = np.abs(p.q) + np.ldexp(np.float32(1), 10)
    p.keys[...] = -np.abs(p.keys) - np.ldexp(np.float32(1), 10)
    last = p.table[0, 62], slice(None), 7  # position 999
    p.keys[0][last] = 0
    p.k[...] = -np.abs(p.k) - np.ldexp(np.float32(1), 10)
    p.k[-1] = 0  # the last row has two
    check(p)


@pytest.mark.parametrize("kinds", [("f32", "bf16"), ("f32", "f32")], ids="-".join)
@pytest.mark.parametrize("q_size, k_size", [(3e38, 3e-38), (1e30, 1e-30), (1e-30, 1e30), (1e-36, 1e36), (1e-38, 3e37)])
@pytest.mark.parametrize("rows", [9, 150])
def test_small_rows_of_large_keys(hip, kinds, q_size, k_size, rows):
    """Scores next to one, of queries and keys that are next to the ends of the type."""
    import torch
    rng = np.random.default_rng(53)
    p = Problem(rng, [rows, 1], [70, 300], heads=4, kv_heads=2, kinds=kinds)
    p.q = (np.clip(p.q / 6, -1, 1) * np.float32(q_size)).astype(np.float32)
    p.k, p.keys = (ref.rounded(a * np.float32(k_size), kind) for a, kind in ((p.k, "f32"), (p.keys, kinds[1])))
    for t, a in ((p.d[0], p.q), (p.d[1], p.k), (p.d_keys, p.keys)):
        t.copy_(torch.from_numpy(a.reshape(t.shape)).to(t.dtype))
    torch.cuda.synchronize()
    session = p.open()
    p.call(session)
    session.sync()
    p.check()
