"""What a batch of sequences needs between the projections of a hybrid model, as data and as runnable passes.

Three operators, each through the entry point a program calls:
  mixer   HipSsmSession.run_device / step_device: the short causal convolution,
          the selective state space scan and the gated group norm of a Mamba-2
          mixer, from ssm_in's rows to ssm_out's, for prompts of several
          lengths and for one token of each sequence
  route   HipRouter.run_device: experts and weights from router logits
  sample  HipBatchSampler.sample_device: the next token of each row of logits

With `own` false the same values come from elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

# heads, head width, groups of heads that share B and C, state size, taps
HYBRID = dict(heads=64, head_dim=64, groups=8, state=128, conv=4)


def listed():
    return [
        # one sequence's next token: the smallest call, latency
        {"name": "mixer_step_1", "path": "step", "sequences": 1, **HYBRID},
        # the next token of some sequences decoded together
        {"name": "mixer_step_48", "path": "step", "sequences": 48, **HYBRID},
        # many sequences, heads of another width, one group, three taps
        {"name": "mixer_step_203", "path": "step", "sequences": 203, "heads": 24, "head_dim": 80,
         "groups": 1, "state": 64, "conv": 3},
        # a short prompt of a new sequence
        {"name": "mixer_prompt_33", "path": "prompt", "sequences": 1, "tokens": 33, "fresh": 1.0, **HYBRID},
        # prompts of several lengths, some continuing: a server's ordinary prefill
        {"name": "mixer_prompts_2311", "path": "prompt", "sequences": 9, "tokens": 2311, "fresh": 0.5, **HYBRID},
        # one long prompt, wide heads, a state of 256
        {"name": "mixer_prompt_wide_3000", "path": "prompt", "sequences": 1, "tokens": 3000, "fresh": 1.0,
         "heads": 32, "head_dim": 128, "groups": 2, "state": 256, "conv": 4},
        # one long prompt's chunk: the largest call
        {"name": "mixer_prompt_8192", "path": "prompt", "sequences": 1, "tokens": 8192, "fresh": 0.0, **HYBRID},
        # one token's experts: biased selection, sigmoid scores (latency)
        {"name": "route_1", "path": "route", "tokens": 1, "experts": 128, "top_k": 6, "score": "sigmoid",
         "bias": True, "groups": 1, "top_groups": 1, "group_rank": 1, "norm": True, "scale": 2.5},
        # a batch over grouped experts
        {"name": "route_grouped_301", "path": "route", "tokens": 301, "experts": 256, "top_k": 8,
         "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "group_rank": 2, "norm": True,
         "scale": 2.5},
        # a long prompt's tokens over 512 experts, softmax scores
        {"name": "route_8192", "path": "route", "tokens": 8192, "experts": 512, "top_k": 10,
         "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_rank": 1, "norm": True,
         "scale": 1.0},
        # one sequence's token with the usual filters (latency)
        {"name": "sample_1", "path": "sample", "rows": 1, "vocab": 128256, "filters": "all"},
        # a large batch, each row with filters of its own
        {"name": "sample_160", "path": "sample", "rows": 160, "vocab": 128256, "filters": "mixed"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


STATE = 64 * 64 * 128  # state elements of a HYBRID sequence


def draw(rng):
    path = rng.choice(["step", "prompt", "prompt", "route", "sample"])
    if path in ("step", "prompt"):
        groups = rng.choice([1, 1, 2, 4, 8])
        head_dim = rng.choice([32, 64, 64, 80, 128])
        state = rng.choice([16, 64, 128, 128, 256])
        heads = groups * rng.choice([2, 3, 4, 7, 8, 16])
        heads = max(groups, min(heads, STATE // (head_dim * state) // groups * groups))
        layout = rng.choice([HYBRID, dict(heads=heads, head_dim=head_dim, groups=groups, state=state,
                                          conv=rng.choice([2, 3, 4, 4]))])
        if path == "step":
            return {"path": path, "sequences": _log(rng, 1, 100), **layout}
        tokens = _log(rng, 2, 6000)
        return {"path": path, "sequences": min(tokens, _log(rng, 1, 24)), "tokens": tokens,
                "fresh": rng.choice([0.0, 0.5, 1.0]), **layout}
    if path == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, 8, 512 // groups)
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(16, top_groups * (experts // groups)))
        bias = rng.random() < 0.5
        return {"path": path, "tokens": _log(rng, 1, 8192), "experts": experts, "top_k": top_k,
                "score": rng.choice(["softmax", "sigmoid"]), "bias": bias, "groups": groups,
                "top_groups": top_groups, "group_rank": rng.choice([1, 2]),
                "norm": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5])}
    return {"path": path, "rows": _log(rng, 1, 160), "vocab": rng.choice([32000, 128256, _log(rng, 8000, 128256)]),
            "filters": rng.choice(["all", "top_k", "top_p", "min_p", "none", "mixed"])}


# ------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _uniform(g, lo, hi, *shape):
    return torch.rand(shape, device="cuda", generator=g) * (hi - lo) + lo


def _lengths(tokens, sequences, rng):
    """`sequences` lengths that sum to `tokens`: log-normal sizes, one of them a single token."""
    if sequences == 1:
        return [tokens]
    share = np.exp(rng.normal(size=sequences))
    lengths = np.floor(share / share.sum() * tokens).astype(int)
    lengths[0] = min(1, tokens)
    lengths[-1] += tokens - lengths.sum()
    return [int(v) for v in lengths]


def _mixer(case, seed):
    """The layer's tensors and ssm_in's rows on the device; the state pool's first half holds the
    sequences' states, its second half receives them (a program that may go back to the earlier ones)."""
    g, rng = _generator(seed), np.random.default_rng(seed)
    h, p, gr, n, w = (case[k] for k in ("heads", "head_dim", "groups", "state", "conv"))
    inner, channels, s = h * p, h * p + 2 * gr * n, case["sequences"]
    step = torch.exp(_uniform(g, math.log(1e-3), math.log(1e-1), h))
    t = {"conv_weight": _randn(g, channels, w) * 0.5, "conv_bias": _randn(g, channels) * 0.1,
         "dt_bias": step + torch.log(-torch.expm1(-step)), "a": -_uniform(g, 1.0, 16.0, h),
         "d": 1 + 0.1 * _randn(g, h), "norm": 1 + 0.1 * _randn(g, inner), "epsilon": 1e-5}
    lengths = [1] * s if case["path"] == "step" else _lengths(case["tokens"], s, rng)
    tokens = sum(lengths)
    x = _randn(g, tokens, inner + channels + h)
    x[:, inner + channels:] *= 0.5
    conv = _randn(g, 2 * s, w - 1, channels)
    ssm = _randn(g, 2 * s, h, p, n) * 0.5
    old = rng.permutation(s)
    if case["path"] == "prompt":
        old[:round(s * case["fresh"])] = -1  # new sequences start from nothing
    t |= {"x": x, "conv_states": conv, "ssm_states": ssm, "lengths": lengths,
          "offsets": torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda"),
          "old": torch.tensor(old, dtype=torch.int32, device="cuda"),
          "new": torch.tensor(s + rng.permutation(s), dtype=torch.int32, device="cuda")}
    return t


def _routes(case, seed):
    g = _generator(seed)
    logits = _randn(g, case["tokens"], case["experts"]) * 1.5
    bias = _randn(g, case["experts"]) * 0.1 if case["bias"] else None
    return {"logits": logits, "bias": bias}


def _rows(case, seed):
    """Logits of an output head (N(0, 3) with some likely tokens), and each row's filters and random number."""
    g, rng = _generator(seed), np.random.default_rng(seed)
    r, v, kind = case["rows"], case["vocab"], case["filters"]
    logits = _randn(g, r, v) * 3
    logits.scatter_add_(1, torch.randint(0, v, (r, 20), device="cuda", generator=g), 6 + _randn(g, r, 20))
    use = {"all": "kpm", "top_k": "k", "top_p": "p", "min_p": "m", "none": "", "mixed": "kpm"}[kind]

    def each(choices, off, letter, dtype):
        if letter not in use:
            return None
        values = rng.choice(choices, size=r)
        if kind == "mixed":
            values = np.where(rng.random(r) < 0.5, values, off)
        return torch.tensor(values, dtype=dtype, device="cuda")

    return {"logits": logits,
            "random": torch.tensor(rng.random(r), dtype=torch.float64, device="cuda").float().clamp(max=1 - 2.0 ** -24),
            "temperature": torch.tensor(rng.choice([0.7, 1.0, 1.3], size=r), dtype=torch.float32, device="cuda"),
            "top_k": each([20, 40, 200], 0, "k", torch.int32),
            "top_p": each([0.8, 0.9, 0.95], 1.0, "p", torch.float32),
            "min_p": each([0.01, 0.05, 0.1], 0.0, "m", torch.float32)}


_STREAM = []


def _stream():
    """The one stream that a program's passes follow each other on."""
    if not _STREAM:
        _STREAM.append(torch.cuda.Stream())
    return _STREAM[0].cuda_stream


def _host(t):
    return None if t is None else t.cpu().numpy()


def prepare(case, seed):
    path = case["path"]
    if path in ("step", "prompt"):
        state = _mixer(case, seed)
        state["y"] = torch.empty((state["x"].shape[0], case["heads"] * case["head_dim"]), device="cuda")
        if own:
            from llambda_amd.ssm import HipSsmSession, SsmLayer
            layer = SsmLayer(heads=case["heads"], head_dim=case["head_dim"], groups=case["groups"],
                             state=case["state"], conv_width=case["conv"],
                             conv_weight=_host(state["conv_weight"]), conv_bias=_host(state["conv_bias"]),
                             dt_bias=_host(state["dt_bias"]), a=_host(state["a"]), d=_host(state["d"]),
                             norm=_host(state["norm"]), norm_epsilon=state["epsilon"])
            state["session"] = HipSsmSession(layer, slots=2 * case["sequences"],
                                             max_tokens=state["x"].shape[0], max_sequences=case["sequences"],
                                             conv_states_ptr=state["conv_states"].data_ptr(),
                                             ssm_states_ptr=state["ssm_states"].data_ptr())
    elif path == "route":
        state = _routes(case, seed)
        state["indices"] = torch.empty((case["tokens"], case["top_k"]), dtype=torch.int32, device="cuda")
        state["weights"] = torch.empty((case["tokens"], case["top_k"]), device="cuda")
        if own:
            from llambda_amd.moe import HipRouter, Routing
            state["router"] = HipRouter(Routing(
                experts=case["experts"], top_k=case["top_k"], score=case["score"], bias=_host(state["bias"]),
                groups=case["groups"], top_groups=case["top_groups"], group_rank=case["group_rank"],
                weights_norm=case["norm"], weights_scale=case["scale"]))
    else:
        state = _rows(case, seed)
        state["tokens"] = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
        if own:
            from llambda_amd.sampling import HipBatchSampler
            state["sampler"] = HipBatchSampler(case["vocab"], case["rows"])
    state["case"] = case
    state["stream"] = _stream()
    torch.cuda.synchronize()
    return state


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def run(state):
    path = state["case"]["path"]
    if not own:
        return (_mixer_plain if path in ("step", "prompt") else _route_plain if path == "route" else _sample_plain)(state)
    if path in ("step", "prompt"):
        session, s = state["session"], state["case"]["sequences"]
        if path == "step":
            session.step_device(_ptr(state["x"]), _ptr(state["y"]), s, _ptr(state["old"]), _ptr(state["new"]),
                                state["stream"])
        else:
            session.run_device(_ptr(state["x"]), _ptr(state["y"]), state["x"].shape[0], _ptr(state["offsets"]), s,
                               _ptr(state["old"]), _ptr(state["new"]), state["stream"])
        return {"y": state["y"], "conv": state["conv_states"][s:], "ssm": state["ssm_states"][s:]}
    if path == "route":
        state["router"].run_device(_ptr(state["logits"]), _ptr(state["indices"]), _ptr(state["weights"]),
                                   state["case"]["tokens"], state["stream"])
        return {"indices": state["indices"], "weights": state["weights"]}
    state["sampler"].sample_device(_ptr(state["logits"]), state["case"]["rows"], _ptr(state["tokens"]),
                                   _ptr(state["random"]), temperature_ptr=_ptr(state["temperature"]),
                                   top_k_ptr=_ptr(state["top_k"]), top_p_ptr=_ptr(state["top_p"]),
                                   min_p_ptr=_ptr(state["min_p"]), stream=state["stream"])
    return {"tokens": state["tokens"]}


# ------------------------------------------------------------------ plain forms

CHUNK = 64


def _silu(v):
    return v / (1 + torch.exp(-v))


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _gated_norm(y, z, s, groups):
    g = (y * _silu(z)).reshape(*y.shape[:-1], groups, -1)
    g = g / torch.sqrt((g * g).mean(-1, keepdim=True) + s["epsilon"])
    return g.reshape(y.shape) * s["norm"]


def _earlier(pool, old):
    """The sequences' states, zeros for new ones."""
    return torch.where((old >= 0).reshape(-1, *[1] * (pool.dim() - 1)), pool[old.clamp(min=0).long()], 0.0)


def _placed(values, new, first):
    out = torch.empty_like(values)
    out[new.long() - first] = values
    return out


def _mixer_plain(s):
    """Sequences padded to whole chunks [b][L]; within a chunk the masked product form, between
    chunks the states by one product with the chunks' decays."""
    c = s["case"]
    h, p, gr, n, w, b = (c[k] for k in ("heads", "head_dim", "groups", "state", "conv", "sequences"))
    inner, channels, q = h * p, h * p + 2 * gr * n, CHUNK if c["path"] == "prompt" else 1
    x, dev = s["x"], s["x"].device
    chunks = max(1, -(-max(s["lengths"]) // q))
    long = chunks * q
    lengths = (s["offsets"][1:] - s["offsets"][:-1]).long()
    row = torch.repeat_interleave(torch.arange(b, device=dev), lengths, output_size=x.shape[0])
    at = torch.arange(x.shape[0], device=dev) - s["offsets"][row].long()
    raw = torch.zeros((b, w - 1 + long, channels), device=dev)
    raw[:, :w - 1] = _earlier(s["conv_states"], s["old"])
    raw[row, w - 1 + at] = x[:, inner:inner + channels]
    u = s["conv_bias"] + sum(s["conv_weight"][:, k] * raw[:, k:k + long] for k in range(w))
    u = _silu(u)
    conv = torch.gather(raw, 1, (lengths[:, None, None] + torch.arange(w - 1, device=dev)[None, :, None])
                        .expand(b, w - 1, channels))
    dt = torch.zeros((b, long, h), device=dev)
    dt[row, at] = _softplus(x[:, inner + channels:] + s["dt_bias"])
    xs = u[..., :inner].reshape(b, chunks, q, h, p).permute(0, 1, 3, 2, 4)        # [b][c][h][q][p]
    bs = u[..., inner:inner + gr * n].reshape(b, chunks, q, gr, n).permute(0, 1, 3, 2, 4)
    cs = u[..., inner + gr * n:].reshape(b, chunks, q, gr, n).permute(0, 1, 3, 2, 4)
    share = h // gr
    dts = dt.reshape(b, chunks, q, h).permute(0, 1, 3, 2)                         # [b][c][h][q]
    # logarithms of decays are differences of long sums: in 64 bits
    run_ = torch.cumsum(dts.double() * s["a"].double()[None, None, :, None], -1)
    total = torch.cumsum(run_[..., -1], 1)                                        # [b][c][h]
    mask = torch.ones((q, q), dtype=torch.bool, device=dev).tril()
    decay = torch.exp(torch.where(mask, run_[..., :, None] - run_[..., None, :], -math.inf)).float()
    m = torch.matmul(cs, bs.transpose(-1, -2)).repeat_interleave(share, 2) * decay * dts[..., None, :]
    left = (torch.exp(run_[..., -1:] - run_).float() * dts)[..., None] * xs       # [b][c][h][q][p]
    bh, ch = bs.repeat_interleave(share, 2), cs.repeat_interleave(share, 2)
    local = torch.matmul(left.transpose(-1, -2), bh)                              # [b][c][h][p][n]
    start = _earlier(s["ssm_states"], s["old"])
    parts = torch.cat([start[:, None], local], 1).permute(0, 2, 1, 3, 4).reshape(b, h, chunks + 1, p * n)
    t = torch.cat([torch.zeros_like(total[:, :1]), total], 1).permute(0, 2, 1)    # [b][h][c + 1]
    mask = torch.ones((chunks + 1, chunks + 1), dtype=torch.bool, device=dev).tril()
    between = torch.exp(torch.where(mask, t[..., :, None] - t[..., None, :], -math.inf)).float()
    states = torch.matmul(between, parts).reshape(b, h, chunks + 1, p, n).permute(0, 2, 1, 3, 4)
    y = torch.matmul(m, xs) + s["d"][None, None, :, None, None] * xs
    y = y + torch.exp(run_).float()[..., None] * torch.matmul(ch, states[:, :-1].transpose(-1, -2))
    y = y.permute(0, 1, 3, 2, 4).reshape(b, long, inner)[row, at]
    return {"y": _gated_norm(y, x[:, :inner], s, gr), "conv": _placed(conv, s["new"], b),
            "ssm": _placed(states[:, -1], s["new"], b)}


def _route_plain(s):
    """In 64 bits: the order of scores that differ by little decides whole numbers."""
    c = s["case"]
    l = s["logits"].double()
    if c["score"] == "softmax":
        e = torch.exp(l - l.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-l))
    choice = score if s["bias"] is None else score + s["bias"].double()
    if c["groups"] > 1:
        t, g = c["tokens"], c["groups"]
        rank = torch.sort(choice.reshape(t, g, -1), dim=2, descending=True).values[:, :, :c["group_rank"]].sum(2)
        best = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        open_ = torch.zeros((t, g), dtype=torch.bool, device=l.device).scatter_(1, best, True)
        choice = torch.where(open_.repeat_interleave(c["experts"] // g, 1), choice, -math.inf)
    indices = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
    weights = torch.gather(score, 1, indices)
    if c["norm"]:
        weights = weights / weights.sum(1, keepdim=True)
    return {"indices": indices.int(), "weights": (weights * c["scale"]).float()}


def _sample_plain(s):
    """In 64 bits: a running sum next to the random number's decides whole numbers."""
    l = s["logits"]
    rows, vocab = l.shape
    value, index = torch.sort(l, dim=1, descending=True, stable=True)
    value = value.double() / s["temperature"].double()[:, None]
    p = torch.exp(value - value[:, :1])
    rank = torch.arange(vocab, device=l.device)[None]
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        p = torch.where((k > 0) & (rank >= k), 0.0, p)
    if s["top_p"] is not None:
        total = torch.cumsum(p, 1)
        keep = total - p < s["top_p"].double()[:, None] * total[:, -1:]
        p = torch.where(keep | (s["top_p"][:, None] >= 1), p, 0.0)
    if s["min_p"] is not None:
        p = torch.where(p >= s["min_p"].double()[:, None], p, 0.0)
    total = torch.cumsum(torch.zeros_like(p).scatter_(1, index, p), 1)
    token = (total <= s["random"].double()[:, None] * total[:, -1:]).sum(1)
    return {"tokens": token.int()}


# ------------------------------------------------------------------ work

def work(case):
    path = case["path"]
    if path in ("step", "prompt"):
        h, p, g, n, w, s = (case[k] for k in ("heads", "head_dim", "groups", "state", "conv", "sequences"))
        t = s if path == "step" else case["tokens"]
        inner, channels = h * p, h * p + 2 * g * n
        read = s - (round(s * case["fresh"]) if path == "prompt" else 0)
        state = 4 * (inner * n + (w - 1) * channels)
        return {"bytes": 4 * t * (2 * inner + channels + h) + state * (read + s)
                + 4 * (channels * (w + 1) + 3 * h + inner),
                # the recurrence: decay and update of each state element, its product with C
                "flops": t * (5 * inner * n + (2 * w + 4) * channels + 10 * inner)}
    if path == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": 4 * t * e + 8 * t * k + (4 * e if case["bias"] else 0), "flops": 10 * t * e}
    return {"bytes": case["rows"] * (4 * case["vocab"] + 4 * 6), "flops": 10 * case["rows"] * case["vocab"]}


# ------------------------------------------------------------------ outputs

def exact(case, seed):
    """What run() returns, in 64 bits; whole numbers have no such value."""
    path = case["path"]
    if path == "sample":
        return None
    if path == "route":
        return {"indices": None, "weights": _exact_weights(case, seed)}
    return _exact_mixer(case, seed)


def _exact_weights(case, seed):
    s = _routes(case, seed)
    l = _host(s["logits"]).astype(np.float64)
    bias = np.zeros(case["experts"]) if s["bias"] is None else _host(s["bias"]).astype(np.float64)
    out = np.empty((case["tokens"], case["top_k"]))
    size = case["experts"] // case["groups"]
    for t in range(case["tokens"]):
        v = np.exp(l[t] - l[t].max()) if case["score"] == "softmax" else 1 / (1 + np.exp(-l[t]))
        v = v / v.sum() if case["score"] == "softmax" else v
        choice = v + bias
        groups = choice.reshape(-1, size)
        best = np.argsort(-np.sort(groups, axis=1)[:, ::-1][:, :case["group_rank"]].sum(1), kind="stable")
        order = [e for e in np.argsort(-choice, kind="stable")
                 if e // size in best[:case["top_groups"]]][:case["top_k"]]
        out[t] = v[order] / (v[order].sum() if case["norm"] else 1) * case["scale"]
    return torch.from_numpy(out).cuda()


def _exact_mixer(case, seed):
    """The recurrence, token by token over all sequences at once."""
    s = _mixer(case, seed)
    h, p, g, n, w, b = (case[k] for k in ("heads", "head_dim", "groups", "state", "conv", "sequences"))
    inner, channels = h * p, h * p + 2 * g * n
    f = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point() and k != "ssm_states"}
    known = s["old"] >= 0
    taps = f["conv_states"][s["old"].clamp(min=0).long()] * known[:, None, None]
    hidden = s["ssm_states"][s["old"].clamp(min=0).long()].double() * known[:, None, None, None]
    y = torch.empty((s["x"].shape[0], inner), dtype=torch.float64, device="cuda")
    begin = np.concatenate([[0], np.cumsum(s["lengths"])])[:-1]
    decay = f["a"][None]
    for t in range(max(s["lengths"])):
        live = [i for i in range(b) if s["lengths"][i] > t]
        rows = torch.tensor([int(begin[i]) + t for i in live], device="cuda")
        i = torch.tensor(live, device="cuda")
        v = f["x"][rows]
        window = torch.cat([taps[i], v[:, None, inner:inner + channels]], 1)
        taps[i] = window[:, 1:]
        u = torch.nn.functional.silu((window * f["conv_weight"].T[None]).sum(1) + f["conv_bias"])
        dt = torch.nn.functional.softplus(v[:, inner + channels:] + f["dt_bias"], threshold=700)
        x_t = u[:, :inner].reshape(-1, h, p)
        b_t = u[:, inner:inner + g * n].reshape(-1, g, n).repeat_interleave(h // g, 1)
        c_t = u[:, inner + g * n:].reshape(-1, g, n).repeat_interleave(h // g, 1)
        now = torch.exp(dt * decay)[..., None, None] * hidden[i] + (dt[..., None] * x_t)[..., None] * b_t[:, :, None]
        hidden[i] = now
        y[rows] = ((now * c_t[:, :, None]).sum(-1) + f["d"][None, :, None] * x_t).reshape(-1, inner)
    gated = (y * torch.nn.functional.silu(f["x"][:, :inner])).reshape(-1, g, inner // g)
    gated = gated * torch.rsqrt(gated.square().mean(-1, keepdim=True) + s["epsilon"])
    conv, ssm = torch.empty_like(taps), torch.empty_like(hidden)
    conv[s["new"].long() - b], ssm[s["new"].long() - b] = taps, hidden
    return {"y": gated.reshape(-1, inner) * f["norm"], "conv": conv, "ssm": ssm}
