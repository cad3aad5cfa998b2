"""What a server needs around attention and drafted tokens, as data and as runnable passes.

Three operators, each through the entry point a program calls:
  attend  HipAttentionSession.run_device: keys and values of new rows into a paged
          cache, and causal attention of the rows over it with grouped heads; packed
          prompts of several lengths, or one row of each sequence
  tree    the same call with each row's parent: drafted tokens that see the cached
          ones and their own ancestors; then accept_device, which moves the keys
          and values of an accepted path behind the cached ones
  score   HipTokenScorer.score_device: log probabilities of given tokens, the
          entropy and the top alternatives of rows of logits

With `own` false the same values come from elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# 32 heads of 128 over 8 of keys and values, the layout of the benchmark's decode token
GROUPED = dict(heads=32, kv_heads=8, head_dim=128)


def listed():
    return [
        # the next token of one sequence: the smallest call, latency
        {"name": "attend_step_1", "path": "attend", "sequences": 1, "tokens": 1, "cached": 4096, "step": True,
         "rows": "f32", "cache": "f16", "page": 64, **GROUPED},
        # the next token of some sequences decoded together
        {"name": "attend_step_48", "path": "attend", "sequences": 48, "tokens": 48, "cached": 150000, "step": True,
         "rows": "f32", "cache": "f16", "page": 64, **GROUPED},
        # a short prompt of a new sequence
        {"name": "attend_prompt_33", "path": "attend", "sequences": 1, "tokens": 33, "cached": 0, "step": False,
         "rows": "f32", "cache": "f16", "page": 64, **GROUPED},
        # prompts of several lengths, some continuing: a server's ordinary prefill
        {"name": "attend_prompts_2311", "path": "attend", "sequences": 9, "tokens": 2311, "cached": 5000, "step": False,
         "rows": "f32", "cache": "f16", "page": 16, **GROUPED},
        # single precision throughout, as the Llama-layout session keeps its cache; narrow heads, seven to a group
        {"name": "attend_prompt_f32_1501", "path": "attend", "sequences": 1, "tokens": 1501, "cached": 0, "step": False,
         "rows": "f32", "cache": "f32", "page": 128, "heads": 28, "kv_heads": 4, "head_dim": 64},
        # rows that come in 16 bits, two long prompts
        {"name": "attend_prompts_bf16_6000", "path": "attend", "sequences": 2, "tokens": 6000, "cached": 0, "step": False,
         "rows": "bf16", "cache": "bf16", "page": 64, **GROUPED},
        # one long prompt's chunk: the largest call
        {"name": "attend_prompt_8192", "path": "attend", "sequences": 1, "tokens": 8192, "cached": 0, "step": False,
         "rows": "f32", "cache": "f16", "page": 64, **GROUPED},
        # a small tree drafted for one sequence (latency)
        {"name": "tree_1x26", "path": "tree", "sequences": 1, "tokens": 26, "cached": 2000,
         "rows": "f32", "cache": "f16", "page": 64, **GROUPED},
        # trees of some sequences, rows in 16 bits, wide heads, eight to a group
        {"name": "tree_16x61", "path": "tree", "sequences": 16, "tokens": 976, "cached": 50000,
         "rows": "bf16", "cache": "bf16", "page": 32, "heads": 16, "kv_heads": 2, "head_dim": 256},
        # one row's drawn token and its alternatives, as a served answer reports them (latency)
        {"name": "score_1", "path": "score", "rows": 1, "vocab": 128256, "given": 1, "top": 5},
        # the rows of drafted tokens: each node's children are scored, twenty alternatives
        {"name": "score_61", "path": "score", "rows": 61, "vocab": 128256, "given": 3, "top": 20},
        # a prompt's own tokens scored
        {"name": "score_2048", "path": "score", "rows": 2048, "vocab": 128256, "given": 1, "top": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["attend", "attend", "tree", "score"])
    if path == "score":
        vocab = rng.choice([32000, 128256, _log(rng, 1000, 128256)])
        return {"path": path, "rows": _log(rng, 1, 1500), "vocab": vocab, "given": rng.choice([0, 1, 1, 4]),
                "top": rng.choice([0, 1, 5, 20, 50])}
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8])
    head_dim = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
    rows, cache = rng.choice([("f32", "f16"), ("f32", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f16", "f16"),
                              ("bf16", "bf16")])
    layout = {"rows": rows, "cache": cache, "page": rng.choice([16, 32, 64, 128, 256]), "heads": heads,
              "kv_heads": kv_heads, "head_dim": head_dim}
    room = 100_000_000 // (kv_heads * head_dim * (2 if cache == "f32" else 1))  # cached tokens of all sequences
    if path == "tree":
        sequences = _log(rng, 1, 24)
        return {"path": path, "sequences": sequences, "tokens": sequences * _log(rng, 1, 100),
                "cached": min(room, sequences * _log(rng, 1, 8000)), **layout}
    if rng.random() < 0.4:
        sequences = _log(rng, 1, 100)
        return {"path": path, "sequences": sequences, "tokens": sequences, "step": True,
                "cached": min(room, sequences * _log(rng, 1, 12000)), **layout}
    tokens = _log(rng, 2, 5000 if heads * head_dim <= 4096 else 2000)
    sequences = min(tokens, _log(rng, 1, 16))
    return {"path": path, "sequences": sequences, "tokens": tokens, "step": False,
            "cached": rng.choice([0, min(room, sequences * _log(rng, 1, 2000))]), **layout}


# ------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _shares(total, sequences, rng):
    """`sequences` whole numbers that sum to `total`: log-normal sizes."""
    share = np.exp(0.7 * rng.normal(size=sequences))
    out = np.floor(share / share.sum() * total).astype(int)
    out[-1] += total - out.sum()
    return out


def _int(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _counts(case, seed):
    """New rows and cached tokens of each sequence; of prompts half are new and one is a single row."""
    rng = np.random.default_rng(seed)
    n, tokens = case["sequences"], case["tokens"]
    if case["path"] == "tree" or case["step"]:
        return np.full(n, tokens // n), _shares(case["cached"], n, rng)
    lengths = _shares(tokens, n, rng)
    cached = np.zeros(n, dtype=int)
    if n > 1:
        lengths[-1] += lengths[0] - min(1, lengths[0])
        lengths[0] = min(1, lengths[0])
    if case["cached"]:
        old = np.arange(n) >= n // 2
        cached[old] = _shares(case["cached"], int(old.sum()), rng)
    return lengths, cached


def _attention(case, seed):
    """The rows q | k | v as a projection leaves them, the pages (in no order) with the cached tokens, trees
    that branch as drafts do (a few long paths, the rest near the root), and each tree's accepted path."""
    g, rng = _generator(seed), np.random.default_rng(seed + 1)
    h, kv, d, page = (case[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    lengths, cached = _counts(case, seed)
    tokens, n = int(lengths.sum()), case["sequences"]
    rows = _randn(g, tokens, (h + 2 * kv) * d)
    rows[:, :h * d] *= 1.5 + torch.rand((tokens, 1), device="cuda", generator=g)  # some rows look at few tokens
    need = -(-(lengths + cached) // page)
    pages, width = (tokens + case["cached"]) // page + n + 3, int(need.max()) + 1  # a few are no sequence's
    order = rng.permutation(pages)
    table = np.zeros((n, width), dtype=np.int64)
    at = 0
    for i in range(n):
        table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
    kind = TYPES[case["cache"]]
    t = {"x": rows.to(TYPES[case["rows"]]), "lengths": lengths, "cached": cached,
         "keys": _randn(g, pages, kv, page, d).to(kind), "values": _randn(g, pages, kv, page, d).to(kind),
         "offsets": _int(np.concatenate([[0], np.cumsum(lengths)])), "context": _int(cached), "table": _int(table)}
    if case["path"] == "tree":
        parents = np.empty((n, tokens // n), dtype=int)
        for j in range(tokens // n):
            near = rng.random(n) < 0.4
            parents[:, j] = np.where(near, j - 1, rng.integers(-1, j, size=n) if j else -1)
        paths, accepted = np.zeros_like(parents), np.zeros(n, dtype=int)
        for i in range(n):
            node, path = int(rng.integers(0, tokens // n)), []
            while node >= 0:
                path.append(node)
                node = int(parents[i, node])
            accepted[i] = len(path)
            paths[i, :len(path)] = path[::-1]
        t |= {"parents": _int(parents.reshape(-1)), "paths": _int(paths), "accepted": _int(accepted)}
    return t


def _logits(case, seed):
    """Logits of an output head (N(0, 3) with some likely tokens); given tokens are likely ones and others."""
    g = _generator(seed)
    r, v = case["rows"], case["vocab"]
    logits = _randn(g, r, v)
    logits *= 3
    likely = torch.randint(0, v, (r, 20), device="cuda", generator=g)
    logits.scatter_add_(1, likely, 6 + _randn(g, r, 20))
    given = torch.where(torch.rand((r, case["given"]), device="cuda", generator=g) < 0.7, likely[:, :case["given"]],
                        torch.randint(0, v, (r, case["given"]), device="cuda", generator=g))
    return {"logits": logits, "given": given.int()}


_STREAM = []


def _stream():
    """The one stream that a program's passes follow each other on."""
    if not _STREAM:
        _STREAM.append(torch.cuda.Stream())
    return _STREAM[0].cuda_stream


def prepare(case, seed):
    if case["path"] == "score":
        state = _logits(case, seed)
        r = case["rows"]
        state |= {"log_probs": torch.empty((r, case["given"]), device="cuda"), "entropy": torch.empty(r, device="cuda"),
                  "top_tokens": torch.empty((r, case["top"]), dtype=torch.int32, device="cuda"),
                  "top_log_probs": torch.empty((r, case["top"]), device="cuda")}
        if own:
            from llambda_amd.sampling import HipTokenScorer
            state["scorer"] = HipTokenScorer(case["vocab"], r, max_top=case["top"])
    else:
        state = _attention(case, seed)
        tokens, (pages, _, page, _) = state["x"].shape[0], state["keys"].shape
        state["y"] = torch.empty((tokens, case["heads"] * case["head_dim"]), dtype=state["x"].dtype, device="cuda")
        if own:
            from llambda_amd.attention import AttentionLayout, HipAttentionSession
            layout = AttentionLayout(heads=case["heads"], kv_heads=case["kv_heads"], head_dim=case["head_dim"],
                                     row_type=case["rows"], cache_type=case["cache"])
            state["session"] = HipAttentionSession(
                layout, pages=pages, page_tokens=page, max_context=state["table"].shape[1] * page,
                max_tokens=tokens, max_sequences=case["sequences"], key_pages_ptr=state["keys"].data_ptr(),
                value_pages_ptr=state["values"].data_ptr())
    state["case"] = case
    state["stream"] = _stream()
    torch.cuda.synchronize()
    return state


def run(state):
    case = state["case"]
    if case["path"] == "score":
        return _score_own(state) if own else _score_plain(state)
    if own:
        _attend_own(state)
    else:
        _attend_plain(state)
    return {"y": state["y"], "keys": state["keys"], "values": state["values"]}


def _attend_own(s):
    c, x, session = s["case"], s["x"], s["session"]
    width, size = c["head_dim"], x.element_size()
    at, stride = x.data_ptr(), x.shape[1]
    tree = c["path"] == "tree"
    session.run_device(at, at + c["heads"] * width * size, at + (c["heads"] + c["kv_heads"]) * width * size,
                       s["y"].data_ptr(), x.shape[0], s["context"].data_ptr(), s["table"].data_ptr(), c["sequences"],
                       offsets_ptr=0 if not tree and c["step"] else s["offsets"].data_ptr(),
                       parents_ptr=s["parents"].data_ptr() if tree else 0,
                       q_stride=stride, k_stride=stride, v_stride=stride, stream=s["stream"])
    if tree:
        session.accept_device(s["context"].data_ptr(), s["table"].data_ptr(), s["paths"].data_ptr(),
                              s["accepted"].data_ptr(), c["sequences"], s["paths"].shape[1], stream=s["stream"])


def _score_own(s):
    c = s["case"]
    s["scorer"].score_device(s["logits"].data_ptr(), c["rows"], given_ptr=s["given"].data_ptr(), given=c["given"],
                             top=c["top"], log_probs_ptr=s["log_probs"].data_ptr(), entropy_ptr=s["entropy"].data_ptr(),
                             top_tokens_ptr=s["top_tokens"].data_ptr(), top_log_probs_ptr=s["top_log_probs"].data_ptr(),
                             stream=s["stream"])
    return {k: s[k] for k in ("log_probs", "entropy", "top_tokens", "top_log_probs")}


# ------------------------------------------------------------------ plain forms

def _attend_plain(s):
    """Sequences in lots of like length, padded; queries in blocks that keep the scores within 1 GB."""
    c, x, dev = s["case"], s["x"], s["x"].device
    h, kv, d, page, n = (c[k] for k in ("heads", "kv_heads", "head_dim", "page", "sequences"))
    g = h // kv
    context, table, offsets = s["context"].long(), s["table"].long(), s["offsets"].long()
    lengths = offsets[1:] - offsets[:-1]
    seq = torch.repeat_interleave(torch.arange(n, device=dev), lengths, output_size=x.shape[0])
    node = torch.arange(x.shape[0], device=dev) - offsets[seq]
    at = context[seq] + node
    where = table[seq, at // page], slice(None), at % page
    s["keys"][where] = x[:, h * d:(h + kv) * d].reshape(-1, kv, d).to(s["keys"].dtype)
    s["values"][where] = x[:, (h + kv) * d:].reshape(-1, kv, d).to(s["values"].dtype)
    q = x[:, :h * d].reshape(-1, kv, g, d)
    y = s["y"].reshape(-1, kv, g, d)
    tree = c["path"] == "tree"
    # trees and steps are padded together in lots, prompts are taken one by one
    lot = max(1, min(n, 600_000_000 // (kv * d * 8 * max(1, int((s["lengths"] + s["cached"]).max()))))) \
        if tree or c["step"] else 1
    for first in range(0, n, lot):
        i = torch.arange(first, min(n, first + lot), device=dev)
        long, rows = (int(v[first:first + lot].max()) for v in (s["lengths"] + s["cached"], s["lengths"]))
        if not rows:
            continue
        used = table[i, :-(-long // page)]
        k = s["keys"][used].transpose(1, 2).reshape(len(i), kv, -1, d)[:, :, :long].float()
        v = s["values"][used].transpose(1, 2).reshape(len(i), kv, -1, d)[:, :, :long].float()
        key = torch.arange(long, device=dev)
        total = (context + lengths)[i]
        v = torch.where((key < total[:, None])[:, None, :, None], v, 0.0)
        k = k.transpose(2, 3).contiguous()
        block = max(1, 250_000_000 // (len(i) * h * long))
        for r0 in range(0, rows, block):
            j = torch.arange(r0, min(rows, r0 + block), device=dev)
            row = torch.minimum(offsets[i][:, None] + j, torch.full_like(offsets[i + 1], x.shape[0] - 1)[:, None])
            real = j < lengths[i][:, None]
            if tree:
                sees = (key < context[i][:, None])[:, None].expand(-1, len(j), -1).clone()
                up = j.expand(len(i), -1).clone()
                for _ in range(rows):
                    sees |= (key == (context[i][:, None] + up)[..., None]) & (up >= 0)[..., None]
                    up = torch.where(up >= 0, s["parents"].long()[offsets[i][:, None] + up.clamp(min=0)], up)
            else:
                sees = key <= (context[i][:, None] + j)[..., None]                   # [b][rows][keys]
            qs = q[row].float().permute(0, 2, 1, 3, 4).reshape(len(i), kv, -1, d)    # [b][kv][rows * g][d]
            w = torch.matmul(qs, k) * (1 / math.sqrt(d))
            w = torch.where(sees.repeat_interleave(g, 1)[:, None], w, -math.inf)
            w = torch.exp(w - w.amax(-1, keepdim=True))
            w = w / w.sum(-1, keepdim=True)
            o = torch.matmul(w, v).reshape(len(i), kv, len(j), g, d).permute(0, 2, 1, 3, 4)
            y[row[real]] = o[real].to(y.dtype)
    if tree:
        j = torch.arange(s["paths"].shape[1], device=dev)
        keep = j < s["accepted"].long()[:, None]
        i = torch.arange(n, device=dev)[:, None].expand_as(keep)[keep]
        old, new = context[i] + s["paths"].long()[keep], context[i] + j.expand_as(keep)[keep]
        for pool in (s["keys"], s["values"]):
            pool[table[i, new // page], :, new % page] = pool[table[i, old // page], :, old % page]


def _score_plain(s):
    """Rows in blocks; sums over the vocabulary in 64 bits."""
    c = s["case"]
    outs = []
    for l in s["logits"].split(256):
        at = sum(o[1].shape[0] for o in outs)
        given = s["given"][at:at + l.shape[0]].long()
        x = l - l.amax(1, keepdim=True)
        e = torch.exp(x.double())
        total = e.sum(1, keepdim=True)
        lse = torch.log(total)
        entropy = (lse - (e * x).sum(1, keepdim=True) / total)[:, 0].float()
        value, index = torch.sort(l, dim=1, descending=True, stable=True) if c["top"] else (l, l.long())
        value, index = value[:, :c["top"]], index[:, :c["top"]].int()
        log = lambda v: (v.double() - lse - l.amax(1, keepdim=True).double()).float()  # noqa: E731
        outs.append((log(torch.gather(l, 1, given)), entropy, index, log(value)))
    return dict(zip(("log_probs", "entropy", "top_tokens", "top_log_probs"), (torch.cat(v) for v in zip(*outs))))


# ------------------------------------------------------------------ work

def work(case):
    if case["path"] == "score":
        r = case["rows"]
        return {"bytes": 4 * r * (case["vocab"] + 2 * case["given"] + 1 + 2 * case["top"]), "flops": 5 * r * case["vocab"]}
    h, kv, d = (case[k] for k in ("heads", "kv_heads", "head_dim"))
    row, cell = (4 if case[k] == "f32" else 2 for k in ("rows", "cache"))
    lengths, cached = _counts(case, 1)
    seen = lengths * cached
    # a tree's rows see their ancestors too: some of the rows before them, at least themselves
    seen = seen + (lengths if case["path"] == "tree" else lengths * (lengths + 1) // 2)
    tokens = int(lengths.sum())
    return {"bytes": tokens * d * (row * (2 * h + 2 * kv) + cell * 2 * kv)
            + cell * 2 * kv * d * int(cached[lengths > 0].sum()),
            "flops": 4 * d * h * int(seen.sum())}


# ------------------------------------------------------------------ outputs

def exact(case, seed):
    """What run() returns, in 64 bits; whole numbers and the pages, which hold roundings of inputs, have no such value."""
    return _exact_scores(case, seed) if case["path"] == "score" else \
        {"y": _exact_attention(case, seed), "keys": None, "values": None}


def _exact_scores(case, seed):
    s = _logits(case, seed)
    given, entropy, top = [], [], []
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        lp = torch.log_softmax(x, 0)
        given.append(lp[s["given"][r].long()])
        entropy.append(-(lp.exp() * lp).sum())
        top.append(torch.topk(lp, case["top"]).values)
    return {"log_probs": torch.stack(given), "entropy": torch.stack(entropy), "top_tokens": None,
            "top_log_probs": torch.stack(top)}


def _exact_attention(case, seed):
    """Sequence by sequence and head by head."""
    s = _attention(case, seed)
    h, kv, d, page = (case[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    out = torch.empty((s["x"].shape[0], h, d), dtype=torch.float64, device="cuda")
    kind, begin = TYPES[case["cache"]], 0
    for i, (n, c) in enumerate(zip(s["lengths"].tolist(), s["cached"].tolist())):
        if not n:
            continue
        x = s["x"][begin:begin + n]
        pages = [int(p) for p in s["table"][i, :-(-c // page)]]
        old = [torch.cat([pool[p].double() for p in pages], 1)[:, :c] if pages
               else torch.empty((kv, 0, d), dtype=torch.float64, device="cuda") for pool in (s["keys"], s["values"])]
        if case["path"] == "tree":
            chain = s["parents"][begin:begin + n].tolist()
            sees = torch.zeros((n, c + n), dtype=torch.bool)
            sees[:, :c] = True
            for r in range(n):
                if chain[r] >= 0:
                    sees[r] = sees[chain[r]]
                sees[r, c + r] = True
            sees = sees.cuda()
        for head in range(h):
            group = head // (h // kv)
            k, v = (torch.cat([pool[group], x[:, at:at + d].to(kind).double()])
                    for pool, at in zip(old, ((h + group) * d, (h + kv + group) * d)))
            for r in range(0, n, 4096):
                q = x[r:r + 4096, head * d:(head + 1) * d].double()
                w = q @ k.T / math.sqrt(d)
                if case["path"] == "tree":
                    w.masked_fill_(~sees[r:r + 4096], -math.inf)
                else:
                    reach = c + r + torch.arange(q.shape[0], device="cuda")
                    w.masked_fill_(torch.arange(c + n, device="cuda") > reach[:, None], -math.inf)
                out[begin + r:begin + r + q.shape[0], head] = torch.softmax(w, 1) @ v
        begin += n
    return out.reshape(-1, h * d)
