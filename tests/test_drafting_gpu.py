"""Attention and token scores as a server uses them: prompts with the scores of their tokens, trees of drafted
tokens, the path of the likeliest kept, then steps from one graph.  Each stage against 64 bits of what it was given."""
import numpy as np
import pytest

import attention_reference as ref
from llambda_amd.attention import AttentionLayout, HipAttentionSession
from llambda_amd.sampling import HipTokenScorer
from test_token_scores_gpu import reference

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, VOCAB, PAGE, LAYERS = 6, 2, 64, 5003, 32, 2
SIZES = [HEADS * DIM, KV * DIM, KV * DIM]


class Server:
    """A cache of 64-bit-checked sequences: `kept[layer][i]` are the keys and values that sequence i has to hold."""

    def __init__(self, kinds, sequences, max_tokens):
        import torch
        self.kinds, self.n = kinds, sequences
        self.type = {"f32": torch.float32, "bf16": torch.bfloat16}[kinds[0]]
        self.rng = np.random.default_rng(31)
        width = 12
        self.session = HipAttentionSession(
            AttentionLayout(HEADS, KV, DIM, row_type=kinds[0], cache_type=kinds[1]), pages=width * sequences + 2,
            page_tokens=PAGE, max_context=width * PAGE, max_tokens=max_tokens, max_sequences=sequences, layers=LAYERS)
        self.table = self.rng.permutation(width * sequences).reshape(sequences, width).astype(np.int32)
        self.d_table = torch.from_numpy(self.table).cuda()
        self.kept = [[np.empty((2, 0, KV, DIM), np.float32) for _ in range(sequences)] for _ in range(LAYERS)]
        self.context = torch.zeros(sequences, dtype=torch.int32, device="cuda")
        self.weights = torch.from_numpy(self.rng.normal(size=(HEADS * DIM, VOCAB)).astype(np.float32) / 4).cuda()
        self.scorer = HipTokenScorer(VOCAB, max_tokens, 8)
        self.stream = torch.cuda.Stream()

    def buffers(self, tokens):
        """q, k, v and the output of all layers, side by side, and what is scored."""
        import torch
        rows = [torch.empty((tokens, sum(SIZES) + SIZES[0]), dtype=self.type, device="cuda") for _ in range(LAYERS)]
        self.fill(rows)
        empty = lambda *s, t=torch.float32: torch.empty(s, dtype=t, device="cuda")  # noqa: E731
        return rows, [empty(tokens, VOCAB), empty(tokens, 1), empty(tokens), empty(tokens, 8, t=torch.int32),
                      empty(tokens, 8)]

    def fill(self, rows):
        import torch
        for r in rows:
            r.copy_(torch.from_numpy(self.rng.normal(size=tuple(r.shape)).astype(np.float32)))

    def run(self, rows, scored, given, offsets=None, parents=None):
        """On self.stream: every layer's attention, a head on the last one's output, its scores."""
        import torch
        tokens, width = rows[0].shape
        size = rows[0].element_size()
        at = [0, *np.cumsum(SIZES).tolist()]
        for layer, r in enumerate(rows):
            q, k, v, y = (r.data_ptr() + a * size for a in at)
            self.session.run_device(q, k, v, y, tokens, self.context.data_ptr(), self.d_table.data_ptr(), self.n,
                                    offsets_ptr=0 if offsets is None else offsets.data_ptr(),
                                    parents_ptr=0 if parents is None else parents.data_ptr(), layer=layer,
                                    q_stride=width, k_stride=width, v_stride=width, output_stride=width,
                                    stream=self.stream.cuda_stream)
        logits, log_probs, entropy, top, top_log_probs = scored
        with torch.cuda.stream(self.stream):
            torch.matmul(rows[-1][:, at[3]:].float(), self.weights, out=logits)
        self.scorer.score_device(logits.data_ptr(), tokens, given_ptr=given.data_ptr(), given=1, top=8,
                                 log_probs_ptr=log_probs.data_ptr(), entropy_ptr=entropy.data_ptr(),
                                 top_tokens_ptr=top.data_ptr(), top_log_probs_ptr=top_log_probs.data_ptr(),
                                 stream=self.stream.cuda_stream)

    def check(self, rows, scored, given, lengths, trees=None):
        """Everything that run left; the new keys and values join those kept."""
        self.session.sync(self.stream.cuda_stream)
        row, cell = self.kinds
        cuts = np.cumsum(SIZES)
        for layer, r in enumerate(rows):
            q, k, v, y = (a.reshape(len(r), -1, DIM) for a in np.split(r.float().cpu().numpy(), cuts, axis=1))
            begin = 0
            for i, n in enumerate(lengths):
                mine = slice(begin, begin + n)
                begin += n
                have = self.kept[layer][i]
                context = have.shape[1]
                have = np.concatenate([have, ref.rounded(np.stack([k[mine], v[mine]]), cell)], axis=1)
                self.kept[layer][i] = have
                want, bound = ref.attention(q[mine], *have, ref.sees(n, context, None if trees is None else trees[i]),
                                            np.float32(1 / np.sqrt(DIM)), row, cell)
                assert np.all(np.abs(y[mine] - want) <= bound)
        logits, log_probs, entropy, top, top_log_probs = (t.cpu().numpy() for t in scored)
        y, w = (a.astype(np.float64) for a in (rows[-1].float().cpu().numpy()[:, cuts[-1]:], self.weights.cpu().numpy()))
        assert np.all(np.abs(logits - y @ w) <= (len(w) + 2) * 2.0 ** -24 * (np.abs(y) @ np.abs(w)))
        for i, (x, g) in enumerate(zip(logits, given.cpu().numpy().reshape(-1))):
            lp, h, order, log_bound, h_bound = reference(x, 8)
            assert abs(entropy[i] - h) <= h_bound and top[i].tolist() == order.tolist()
            for got, w in ((log_probs[i, 0], lp[g]), (top_log_probs[i], lp[order])):
                assert np.all(np.abs(got - w) <= log_bound + np.abs(w) * 2.0 ** -24)

    def check_cache(self):
        for layer in range(LAYERS):
            for i, have in enumerate(self.kept[layer]):
                for got, want in zip(self.session.read(self.table[i], 0, have.shape[1], layer=layer), have):
                    assert np.array_equal(ref.loaded(got, self.kinds[1]), want)


@pytest.mark.parametrize("kinds", [("f32", "f16"), ("bf16", "bf16"), ("f32", "f32")], ids="-".join)
def test_prompts_trees_accepted_paths_and_steps(hip, kinds):
    import torch
    lengths = [37, 1, 150]
    s = Server(kinds, len(lengths), sum(lengths))
    rng = s.rng

    def on_device(a):
        return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")

    def offsets(n):
        return on_device(np.concatenate([[0], np.cumsum(n)]))

    # prompts
    rows, scored = s.buffers(sum(lengths))
    given, ends = on_device(rng.integers(0, VOCAB, size=sum(lengths))), offsets(lengths)
    torch.cuda.synchronize()
    s.run(rows, scored, given, ends)
    s.check(rows, scored, given, lengths)
    for _ in range(2):  # drafts
        s.context.copy_(on_device([have.shape[1] for have in s.kept[0]]))
        trees = [[-1] + [int(rng.integers(max(-1, j - 3), j)) for j in range(1, n)] for n in (19, 7, 33)]
        sizes = [len(t) for t in trees]
        rows, scored = s.buffers(sum(sizes))
        drafted = rng.integers(0, VOCAB, size=sum(sizes))
        given, ends = on_device(drafted), offsets(sizes)
        parents = on_device(np.concatenate(trees))
        torch.cuda.synchronize()
        s.run(rows, scored, given, ends, parents)
        s.check(rows, scored, given, sizes, trees)
        # from each node on to the likeliest of its children's tokens
        logits = scored[0].cpu().numpy()
        paths, begin = [], 0
        for tree in trees:
            path, node = [], -1
            while True:
                children = [j for j, parent in enumerate(tree) if parent == node]
                if not children:
                    break
                node = max(children, key=lambda j: logits[begin + max(node, 0), drafted[begin + j]])
                path.append(node)
            paths.append(path)
            begin += len(tree)
        held = np.zeros((len(trees), 40), np.int32)
        for i, path in enumerate(paths):
            held[i, :len(path)] = path
        d_paths, counts = on_device(held), on_device([len(path) for path in paths])
        torch.cuda.synchronize()
        s.session.accept_device(s.context.data_ptr(), s.d_table.data_ptr(), d_paths.data_ptr(), counts.data_ptr(),
                                len(trees), 40, stream=s.stream.cuda_stream)
        s.session.sync(s.stream.cuda_stream)
        for layer in s.kept:
            for i, (path, n) in enumerate(zip(paths, sizes)):
                old = layer[i].shape[1] - n
                layer[i] = layer[i][:, list(range(old)) + [old + j for j in path]]
        s.check_cache()
    # steps, from one graph
    n = len(lengths)
    rows, scored = s.buffers(n)
    given = on_device(rng.integers(0, VOCAB, size=n))
    for step in range(4):
        s.context.copy_(on_device([have.shape[1] for have in s.kept[0]]))
        s.fill(rows)
        given.copy_(on_device(rng.integers(0, VOCAB, size=n)))
        torch.cuda.synchronize()
        if step == 0:
            s.run(rows, scored, given)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s.stream, capture_error_mode="relaxed"):
                s.run(rows, scored, given)
        else:
            with torch.cuda.stream(s.stream):
                graph.replay()
        torch.cuda.synchronize()
        s.check(rows, scored, given, [1] * n)
    s.check_cache()
