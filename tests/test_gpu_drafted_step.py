"""A drafted decoding step as a server makes it, all of it in one captured graph: plan, tree, and in each layer the norms of heads with their rotation,
append and attention of the trees; verification, and the branch that stays.  Every operator's results against its definition on what it was given."""
import numpy as np
import pytest

from tests import drafts_model, tree_attention_model
from tests.paged_model import Model
from tests.test_gpu_drafts import ints
from tests.test_gpu_paged_attention import compare

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


class Decoder:
    """Two layers of attention with random weights, and buffers for up to `most` nodes of each of n requests."""

    def __init__(self, tq, rng, n, most, heads, group, dim, page, pages, vocab, drawn, layers=2):
        self.n, self.most, self.heads, self.group, self.dim, self.layers, self.drawn = n, most, heads, group, dim, layers, drawn
        rows, hidden = n * most, heads * group * dim
        weight = lambda *shape: torch.from_numpy((rng.standard_normal(shape) / np.sqrt(shape[0])).astype(np.float16)).cuda()      # noqa: E731
        self.tq, self.c = tq, tq.PagedKVCache(layers, heads, dim, pages, page, n, pages, rows)
        self.m = [Model(heads, dim, pages, page) for _ in range(layers)]
        self.qkv = [weight(hidden, (group + 2) * heads * dim) for _ in range(layers)]
        self.norms = [[(1 + weight(1, dim)[0]).contiguous() for _ in range(2)] for _ in range(layers)]
        self.head = weight(hidden, vocab)
        whole = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")      # noqa: E731
        self.counts, self.parents, self.tokens, self.positions = whole(n), whole(rows), whole(rows), whole(rows)
        self.starts, self.path, self.kept, self.next, self.lengths = whole(n + 1), whole(n, most), whole(n), whole(n), whole(n)
        self.x = torch.zeros((rows, hidden), dtype=torch.float16, device="cuda")
        self.draft, self.uniforms = torch.zeros((rows, vocab), device="cuda"), torch.zeros(rows, device="cuda")
        self.target = torch.zeros((rows, vocab), device="cuda")
        self.raw = [torch.zeros((rows, (group + 2) * heads, dim), dtype=torch.float16, device="cuda") for _ in range(layers)]
        self.mixed = [torch.zeros_like(r) for r in self.raw]
        self.out = [torch.zeros((rows, heads * group, dim), dtype=torch.float16, device="cuda") for _ in range(layers)]
        self.lse = [torch.zeros((rows, heads * group), device="cuda") for _ in range(layers)]

    def split(self, x):
        q = self.heads * self.group
        return x[:, :q], x[:, q:q + self.heads], x[:, q + self.heads:]

    def step(self, stream):
        self.c.plan(self.counts, self.n * self.most, self.most, starts=self.starts, stream=stream)
        self.c.tree(self.parents, positions=self.positions, stream=stream)
        x = self.x
        for i in range(self.layers):
            self.raw[i].copy_((x @ self.qkv[i]).view(self.raw[i].shape))
            self.mixed[i].copy_(self.raw[i])
            q, k, v = self.split(self.mixed[i])
            self.tq.qk_norm_rope(q, k, *self.norms[i], self.positions, theta=1e4, stream=stream)
            self.c.append(i, k, v, stream=stream)
            self.c.tree_attention(i, q, out=self.out[i], lse=self.lse[i], stream=stream)
            x = self.out[i].view(x.shape)
        self.target.copy_(torch.softmax(3 * (x @ self.head).float(), 1))
        self.tq.verify_drafts(self.starts, self.parents, self.tokens, self.target, self.draft if self.drawn else None, self.uniforms, self.path, self.kept, self.next,
                              stream=stream)
        self.c.keep(self.path, self.kept, lengths=self.lengths, stream=stream)

    def inputs(self, rng, counts, spread):
        vocab = self.draft.shape[1]
        self.trees = drafts_model.trees(rng, counts, spread)
        draft = np.exp(rng.standard_normal(self.draft.shape))
        draft = (draft / draft.sum(1, keepdims=True)).astype(np.float32)
        tokens, at = rng.integers(0, vocab, len(draft)), 0
        for par in self.trees:
            for j, p in enumerate(par):
                if p >= 0:
                    q = draft[at + p].astype(np.float64)
                    tokens[at + j] = rng.choice(vocab, p=q / q.sum())
            at += len(par)
        self.counts.copy_(ints(counts))
        self.parents.fill_(-9)
        self.parents[:at] = ints([p for par in self.trees for p in par])
        self.tokens.copy_(ints(tokens))
        self.draft.copy_(torch.from_numpy(draft))
        self.uniforms.copy_(torch.from_numpy(rng.random(len(draft)).astype(np.float32)))
        self.x.copy_(torch.from_numpy(rng.standard_normal(self.x.shape).astype(np.float16)))

    def check(self, counts):
        """What the last step did; tokens that it kept beside each request's first."""
        self.c.check_status()
        total, n = sum(counts), self.n
        held = [self.m[0].lengths.get(i, 0) for i in range(n)]
        positions = [h + d for h, par in zip(held, self.trees) for d in drafts_model.depths(par)]
        assert self.positions.tolist() == positions + [0] * (n * self.most - total)
        for i, m in enumerate(self.m):
            m.plan(counts)
            raw, mixed = self.raw[i][:total].cpu().numpy(), self.mixed[i][:total].cpu().numpy()
            for which, (x, y) in enumerate(zip(self.split(raw), self.split(mixed))):
                if which < 2:
                    want, tol = drafts_model.qk_norm_rope(x, self.norms[i][which].cpu().numpy(), positions, 1e4, 1e-6)
                    assert (np.abs(y.astype(np.float64) - want) <= tol).all()
                else:
                    assert np.array_equal(x, y)
            q, k, v = self.split(mixed)
            m.append(0, k)
            m.append(1, v)
            compare(self.out[i][:total], self.lse[i][:total], tree_attention_model.attention(m, q, self.trees))
            assert (self.lse[i][total:] == -5).all()          # rows behind the last request, left as they were
        target, draft, tokens, u = (t.cpu().numpy() for t in (self.target, self.draft, self.tokens, self.uniforms))
        paths, following = [], []
        at = np.concatenate([[0], np.cumsum(counts)])
        for i, par in enumerate(self.trees):
            rows = slice(at[i], at[i + 1])
            path, token = drafts_model.verify(par, tokens[rows], target[rows], draft[rows] if self.drawn else None, u[rows], self.most)
            paths.append(path)
            following.append(token)
        assert self.starts.tolist() == at.tolist() and self.kept.tolist() == [len(p) for p in paths] and self.next.tolist() == following
        assert self.path.tolist() == [p + [-1] * (self.most - len(p)) for p in paths]
        want = drafts_model.kept_lengths(self.m[0], paths)
        for m in self.m:
            for which in (0, 1):
                drafts_model.keep(m, which, paths)
            m.truncate(want)
        assert self.lengths.tolist() == want and self.c.free_pages() == len(self.m[0].stack)
        return sum(max(0, len(p) - 1) for p in paths)


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("heads,group,dim,page", [(2, 3, 64, 16), (1, 7, 128, 64)])
def test_steps_of_a_captured_graph(tq, drawn, heads, group, dim, page):
    rng = np.random.default_rng(dim + drawn)
    d = Decoder(tq, rng, 5, 14, heads, group, dim, page, 60, 50, drawn)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        d.step(side)        # (no tokens)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            d.step(side)
    torch.cuda.synchronize()
    more = 0
    for counts, spread in (([14, 9, 0, 1, 14], 1), ([3, 14, 5, 0, 14], 3), ([14, 14, 14, 14, 14], 20), ([0, 0, 0, 0, 0], 1), ([1, 1, 1, 1, 1], 1), ([8, 14, 2, 14, 11], 2)):
        d.inputs(rng, counts, spread)
        for lse in d.lse:
            lse.fill_(-5)
        graph.replay()
        torch.cuda.synchronize()
        more += d.check(counts)
    assert more > 0
    d.c.close()
