"""GPU tests of results that share memory with arguments: refused in front of any launch, where CTAs would read what others have written."""
import numpy as np
import pytest

from tests import drafts_model
from tests.test_gpu_drafts import batch, ints, on_device, outputs

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_results_of_a_verification_over_the_rows(tq, dtype):
    """Over the target's or the draft's rows: refused.  Between rows that are apart, or behind the last: as anywhere."""
    rng = np.random.default_rng(1)
    counts, vocab, pad = [5, 6], 40, 16
    parents, tokens, target, draft, u = batch(rng, counts, vocab, 2, True, dtype)
    args = ints([0, 5, 11]), ints(np.concatenate(parents)), ints(tokens)
    uniforms, es = torch.from_numpy(u).cuda(), np.dtype(dtype).itemsize
    want = [drafts_model.verify(parents[i], tokens[r], target[r], draft[r], u[r], 2) for i, r in enumerate((slice(0, 5), slice(5, 11)))]
    for which in (0, 1):
        rows = [on_device(x, pad) for x in (target, draft)]
        numbers = rows[which].as_strided((11 * (vocab + pad),), (1,)).view(torch.int32)
        row = (vocab + pad) * es // 4      # of whole numbers
        for change in ({"next": numbers[:2]}, {"kept": numbers[vocab * es // 4 - 1:][:2]}, {"path": numbers[10 * row:][:4].view(2, 2)}, {"path": numbers[row - 3:][:4].view(2, 2)},
                       {"next": numbers[4 * row - 1:][:2]}, {"kept": numbers[10 * row + 1:][:2]}):
            with pytest.raises(tq.TQError, match="must not be where"):
                tq.verify_drafts(*args, *rows, uniforms, **{**outputs(2, 2), **change})
        gap = numbers[3 * row + vocab * es // 4:][:pad * es // 4]
        out = {"path": gap[:4].view(2, 2), "kept": gap[4:6], "next": gap[6:8]}
        tq.verify_drafts(*args, *rows, uniforms, **out)
        assert out["next"].tolist() == [t for _, t in want] and out["path"].tolist() == [p + [-1] * (2 - len(p)) for p, _ in want]
        assert torch.equal(rows[which].cpu(), torch.from_numpy((target, draft)[which]))


def test_results_of_norms_over_their_arguments(tq):
    rows, heads, kv, dim = 33, 4, 2, 64
    step = (heads + 2 * kv) * dim
    block = torch.randn((rows + 1, step), device="cuda").half()
    flat, before = block.view(-1), block.clone()
    slot = lambda at, n, stride=step: flat[at:].as_strided((rows, n, dim), (stride, dim, 1))      # noqa: E731
    q, k = slot(0, heads), slot(heads * dim, kv)
    w, positions = torch.ones((2, dim), device="cuda").half(), torch.arange(rows, dtype=torch.int32, device="cuda")
    apart = lambda n: torch.empty((rows, n, dim), dtype=torch.float16, device="cuda")      # noqa: E731
    many = torch.zeros(rows * heads * dim + 8, dtype=torch.float16, device="cuda")
    inside = many.view(torch.int32)[3:3 + rows]
    cases = [((slot(0, heads, heads * dim), apart(kv)), {}), ((slot(step, heads), apart(kv)), {}),       # packed in place; a row further
             ((slot(dim, heads), apart(kv)), {}), ((slot(heads * dim, heads), apart(kv)), {}),           # a head further; over the keys
             ((apart(heads), slot(0, kv)), {}), ((apart(heads), slot(heads * dim - dim, kv)), {}),       # the keys' over the queries, wholly and by a head
             ((slot((heads + kv) * dim - dim, kv + 1), apart(kv)), {"queries": apart(kv + 1)}),
             ((slot(0, heads), slot(2 * dim, kv)), {}),
             ((many[:rows * heads * dim].view(rows, heads, dim), apart(kv)), {"positions": inside}),
             ((many[:rows * heads * dim].view(rows, heads, dim), apart(kv)), {"query_weight": many[100 * 8:][:dim]}),
             ((apart(heads), many[:rows * kv * dim].view(rows, kv, dim)), {"key_weight": many[:dim]}),
             ((many[:rows * heads * dim].view(rows, heads, dim), many[8:8 + rows * kv * dim].view(rows, kv, dim)), {})]
    for out, change in cases:
        args = {"queries": q, "keys": k, "query_weight": w[0], "key_weight": w[1], "positions": positions, **change}
        with pytest.raises(tq.TQError, match="must (not )?be"):
            tq.qk_norm_rope(**args, out=out)
    assert torch.equal(block, before)
    want = tq.qk_norm_rope(q, k, *w, positions, out=(apart(heads), apart(kv)))
    # another slot of the same rows, then in place
    tq.qk_norm_rope(q, k, *w, positions, out=(apart(heads), slot((heads + kv) * dim, kv)))
    assert torch.equal(slot((heads + kv) * dim, kv), want[1])
    tq.qk_norm_rope(q, k, *w, positions)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    # one row has no stride
    q1, k1 = slot(0, heads)[:1].clone(), slot(heads * dim, kv)[:1].clone()
    want = tq.qk_norm_rope(q1, k1, *w, positions[:1], out=(torch.empty_like(q1), torch.empty_like(k1)))
    tq.qk_norm_rope(q1, k1, *w, positions[:1], out=(q1.as_strided((1, heads, dim), (5 * step, dim, 1)), k1))
    assert torch.equal(q1, want[0]) and torch.equal(k1, want[1])


def test_positions_over_parents(tq):
    """At the same address: in their place.  Shifted: refused, since a request's would lie over another one's parents."""
    c = tq.PagedKVCache(1, 1, 64, 40, 16, 20, 4, 256)
    c.plan(np.array([3, 0, 9], np.int32))
    c.plan(np.array([5] * 20, np.int32))
    block = ints([0] * 4 + [-1, 0, 0, 1, 3] * 20 + [0] * 4)
    for at in (0, 1, 3, 5, 8):
        with pytest.raises(tq.TQError, match="must not be where"):
            c.tree(block[4:104], positions=block[at:at + 100])
    positions = torch.zeros(100, dtype=torch.int32, device="cuda")
    c.tree(block[4:104], positions=positions)
    c.tree(block[4:104], positions=block[4:104])
    want = [held + d for held in [3, 0, 9] + [0] * 17 for d in (0, 1, 1, 2, 3)]
    assert positions.tolist() == want and block.tolist() == [0] * 4 + want + [0] * 4
    torch.cuda.synchronize()
    c.check_status()
    c.close()


@pytest.mark.parametrize("counts", [[2, 1, 4], [40, 3, 70]])
def test_results_of_attention_over_the_queries(tq, counts):
    """In place, as chains through both calls: few rows, many, and both in a batch over a context that several CTAs share."""
    c = tq.PagedKVCache(1, 2, 64, 120, 64, 3, 60, 4096)
    x = torch.randn((3500, 2, 64), device="cuda").half()
    c.plan(np.array([3000, 0, 500], np.int32))
    c.append(0, x, x)
    tokens, heads = sum(counts), 6
    c.plan(np.array(counts, np.int32))
    c.tree()
    c.append(0, x[:tokens], x[:tokens])
    step = heads * 64 + 2 * 64
    block = torch.randn((tokens + 1) * step, device="cuda").half()
    slot = lambda at=0, stride=step: block[at:].as_strided((tokens, heads, 64), (stride, 64, 1))      # noqa: E731
    before, numbers = block.clone(), block.view(torch.float32)
    for call in (c.attention, c.tree_attention):
        for out in (slot(stride=heads * 64), slot(step), slot(64), slot(2 * 64)):
            with pytest.raises(tq.TQError, match="must be where"):
                call(0, slot(), out=out)
        apart = torch.empty((tokens, heads, 64), dtype=torch.float16, device="cuda")
        for out, lse in ((apart, numbers[:tokens * heads]), (apart, apart.view(-1).view(torch.float32)[:tokens * heads])):
            with pytest.raises(tq.TQError, match="lse must not be"):
                call(0, slot(), out=out, lse=lse.view(tokens, heads))
        assert torch.equal(block, before)
        call(0, slot(), out=apart)
        call(0, slot(), out=slot())
        assert torch.equal(slot(), apart)
        block.copy_(before)
    torch.cuda.synchronize()
    c.check_status()
    c.close()
