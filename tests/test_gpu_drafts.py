"""GPU tests of a drafted decoding step's calls without a cache: norms of heads with their rotation, and the verification of drafts."""
import numpy as np
import pytest

from tests import drafts_model

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def slices(x, pad, shift):
    """x [tokens, heads, dim] with `pad` elements behind each token's heads, `shift` elements from an aligned address."""
    n, h, d = x.shape
    room = torch.full((shift + n * (h * d + pad) + 8,), 7.0, dtype=x.dtype, device="cuda")
    view = room[shift:].as_strided((n, h, d), (h * d + pad, d, 1))
    view.copy_(x)
    return room, view


def check_rope(tq, rng, rows, heads, kv, dim, positions, theta=1e4, eps=1e-6, pad=0, shift=0, in_place=False, gain=1.0):
    xs = [(gain * rng.standard_normal((rows, h, dim)) * np.exp(rng.standard_normal((rows, h, 1)))).astype(np.float16) for h in (heads, kv)]
    ws = [(1 + 0.3 * rng.standard_normal(dim)).astype(np.float16) for _ in range(2)]
    rooms, views = zip(*(slices(torch.from_numpy(x).cuda(), pad, shift) for x in xs))
    wd = [torch.from_numpy(w).cuda() for w in ws]
    outs, to = (rooms, views) if in_place else zip(*(slices(torch.full_like(v, 3.0), pad, shift) for v in views))
    got = tq.qk_norm_rope(*views, *wd, ints(positions), theta=theta, eps=eps, out=None if in_place else to)
    torch.cuda.synchronize()
    for g, room, x, w in zip(got, outs, xs, ws):
        want, tol = drafts_model.qk_norm_rope(x, w, positions, theta, eps)
        g, fine = g.cpu().numpy().astype(np.float64), ~np.isnan(want)        # (an infinity in a head: it and its pair are not numbers)
        assert np.array_equal(np.isnan(g), ~fine)
        worst = np.max(np.abs(g - want)[fine] / tol[fine])
        assert worst <= 1, f"off by {worst} times the bound"
        n, h, d = x.shape      # what lies between the rows is as it was
        rest = torch.cat([room[:shift], room[shift:].as_strided((n, pad), (h * d + pad, 1), shift + h * d).flatten(), room[shift + n * (h * d + pad):]])
        assert (rest == 7.0).all()


@pytest.mark.parametrize("dim", [16, 48, 64, 80, 128, 256, 512])
@pytest.mark.parametrize("heads,kv", [(1, 1), (28, 4), (3, 5), (40, 8)])
@pytest.mark.parametrize("rows,pad,shift", [(1, 0, 0), (7, 8, 0), (33, 3, 1), (5, 0, 4)])
def test_norms_and_rotation(tq, dim, heads, kv, rows, pad, shift):
    rng = np.random.default_rng(dim + heads + rows)
    check_rope(tq, rng, rows, heads, kv, dim, rng.integers(0, 4096, rows), pad=pad, shift=shift, in_place=rows == 7)


@pytest.mark.parametrize("theta", [10.0, 1e4, 1e6, 5e8])
def test_far_and_negative_positions(tq, theta):
    rng = np.random.default_rng(1)
    # (a double of position times frequency has 2^-22 turns left at 2^31; half of that and the rest are in the bound's place up to 2^24)
    check_rope(tq, rng, 12, 4, 2, 128, [0, 1, -1, 131071, 131072, -131072, 1 << 20, (1 << 20) + 1, 1 << 24, -(1 << 24), 12345677, 3], theta=theta)


@pytest.mark.parametrize("gain,eps", [(0.0, 1e-6), (1e-4, 0.0), (1e-4, 1e-2), (2000.0, 1e-6)])
def test_small_and_large_heads(tq, gain, eps):
    rng = np.random.default_rng(2)
    check_rope(tq, rng, 9, 4, 1, 64, np.arange(9), eps=eps, gain=gain)


def test_many_rows(tq):
    rng = np.random.default_rng(3)
    check_rope(tq, rng, 3001, 8, 2, 64, rng.integers(0, 1 << 17, 3001))


def test_heads_that_are_not_numbers(tq):
    x = torch.randn((3, 4, 64), device="cuda").half()
    x[0, 1, 3], x[2, 0, 63] = float("nan"), float("inf")
    k, w = torch.randn((3, 1, 64), device="cuda").half(), torch.ones(64, device="cuda").half()
    q, _ = tq.qk_norm_rope(x, k, w, w, ints([5, 6, 7]), out=(torch.empty_like(x), torch.empty_like(k)))
    lost = torch.isnan(q).any(2)
    assert lost[0].tolist() == [False, True, False, False] and lost[2].tolist() == [True, False, False, False] and not lost[1].any()


def test_heads_of_zeros_without_eps_are_not_numbers(tq):
    """0 / sqrt(0): as the formula has it."""
    x, w = torch.zeros((1, 1, 64), device="cuda").half(), torch.ones(64, device="cuda").half()
    q, k = tq.qk_norm_rope(x, x.clone(), w, w, ints([5]), eps=0.0, out=(torch.zeros_like(x), torch.zeros_like(x)))
    assert torch.isnan(q).all() and torch.isnan(k).all()


# ---- verification -------------------------------------------------------------------------------------------------------

def softmaxes(rng, rows, vocab, sharp):
    x = sharp * rng.standard_normal((rows, vocab))
    p = np.exp(x - x.max(1, keepdims=True)) if rows else x
    return x, p / p.sum(1, keepdims=True) if rows else x


def batch(rng, counts, vocab, spread, drawn, dtype=np.float32, sharp=2.0, pad=0):
    """Parents, tokens, target, draft, uniforms of all rows."""
    parents = drafts_model.trees(rng, counts, spread)
    rows = sum(counts) + pad
    x, target = softmaxes(rng, rows, vocab, sharp)
    _, noise = softmaxes(rng, rows, vocab, 0.5)
    draft = target * noise
    draft = (draft / draft.sum(1, keepdims=True)).astype(dtype) if rows else draft.astype(dtype)
    tokens, at = rng.integers(0, vocab, rows), 0
    for par in parents:
        for j, p in enumerate(par):
            if p >= 0:
                q = draft[at + p].astype(np.float64)
                tokens[at + j] = rng.choice(vocab, p=q / q.sum()) if drawn else np.argsort(-q, kind="stable")[sum(o == p for o in par[:j]) % vocab]
        at += len(par)
    return parents, tokens.astype(np.int32), target.astype(dtype), draft if drawn else None, rng.random(rows).astype(np.float32)


def on_device(x, pad=0, shift=0):
    """Rows `pad` elements apart, `shift` elements from an aligned address; behind them numbers that would win."""
    if x is None:
        return None
    rows, vocab = x.shape
    room = torch.full((shift + rows * (vocab + pad) + 8,), 9.0, device="cuda", dtype=torch.float32 if x.dtype == np.float32 else torch.float16)
    view = room[shift:].as_strided((rows, vocab), (vocab + pad, 1))
    view.copy_(torch.from_numpy(x))
    return view


def outputs(n, width):
    return {"path": torch.full((n, width), 77, dtype=torch.int32, device="cuda"), "kept": torch.full((n,), 77, dtype=torch.int32, device="cuda"),
            "next": torch.full((n,), 77, dtype=torch.int32, device="cuda")}


def check_verify(tq, counts, width, parents, tokens, target, draft, u, pad=0, shift=0):
    starts = np.concatenate([[0], np.cumsum(counts)])
    out = outputs(len(counts), width)
    flat = np.concatenate([np.asarray(p, np.int32) for p in parents] + [np.full(len(tokens) - starts[-1], -1, np.int32)])
    tq.verify_drafts(ints(starts), ints(flat), ints(tokens), on_device(target, pad, shift), on_device(draft, pad, shift), torch.from_numpy(u).cuda(), **out)
    torch.cuda.synchronize()
    got = {k: v.cpu().numpy() for k, v in out.items()}
    kept = []
    for i, c in enumerate(counts):
        rows = slice(starts[i], starts[i] + c)
        path, token = drafts_model.verify(parents[i], tokens[rows], target[rows], None if draft is None else draft[rows], u[rows], width)
        assert got["kept"][i] == len(path) and got["path"][i].tolist() == path + [-1] * (width - len(path)) and got["next"][i] == token, f"request {i}"
        kept.append(len(path))
    return kept


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("vocab,pad,shift", [(1, 0, 0), (2, 0, 0), (7, 1, 1), (128, 0, 0), (1000, 0, 0), (1001, 0, 0), (5003, 5, 3), (32000, 0, 0), (50257, 0, 0)])
def test_verification(tq, drawn, dtype, vocab, pad, shift):
    rng = np.random.default_rng(vocab)
    counts = [1, 2, 9, 0, 16, 5, 8] if vocab > 2000 else [1, 2, 9, 0, 16, 5, 33, 8, 60, 4, 4, 4, 4]
    for spread in (1, 4):
        check_verify(tq, counts, 6, *batch(rng, counts, vocab, spread, drawn, dtype, pad=3), pad=pad, shift=shift)


@pytest.mark.parametrize("drawn", [True, False])
def test_long_chains_and_the_path_s_width(tq, drawn):
    """Drafts that are all accepted (the target's and the draft's rows are points): the path ends at its width, or at the 1024th node."""
    rng = np.random.default_rng(0)
    vocab = 50
    counts = [1500, 3, 40]
    parents, tokens, target, draft, u = batch(rng, counts, vocab, 1, drawn)
    target[:] = 0
    at = 0
    for c in counts:
        for j in range(c):
            target[at + j, tokens[at + j + 1] if j + 1 < c else 3] = 1
        at += c
    draft = target.copy() if drawn else None
    for width in (1, 2, 39, 40, 41, 2000):
        kept = check_verify(tq, counts, width, parents, tokens, target, draft, u)
        assert kept == [min(c, width, 1024) for c in counts]


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 1.0, np.nan, -0.5])
def test_random_numbers_at_their_ends(tq, drawn, u):
    rng = np.random.default_rng(4)
    counts, vocab = [5, 9, 3], 300
    parents, tokens, target, draft, us = batch(rng, counts, vocab, 3, drawn)
    target[:, ::3] = 0
    us[:] = u
    if np.isnan(u) or u < 0 or u >= 1:
        starts = np.concatenate([[0], np.cumsum(counts)])      # (not random numbers of [0, 1): some token that can be, and no node outside the tree)
        out = outputs(3, 4)
        tq.verify_drafts(ints(starts), ints(np.concatenate(parents)), ints(tokens), on_device(target), on_device(draft), torch.from_numpy(us).cuda(), **out)
        for i in range(3):
            k, path = int(out["kept"][i]), out["path"][i].tolist()
            assert 1 <= k <= 4 and path[0] == 0 and all(parents[i][b] == a for a, b in zip(path[:k], path[1:k]))
            assert target[starts[i] + path[k - 1], int(out["next"][i])] > 0
    else:
        check_verify(tq, counts, 4, parents, tokens, target, draft, us)


def test_rows_of_which_nothing_is_left(tq):
    """Targets that their drafts cover: the target's row again; rows without a positive number: no token."""
    rng = np.random.default_rng(6)
    counts, vocab = [4, 4, 4, 1], 2000
    parents, tokens, target, draft, u = batch(rng, counts, vocab, 1, True)
    u[:] = 0.999
    draft[:4] = 2 * target[:4] + 0.1
    target[4:8] = 0
    target[8:12, 1:] = np.nan
    target[8:12, 0] = -1
    target[12] = 0
    target[12, 1999] = 1e-30
    check_verify(tq, counts, 3, parents, tokens, target, draft, u)
    check_verify(tq, counts, 3, parents, tokens, target, None, u)


@pytest.mark.parametrize("drawn", [True, False])
def test_siblings_of_the_same_token(tq, drawn):
    rng = np.random.default_rng(7)
    counts, vocab = [9] * 40, 5
    parents, tokens, target, draft, u = batch(rng, counts, vocab, 9, drawn)
    parents = [[-1] + [0] * 8 for _ in counts]
    tokens[:] = rng.integers(0, 2, len(tokens))
    check_verify(tq, counts, 3, parents, tokens, target, draft, u)


@pytest.mark.parametrize("drawn", [True, False])
def test_nodes_that_are_nobody_s_children(tq, drawn):
    rng = np.random.default_rng(8)
    counts, vocab = [12] * 30, 64
    parents, tokens, target, draft, u = batch(rng, counts, vocab, 3, drawn)
    for par in parents:
        for j in rng.integers(1, 12, 4):
            par[j] = int(rng.choice([-1, -7, j, j + 1, 11, 1 << 30, -(1 << 31)]))
    at = rng.integers(0, len(tokens), 40)
    tokens[at] = rng.choice([-1, 64, 1 << 30, -(1 << 31), (1 << 31) - 1], 40)
    check_verify(tq, counts, 8, parents, tokens, target, draft, u)


def test_starts_outside_the_rows(tq):
    rng = np.random.default_rng(9)
    parents, tokens, target, draft, u = batch(rng, [5, 6], 40, 2, True)
    starts = [3, 2, 1 << 30, 11, 12, -5, 0, 5]       # backwards, beyond, empty, negative, and one that is fine
    out = outputs(7, 4)
    tq.verify_drafts(ints(starts), ints(np.concatenate(parents)), ints(tokens), on_device(target), on_device(draft), torch.from_numpy(u).cuda(), **out)
    path, token = drafts_model.verify(parents[0], tokens[:5], target[:5], draft[:5], u[:5], 4)
    assert out["kept"].tolist() == [0] * 6 + [len(path)] and out["next"].tolist() == [-1] * 6 + [token]
    assert out["path"].tolist() == [[-1] * 4] * 6 + [path + [-1] * (4 - len(path))]


def test_no_requests_and_no_rows(tq):
    rng = np.random.default_rng(10)
    parents, tokens, target, draft, u = batch(rng, [0, 0], 40, 2, True)
    out = outputs(2, 4)
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    rows = torch.zeros((0, 40), device="cuda")
    tq.verify_drafts(ints([0, 0, 0]), empty, empty, rows, rows, torch.zeros(0, device="cuda"), **out)
    assert out["kept"].tolist() == [0, 0] and out["next"].tolist() == [-1, -1]
    out = outputs(0, 4)
    tq.verify_drafts(ints([0]), empty, empty, rows, None, torch.zeros(0, device="cuda"), **out)


def test_a_large_vocabulary_on_another_stream_and_replayed(tq):
    """2^20 tokens, the most; a captured call on new numbers."""
    rng = np.random.default_rng(11)
    counts, vocab = [3, 2], 1 << 20
    for drawn in (True, False):
        sets = [batch(rng, counts, vocab, 1, drawn, sharp=6.0) for _ in range(2)]
        dev = [torch.from_numpy(x).cuda() if x is not None else None for x in sets[0][1:]]
        starts, parents, out = ints([0, 3, 5]), ints(np.concatenate(sets[0][0])), outputs(2, 3)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        call = lambda: tq.verify_drafts(starts, parents, *dev, **out, stream=side)      # noqa: E731
        with torch.cuda.stream(side):
            call()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                call()
        for s in sets[::-1]:
            for d, x in zip(dev, s[1:]):
                if d is not None:
                    d.copy_(torch.from_numpy(x))
            graph.replay()
            torch.cuda.synchronize()
            for i, rows in enumerate((slice(0, 3), slice(3, 5))):
                path, token = drafts_model.verify(s[0][i], s[1][rows], s[2][rows], None if s[3] is None else s[3][rows], s[4][rows], 3)
                assert out["path"][i].tolist()[:len(path)] == path and int(out["kept"][i]) == len(path) and int(out["next"][i]) == token


def test_results_where_arguments_are(tq):
    rng = np.random.default_rng(12)
    parents, tokens, target, draft, u = batch(rng, [5, 6], 40, 2, True)
    starts, drafted, uniforms = ints([0, 5, 11]), ints(tokens), torch.from_numpy(u).cuda()
    out = outputs(2, 4)
    for change in ({"next": drafted[3:5]}, {"kept": starts[1:]}, {"next": out["kept"]}, {"kept": out["path"].view(-1)[6:]}, {"path": uniforms.view(torch.int32)[:8].view(2, 4)}):
        with pytest.raises(tq.TQError, match="must not be where"):
            tq.verify_drafts(starts, ints(np.concatenate(parents)), drafted, on_device(target), on_device(draft), uniforms, **{**out, **change})


@pytest.mark.parametrize("drawn", [True, False])
def test_as_many_requests_as_there_may_be(tq, drawn):
    """65536 requests of one to three nodes: more clusters than the device holds at once, in any order."""
    rng = np.random.default_rng(13)
    distinct = 512
    counts = rng.integers(1, 4, distinct).tolist()
    parents, tokens, target, draft, u = batch(rng, counts, 9, 2, drawn)
    starts, times = np.concatenate([[0], np.cumsum(counts)]), 65536 // distinct
    rows, out = int(starts[-1]), outputs(65536, 3)
    many = ints(np.concatenate([starts[:-1] + k * rows for k in range(times)] + [[times * rows]]))
    again = lambda x: None if x is None else torch.from_numpy(np.concatenate([x] * times)).cuda()      # noqa: E731
    tq.verify_drafts(many, again(np.concatenate([np.asarray(p, np.int32) for p in parents])), again(tokens), again(target), again(draft), again(u), **out)
    torch.cuda.synchronize()
    want = [drafts_model.verify(parents[i], tokens[s:e], target[s:e], None if draft is None else draft[s:e], u[s:e], 3) for i, (s, e) in enumerate(zip(starts, starts[1:]))]
    assert out["kept"].tolist() == [len(p) for p, _ in want] * times and out["next"].tolist() == [t for _, t in want] * times
    assert out["path"].tolist() == [p + [-1] * (3 - len(p)) for p, _ in want] * times
