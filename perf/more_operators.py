"""A step of drafted decoding as cases that can be timed and whose results can be compared.

A request's drafts are a tree: its node 0 is the token that the last step ended with, every other node has a parent in front of
it, and all of them go through the model at once.  Four kinds of pass:

  rope     the norms of each head's query and key and the rotation by the nodes' positions, in one pass
  tree     attention of the nodes over a paged 8-bit cache: a node sees its request's older tokens, its ancestors and itself
  verify   which drafts stay: a walk down each tree that tests children against the target's probabilities with given random
           numbers, and the token that follows
  keep     the cache's side: nodes planned and appended, the accepted branch moved up in all layers, everything behind it given
           back, and the pages that hold the branch read; then the step is taken back, so that a pass can be repeated

Shapes are those of bench.py (Qwen2.5-7B- and 32B-shaped layers: 28 query heads on 4 KV heads and 40 on 8, of 128 dimensions,
contexts of 4k to 128k tokens, 151936 vocabulary entries) and generic ones; draw() spreads over the same ranges.

The definitions.

rope: x [D] of a head becomes y = x / sqrt(mean(x^2) + eps) * w, and (y_i, y_{i + D/2}) is rotated by position * theta^(-2 i / D).

tree: node j of a request that held L tokens has depth d_j (0 without a parent, otherwise its parent's + 1) and position L + d_j.
It sees the tokens 0 .. L - 1, its ancestors and itself; with a window w, of those the ones at positions above L + d_j - w.

verify: p is the target's row of the present node (node 0 at first), q the draft's, w = p and Z = 1.  Its children c come in order; with x
the child's token, c is accepted where u_c Z q(x) < w(x), and becomes the present node; otherwise w becomes max(w - Z q, 0) and Z the
sum of that.  Without a draft's rows a child is accepted where u_c Z < w(x); otherwise Z becomes Z - w(x) and w(x) 0.  Where no
child is accepted, the next token is the first one up to which the sum of w is above u_0 times all of it (w = p again where nothing
is left of it).

keep: a page holds `page` tokens as whole numbers -127 .. 127 times a power of two for each page and head, the smallest with which
the largest magnitude does not round to more than 127 (2^-100 at least).  Tokens that join a page make its scale larger where they
must, never smaller, and what the page holds is rounded again then.  The i-th token of a branch moves to the place of the i-th new
token: as it is within its page, as its value joins another one otherwise.
"""
import math
import random

import torch

own = False
DEV = "cuda"
EPS, THETA = 1e-6, 1e6


def _heads(q, kv, dim):
    return {"q_heads": q, "kv_heads": kv, "dim": dim}


LAYER_7B, LAYER_32B = _heads(28, 4, 128), _heads(40, 8, 128)


def _rope(rows, layer, far, apart=False, shape=1, name=None):
    """`far`: positions go up to it; `apart`: queries and keys are slices of one projection's rows."""
    c = {"kind": "rope", "rows": rows, **layer, "far": far, "apart": apart, "shape": shape}
    return {"name": name, **c} if name else c


def _tree(requests, nodes, context, page, layer, spread, window=0, pad=0, even=False, shape=1, name=None):
    """Trees of up to `nodes` nodes, a node's parent among the `spread` nodes in front of it (1: chains), over up to `context` tokens."""
    c = {"kind": "tree", "requests": requests, "nodes": nodes, "context": context, "page": page, **layer, "spread": spread,
         "window": window, "pad": pad, "even": even, "shape": shape}
    return {"name": name, **c} if name else c


def _verify(requests, nodes, vocab, spread, drafts, dtype="float32", pad=0, even=False, shape=1, name=None):
    """`drafts`: children were drawn from a draft model's rows; otherwise they were chosen (its most likely tokens)."""
    c = {"kind": "verify", "requests": requests, "nodes": nodes, "vocab": vocab, "spread": spread, "drafts": drafts, "dtype": dtype,
         "pad": pad, "even": even, "shape": shape}
    return {"name": name, **c} if name else c


def _keep(requests, nodes, context, page, layer, spread, layers, pad=0, even=False, shape=1, name=None):
    c = {"kind": "keep", "requests": requests, "nodes": nodes, "context": context, "page": page, **layer, "spread": spread,
         "layers": layers, "pad": pad, "even": even, "shape": shape}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the smallest call: one user's eight nodes, slices of a fused projection's rows
        _rope(8, LAYER_7B, 4096, apart=True, name="rope_one"),
        # a prompt, far into a context
        _rope(8192, LAYER_32B, 131072, name="rope_prompt_8k"),
        # eight nodes of one user
        _tree(1, 8, 4096, 64, LAYER_7B, 3, even=True, name="tree_one"),
        # a served batch of small trees, small pages and heads, under a sliding window; rows behind the last as a captured batch has
        _tree(61, 5, 1000, 16, _heads(16, 4, 64), 2, window=512, pad=3, name="tree_window_61"),
        # a served batch of unequal contexts and trees
        _tree(16, 16, 8192, 64, LAYER_7B, 4, name="tree_batch_16"),
        # ... of the larger model, with wider trees
        _tree(32, 31, 16384, 32, LAYER_32B, 8, name="tree_batch_32"),
        # two long conversations with large trees
        _tree(2, 64, 131072, 128, LAYER_32B, 8, name="tree_long_2"),
        # one user's chain of drafts from a small model
        _verify(1, 8, 151936, 1, True, even=True, name="verify_chain_one"),
        # a served batch of trees drawn from a draft model
        _verify(64, 16, 151936, 3, True, name="verify_drawn_64"),
        # chosen drafts, probabilities in halves, a vocabulary of odd size
        _verify(32, 60, 50257, 8, False, dtype="float16", pad=5, name="verify_chosen_32"),
        # one user, four layers
        _keep(1, 8, 4096, 64, LAYER_7B, 3, 4, even=True, name="keep_one"),
        # a served batch, small pages: branches that cross pages
        _keep(64, 31, 2048, 16, LAYER_32B, 4, 4, name="keep_batch_64"),
    ]


def _spread(rng, low, high):
    """A whole number, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rope", "tree", "tree", "verify", "keep"])
    page, kv = rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 4, 8])
    layer = _heads(kv * rng.choice([1, 2, 4, 5, 7, 8, 16]), kv, rng.choice([64, 128, 128]))
    shape, pad, even, spread = rng.randrange(1 << 20), rng.choice([0, 0, 1, 5]), rng.random() < 0.2, rng.choice([1, 2, 3, 4, 8, 16])
    if kind == "rope":
        room = 8192 * 48 * 128 // ((layer["q_heads"] + kv) * layer["dim"])
        return _rope(_spread(rng, 1, min(8192, room)), layer, _spread(rng, 1, 1 << 20), rng.random() < 0.5, shape)
    if kind == "tree":
        requests = _spread(rng, 1, 100)
        nodes = _spread(rng, 1, 64)
        room = 6.0e8 / (requests * layer["q_heads"] * nodes)       # (query, key) pairs that the plain form can hold
        context = _spread(rng, 1, max(2, min(131072, int(room), 300000 // requests)))
        return _tree(requests, nodes, context, page, layer, spread, rng.choice([0, 0, 0, _spread(rng, 1, 8192)]), pad, even, shape)
    if kind == "verify":
        nodes = _spread(rng, 1, 64)
        vocab = _spread(rng, 100, 160000)
        requests = _spread(rng, 1, max(1, min(200, int(64 * 16 * 151936 / (nodes * vocab)))))
        return _verify(requests, nodes, vocab, spread, rng.random() < 0.6, rng.choice(["float32", "float32", "float16"]), pad, even, shape)
    requests, layers = _spread(rng, 1, 64), rng.choice([1, 2, 4])
    return _keep(requests, _spread(rng, 1, 31), _spread(rng, 1, 2048), page, layer, spread, layers, pad, even, shape)


def _tokens(case):
    """(tokens held, parents of the new ones) of each request: by the case alone."""
    rng = random.Random(case["shape"])
    held, parents = [], []
    for _ in range(case["requests"]):
        top = case.get("context", 1)
        held.append(top if case["even"] else int(round(math.exp(rng.uniform(math.log(max(1, top / 8)), math.log(top))))))
        n = case["nodes"] if case["even"] else rng.randrange((case["nodes"] + 1) // 2, case["nodes"] + 1)
        parents.append([-1] + [max(0, j - 1 - rng.randrange(case["spread"])) for j in range(1, n)])
    return held, parents


def _depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _ancestors(parents):
    """ancestors[j][i]: i is an ancestor of j, or j."""
    rows = []
    for j, p in enumerate(parents):
        row = list(rows[p]) if p >= 0 else [False] * len(parents)
        row[j] = True
        rows.append(row)
    return rows


def _branches(parents, seed):
    """A node each, with the way down to it: what a verification found."""
    rng = random.Random(seed)
    paths = []
    for par in parents:
        j, path = rng.randrange(len(par)), []
        while j >= 0:
            path.append(j)
            j = par[j]
        paths.append(path[::-1])
    return paths


def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["rows"] * (case["q_heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 4 * n + 4 * case["rows"] + 4 * case["dim"], "flops": 7 * n}
    held, parents = _tokens(case)
    total = sum(map(len, parents))
    if kind == "verify":
        # a row of each of the models where the walk ends; tokens, parents and random numbers
        size = 4 if case["dtype"] == "float32" else 2
        rows = len(held) * (2 if case["drafts"] else 1)
        return {"bytes": rows * case["vocab"] * size + 12 * total + 8 * len(held), "flops": 2 * rows * case["vocab"]}
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    if kind == "tree":
        seen = pairs = 0
        for h, par in zip(held, parents):
            depths = _depths(par)
            first = max(0, h + 1 - case["window"]) if case["window"] else 0
            seen += max(0, h - first) + len(par)
            for d in depths:
                pairs += min(case["window"], h + d + 1) if case["window"] else h + d + 1
        return {"bytes": 2 * heads * seen * dim + total * case["q_heads"] * (dim * 4 + 4), "flops": 4 * dim * case["q_heads"] * pairs}
    paths = _branches(parents, case["shape"])
    pages = sum((h + len(p) - 1) // page - h // page + 1 for h, p in zip(held, paths))
    moved = sum(a != i for p in paths for i, a in enumerate(p))
    # keys and values read and written as bytes, moved as bytes, the branch's pages read as bytes and written as fp16
    return {"bytes": 2 * case["layers"] * heads * (total * dim * 3 + moved * dim * 2 + pages * (page * dim * 3 + 8)), "flops": 0}


def _values(gen, tokens, case, gain):
    """Keys or values of `tokens` tokens: of unequal strength from channel to channel and from token to token, as a model's are."""
    x = torch.randn((tokens, case["kv_heads"], case["dim"]), generator=gen, device=DEV)
    x *= torch.exp(0.5 * torch.randn((tokens, 1, 1), generator=gen, device=DEV))
    return (x * gain).half()


def _kv(case, seed):
    """For each layer the keys and values of the held tokens and of the new ones (with rows behind the last)."""
    held, parents = _tokens(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    total, pad = sum(map(len, parents)), case["pad"]
    layers = []
    for _ in range(case.get("layers", 1)):
        gains = [torch.exp(s * torch.randn((1, case["kv_heads"], case["dim"]), generator=gen, device=DEV)) for s in (0.4, 0.2)]
        layers.append([(_values(gen, sum(held), case, g), _values(gen, total + pad, case, g)) for g in gains])
    q = torch.randn((total + pad, case.get("q_heads", 1), case["dim"]), generator=gen, device=DEV).half() if case["kind"] == "tree" else None
    return layers, q


def _rope_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n, q, k, dim = case["rows"], case["q_heads"], case["kv_heads"], case["dim"]
    rows = torch.randn((n, q + 2 * k if case["apart"] else q + k, dim), generator=gen, device=DEV)
    rows = (rows * torch.exp(torch.randn((n, rows.shape[1], 1), generator=gen, device=DEV))).half()
    x = [rows[:, :q], rows[:, q:q + k]]
    if not case["apart"]:
        x = [t.contiguous() for t in x]
    weights = [(1 + 0.3 * torch.randn(dim, generator=gen, device=DEV)).half() for _ in range(2)]
    first = random.Random(case["shape"]).randrange(max(1, case["far"] - n + 1))
    positions = (first + torch.arange(n, device=DEV)).clamp(max=case["far"]).int()
    return x, weights, positions


def _verify_inputs(case, seed):
    """Starts, parents, tokens, the target's and the draft's rows (None), random numbers."""
    _, parents = _tokens(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, total, vocab = getattr(torch, case["dtype"]), sum(map(len, parents)), case["vocab"]
    rows = total + case["pad"]
    flat = torch.tensor([p for par in parents for p in par] + [-1] * case["pad"], dtype=torch.int32, device=DEV)
    starts = [0]
    for par in parents:
        starts.append(starts[-1] + len(par))
    target, draft = torch.empty((rows, vocab), dtype=dtype, device=DEV), torch.empty((rows, vocab), dtype=dtype, device=DEV)
    for r in range(0, rows, 256):        # logits of a few likely tokens and many unlikely ones; the draft's are nearly the target's
        e = min(rows, r + 256)
        logits = 4 * torch.randn((e - r, vocab), generator=gen, device=DEV)
        target[r:e] = torch.softmax(logits, 1).to(dtype)
        draft[r:e] = torch.softmax(logits + 0.7 * torch.randn((e - r, vocab), generator=gen, device=DEV), 1).to(dtype)
    # a child's token: drawn from its parent's row, or the next most likely one of it
    up = torch.cat([torch.tensor([max(p, 0) + s for p in par], device=DEV) for par, s in zip(parents, starts)])
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    if case["drafts"]:
        for r in range(0, total, 256):
            at = up[r:min(total, r + 256)]
            sums = torch.cumsum(draft[at].double(), 1)
            u = torch.rand((at.shape[0], 1), generator=gen, device=DEV, dtype=torch.float64) * sums[:, -1:]
            tokens[r:r + at.shape[0]] = torch.searchsorted(sums, u, right=True)[:, 0].clamp(max=vocab - 1)
    else:
        rank, turns = {}, []
        for i, s in enumerate(starts[:-1]):
            for p in parents[i]:
                rank[i, p] = rank.get((i, p), -1) + 1
                turns.append(rank[i, p])
        most = min(vocab, max(turns) + 1)
        best = torch.cat([torch.topk(draft[r:r + 256].float(), most, 1).indices for r in range(0, rows, 256)])
        tokens[:total] = best[up, torch.tensor(turns, device=DEV).clamp(max=most - 1)]
    uniforms = torch.rand((rows,), generator=gen, device=DEV)
    return {"starts": torch.tensor(starts, dtype=torch.int32, device=DEV), "parents": flat, "tokens": tokens.int(), "target": target,
            "draft": draft if case["drafts"] else None, "uniforms": uniforms, "most": max(map(len, parents)),
            "width": 1 + max(max(_depths(par)) for par in parents)}


# ---- the plain form ---------------------------------------------------------------------------------------------------

def _plain_rope(s):
    out = []
    dim = s["x"][0].shape[2]
    frequency = THETA ** (-torch.arange(0, dim, 2, device=DEV, dtype=torch.float64) / dim)
    angle = s["positions"].double()[:, None, None] * frequency
    c, sn = torch.cos(angle).float(), torch.sin(angle).float()
    for x, w in zip(s["x"], s["weights"]):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = y[..., :dim // 2], y[..., dim // 2:]
        out.append(torch.cat([a * c - b * sn, b * c + a * sn], -1).half())
    return out


def _plain_scale(top):
    """The power of two for a largest magnitude."""
    m, x = torch.frexp(top)
    e = torch.where(m * 128 < 127.5, x - 7, x - 6)
    e = torch.where(top == 0, -100, e).clamp(min=-100)
    return ((e + 127) << 23).view(torch.float32)


def _plain_join(codes, scales, x, request, place, page):
    """x [tokens, heads, dim] joins request[t]'s cache at token place[t]; codes [n, tokens, heads, dim], scales [n, pages, heads]; what a
    page holds in front of them stays, another one's scale begins anew."""
    n, pages, heads = scales.shape
    cell = request * pages + place // page
    x = x.float()
    top = torch.zeros((n * pages, heads), device=DEV).index_reduce_(0, cell, x.abs().amax(-1), "amax").reshape(n, pages, heads)
    first = torch.full((n * pages,), page, device=DEV).index_reduce_(0, cell, place % page, "amin").reshape(n, pages)
    held = torch.where((first == 0)[..., None], 0, scales)
    scale = torch.where((first == page)[..., None], scales, torch.maximum(held, _plain_scale(top)))
    ratio = (scales / scale).repeat_interleave(page, 1)[..., None]
    older = (torch.arange(page, device=DEV) < first[..., None]).reshape(n, pages * page)[..., None, None]
    codes.copy_(torch.where(older, torch.round(codes.float() * ratio).to(torch.int8), codes))
    codes[request, place] = torch.round(x / scale[request, place // page][..., None]).to(torch.int8)
    scales.copy_(scale)


def _plain_keep(codes, scales, request, source, place, page):
    """The tokens at `source` move to `place`, within one tensor of one layer."""
    n, pages, heads = scales.shape
    moving = codes[request, source].float()
    values = moving * scales[request, source // page][..., None]
    foreign = source // page != place // page
    cell = request * pages + place // page
    need = torch.zeros((n * pages, heads), device=DEV)
    need.index_reduce_(0, cell, values.abs().amax(-1) * foreign[:, None], "amax")
    need = need.reshape(n, pages, heads)
    scale = torch.where(need > 0, torch.maximum(scales, _plain_scale(need)), scales)
    ratio = (scales / scale).repeat_interleave(page, 1)[..., None]
    codes.copy_(torch.round(codes.float() * ratio).to(torch.int8))
    to = scale[request, place // page][..., None]
    stay = torch.round(moving * (scales[request, place // page][..., None] / to))
    codes[request, place] = torch.where(foreign[:, None, None], torch.round(values / to), stay).to(torch.int8)
    scales.copy_(scale)


def _plain_depths(parents, request, j, most):
    """Depths of all nodes, and ancestors [tokens, most]: node j's, and itself, by index in its request."""
    total = parents.shape[0]
    index = torch.arange(total, device=DEV)
    depth = torch.zeros(total, dtype=torch.long, device=DEV)
    above = torch.zeros((total, most), dtype=torch.bool, device=DEV)
    at = j.clone()
    for _ in range(most):
        live = at >= 0
        above[index, at.clamp(min=0)] |= live
        up = torch.where(live, parents[(index - j + at.clamp(min=0))], -1)
        depth += up >= 0
        at = up
    return depth, above


def _plain_tree(s):
    q, page, most = s["q"], s["page"], s["most"]
    (k, k_scale), (v, v_scale) = s["cache"][0]
    n, tokens, heads, dim = k.shape
    group = q.shape[1] // heads
    k = k.float() * k_scale.repeat_interleave(page, 1)[..., None]
    v = v.float() * v_scale.repeat_interleave(page, 1)[..., None]
    depth, above = _plain_depths(s["parents"], s["request"], s["j"], most)
    live = s["request"].shape[0]
    x = torch.zeros((n, most, heads * group, dim), device=DEV)
    x[s["request"], s["j"]] = q[:live].float()
    x = x.reshape(n, most, heads, group, dim).permute(0, 2, 1, 3, 4).reshape(n, heads, most * group, dim)
    scores = torch.matmul(x, k.permute(0, 2, 3, 1)) * (1 / math.sqrt(dim))
    # what each node sees: older tokens, and of the new ones its ancestors
    t = torch.arange(tokens, device=DEV)[None]
    held = s["held"][s["request"]][:, None]
    local = t - held
    up = torch.gather(above, 1, local.clamp(0, most - 1)) & (local >= 0) & (local < most)
    seen = (local < 0) | up
    if s["window"]:
        starts = (torch.arange(live, device=DEV) - s["j"])[:, None]
        place = torch.where(local < 0, t, held + depth[(starts + local.clamp(min=0)).clamp(max=live - 1)])
        seen &= place > held + depth[:, None] - s["window"]
    mask = torch.ones((n, most, tokens), dtype=torch.bool, device=DEV)
    mask[s["request"], s["j"]] = seen
    scores = scores.reshape(n, heads, most, group, tokens).masked_fill_(~mask[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp_(scores.sub_(top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.reshape(n, heads, most * group, tokens), v.transpose(1, 2)).reshape(n, heads, most, group, dim) / total
    lse = (top + torch.log(total))[..., 0]
    result, sums = torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV)
    result[:live] = out.permute(0, 2, 1, 3, 4).reshape(n, most, heads * group, dim)[s["request"], s["j"]].half()
    sums[:live] = lse.permute(0, 2, 1, 3).reshape(n, most, heads * group)[s["request"], s["j"]]
    return result, sums


def _plain_verify(s):
    starts, parents, tokens, u = s["starts"].long(), s["parents"].long(), s["tokens"].long(), s["uniforms"].double()
    n, vocab, drawn = starts.shape[0] - 1, s["target"].shape[1], s["draft"] is not None
    first, count = starts[:-1], starts[1:] - starts[:-1]
    each = torch.arange(n, device=DEV)
    now = torch.zeros(n, dtype=torch.long, device=DEV)
    path = torch.full((n, s["width"]), -1, dtype=torch.long, device=DEV)
    path[:, 0] = 0
    kept = torch.ones(n, dtype=torch.long, device=DEV)
    w, z = s["target"][first].double(), torch.ones(n, dtype=torch.float64, device=DEV)
    q = s["draft"][first].double() if drawn else None
    for j in range(1, s["most"]):
        row = (first + j).clamp(max=parents.shape[0] - 1)
        child = (j < count) & (parents[row] == now)
        x = tokens[row]
        here = w[each, x]
        take = child & ((u[row] * z * q[each, x] if drawn else u[row] * z) < here)
        leave = child & ~take
        # the ones that stay behind: what is left of their distribution
        if drawn:
            rest = (w - z[:, None] * q).clamp_(min=0)
            w = torch.where(leave[:, None], rest, w)
            z = torch.where(leave, rest.sum(1), z)
        else:
            z = torch.where(leave, z - here, z)
            w[each, x] = torch.where(leave, 0, here)
        now = torch.where(take, j, now)
        path[each, torch.where(take, kept, 0)] = torch.where(take, now, 0)
        kept += take
        w = torch.where(take[:, None], s["target"][row].double(), w)
        z = torch.where(take, 1, z)
        if drawn:
            q = torch.where(take[:, None], s["draft"][row].double(), q)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, s["target"][first + now].double())
    sums = torch.cumsum(w, 1)
    token = torch.searchsorted(sums, (u[first] * sums[:, -1])[:, None], right=True)[:, 0].clamp(max=vocab - 1)
    return {"path": path.int(), "kept": kept.int(), "next": token.int()}


# ---- both -------------------------------------------------------------------------------------------------------------

def _prepare_cache(case, seed):
    held, parents = _tokens(case)
    layers, q = _kv(case, seed)
    page, n, pad = case["page"], len(held), case["pad"]
    counts = [len(p) for p in parents]
    total, most, width = sum(counts), max(counts), max(-(-(h + c) // page) for h, c in zip(held, counts))
    flat = torch.tensor([p for par in parents for p in par] + [-1] * pad, dtype=torch.int32, device=DEV)
    ints = {"dtype": torch.int32, "device": DEV}
    s = {"kind": case["kind"], "q": q, "page": page, "most": most, "total": total, "window": case.get("window", 0)}
    if case["kind"] == "keep":
        paths = _branches(parents, case["shape"])
        s["path"] = torch.full((n, max(map(len, paths))), -1, **ints)
        for i, p in enumerate(paths):
            s["path"][i, :len(p)] = torch.tensor(p, **ints)
        s["kept"] = torch.tensor([len(p) for p in paths], **ints)
        s["new"] = [[x[1] for x in kv] for kv in layers]
        spots = [range(h // page, (h + len(p) - 1) // page + 1) for h, p in zip(held, paths)]
    if own:
        import turboquant_mlx_core_b200 as tq
        cache = tq.PagedKVCache(len(layers), case["kv_heads"], case["dim"], sum(-(-(h + c) // page) for h, c in zip(held, counts)) + 7, page,
                                max_requests=n, max_pages_per_request=width, max_tokens=max(total + pad, sum(held)))
        cache.plan(torch.tensor(held, **ints), sum(held), max(held))
        for i, kv in enumerate(layers):
            cache.append(i, kv[0][0], kv[1][0])
        s |= {"cache": cache, "parents": flat, "counts": torch.tensor(counts, **ints), "rows": total + pad, "held": torch.tensor(held, **ints),
              "positions": torch.empty(total + pad, **ints), "lengths": torch.empty(n, **ints)}
        if case["kind"] == "tree":
            cache.plan(s["counts"], total + pad, most)
            cache.tree(flat, positions=s["positions"])
            cache.append(0, layers[0][0][1], layers[0][1][1])
            s |= {"out": torch.zeros_like(q), "lse": torch.zeros(q.shape[:2], device=DEV)}
        else:
            tables = torch.empty((n, width), **ints)
            cache.plan(s["counts"], total + pad, most, tables=tables)
            cache.truncate(s["held"])
            s["pages"] = torch.cat([tables[i, r.start:r.stop] for i, r in enumerate(spots)])
            size = (s["pages"].shape[0], page, case["kv_heads"], case["dim"])
            s["values"] = [[torch.empty(size, dtype=torch.float16, device=DEV) for _ in range(2)] for _ in layers]
            rest = [c - len(p) for c, p in zip(counts, paths)]
            s |= {"rest": torch.tensor(rest, **ints), "rest_sizes": (sum(rest), max(rest))}
    else:
        old = torch.tensor(held, device=DEV)
        request = torch.repeat_interleave(torch.arange(n, device=DEV), torch.tensor(counts, device=DEV))
        j = torch.arange(total, device=DEV) - torch.repeat_interleave(torch.tensor([sum(counts[:i]) for i in range(n)], device=DEV), torch.tensor(counts, device=DEV))
        s |= {"request": request, "j": j, "held": old, "parents": flat[:total].long(), "cache": []}
        r0 = torch.repeat_interleave(torch.arange(n, device=DEV), old)
        p0 = torch.cat([torch.arange(h, device=DEV) for h in held])
        for kv in layers:
            s["cache"].append([])
            for x, more in kv:
                codes = torch.zeros((n, width * page, case["kv_heads"], case["dim"]), dtype=torch.int8, device=DEV)
                scales = torch.full((n, width, case["kv_heads"]), 2.0 ** -100, device=DEV)
                _plain_join(codes, scales, x, r0, p0, page)
                if case["kind"] == "tree":
                    _plain_join(codes, scales, more[:total], request, old[request] + j, page)
                s["cache"][-1].append((codes, scales))
        if case["kind"] == "keep":
            s["spot"] = (torch.cat([torch.full((len(r),), i, device=DEV) for i, r in enumerate(spots)]), torch.cat([torch.arange(r.start, r.stop, device=DEV) for r in spots]))
            s["padded"] = total + pad
    if case["kind"] == "keep":
        run(s)      # the first pass may make a scale larger that the later ones find as it is
    return s


def prepare(case, seed):
    if case["kind"] == "rope":
        x, weights, positions = _rope_inputs(case, seed)
        return {"kind": "rope", "x": x, "weights": weights, "positions": positions, "out": [torch.empty(t.shape, dtype=t.dtype, device=DEV) for t in x]}
    if case["kind"] == "verify":
        s = {"kind": "verify", **_verify_inputs(case, seed)}
        n, ints = s["starts"].shape[0] - 1, {"dtype": torch.int32, "device": DEV}
        s["outputs"] = {"path": torch.empty((n, s["width"]), **ints), "kept": torch.empty(n, **ints), "next": torch.empty(n, **ints)}
        return s
    return _prepare_cache(case, seed)


def run(s):
    if s["kind"] == "rope":
        if own:
            import turboquant_mlx_core_b200 as tq
            tq.qk_norm_rope(*s["x"], *s["weights"], s["positions"], theta=THETA, eps=EPS, out=s["out"])
            return s["out"]
        return _plain_rope(s)
    if s["kind"] == "verify":
        if own:
            import turboquant_mlx_core_b200 as tq
            tq.verify_drafts(s["starts"], s["parents"], s["tokens"], s["target"], s["draft"], s["uniforms"], **s["outputs"])
            return s["outputs"]
        return _plain_verify(s)
    if s["kind"] == "tree":
        if own:
            s["cache"].tree_attention(0, s["q"], window=s["window"], out=s["out"], lse=s["lse"])
            return s["out"], s["lse"]
        return _plain_tree(s)
    if own:
        cache = s["cache"]
        cache.plan(s["counts"], s["rows"], s["most"])
        cache.tree(s["parents"], positions=s["positions"])
        for i, kv in enumerate(s["new"]):
            cache.append(i, *kv)
        cache.keep(s["path"], s["kept"], lengths=s["lengths"])
        for i, kv in enumerate(s["values"]):
            cache.read_pages(i, s["pages"], *kv)
        cache.plan(s["rest"], *s["rest_sizes"])      # (each request's pages again, so that the next pass takes them in this one's order)
        cache.truncate(s["held"])
        return s["positions"], s["lengths"], s["values"]
    total, page, held = s["total"], s["page"], s["held"]
    depth, _ = _plain_depths(s["parents"], s["request"], s["j"], s["most"])
    positions = torch.zeros(s["padded"], dtype=torch.int32, device=DEV)
    positions[:total] = held[s["request"]] + depth
    live = s["path"] >= 0
    request, i = torch.nonzero(live, as_tuple=True)
    source, place = held[request] + s["path"][live], held[request] + i
    values = []
    for cache, kv in zip(s["cache"], s["new"]):
        values.append([])
        for (codes, scales), x in zip(cache, kv):
            _plain_join(codes, scales, x[:total], s["request"], held[s["request"]] + s["j"], page)
            _plain_keep(codes, scales, request, source, place, page)
            n, _, heads, dim = codes.shape
            values[-1].append((codes.reshape(n, -1, page, heads, dim)[s["spot"]].float() * scales[s["spot"]][:, None, :, None]).half())
    return positions, (held + s["kept"]).int(), values


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

def _power(e):
    """2^e by its bits: a library's power need not be exact."""
    return ((e + 1023) << 52).view(torch.float64)


def _exponent(top):
    """The smallest e with which top / 2^e rounds to 127 at most."""
    e = torch.clamp(torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 127.5)), -900, 900).long()
    e = torch.where(top * _power(-e) >= 127.5, e + 1, e)
    e = torch.where(top * _power(1 - e) < 127.5, e - 1, e)
    return torch.clamp(e, min=-100)


class _Request:
    """One request's keys or values: whole numbers [pages, page, heads, dim] and exponents [pages, heads]."""

    def __init__(self, tokens, case):
        pages = -(-tokens // case["page"])
        self.page, self.codes = case["page"], torch.zeros((pages, case["page"], case["kv_heads"], case["dim"]), dtype=torch.float64, device=DEV)
        self.e = torch.full((pages, case["kv_heads"]), -100, device=DEV)

    def raised(self, page, e, rows):
        self.codes[page, :rows] = torch.round(self.codes[page, :rows] * _power(self.e[page] - e)[None, :, None])
        self.e[page] = e

    def join(self, x, begin):
        """Tokens `begin` and on."""
        x = x.double()
        at, page = begin % self.page, begin // self.page
        if at:      # beside older ones
            n = min(self.page - at, x.shape[0])
            self.raised(page, torch.maximum(_exponent(x[:n].abs().amax((0, 2))), self.e[page]), at)
            self.codes[page, at:at + n] = torch.round(x[:n] * _power(-self.e[page])[None, :, None])
            x, page = x[n:], page + 1
        if x.shape[0]:
            pages, place = -(-x.shape[0] // self.page), torch.arange(x.shape[0], device=DEV)
            full = torch.cat([x, x.new_zeros((pages * self.page - x.shape[0], *x.shape[1:]))]).reshape(pages, self.page, *x.shape[1:])
            self.e[page:page + pages] = _exponent(full.abs().amax((1, 3)))
            scaled = torch.round(full * _power(-self.e[page:page + pages])[:, None, :, None])
            self.codes[page + place // self.page, place % self.page] = scaled.flatten(0, 1)[:x.shape[0]]

    def keep(self, path, begin):
        for page in range(begin // self.page, (begin + len(path) - 1) // self.page + 1):
            mine = [(begin + a, begin + i) for i, a in enumerate(path) if (begin + i) // self.page == page]
            for a, i in mine:
                if a // self.page == page:
                    self.codes[page, i % self.page] = self.codes[page, a % self.page]
            others = [(a, i) for a, i in mine if a // self.page != page]
            if not others:
                continue
            x = torch.stack([self.codes[a // self.page, a % self.page] * _power(self.e[a // self.page])[:, None] for a, _ in others])
            top = x.abs().amax((0, 2))
            self.raised(page, torch.where(top > 0, torch.maximum(self.e[page], _exponent(top)), self.e[page]), self.page)
            for (_, i), v in zip(others, x):
                self.codes[page, i % self.page] = torch.round(v * _power(-self.e[page])[:, None])

    def values(self):
        return self.codes * _power(self.e)[:, None, :, None]


def exact(case, seed):
    if case["kind"] == "rope":
        x, weights, positions = _rope_inputs(case, seed)
        out, half = [], case["dim"] // 2
        for t, w in zip(x, weights):
            t = t.double()
            y = t / torch.sqrt((t ** 2).sum(2, keepdim=True) / case["dim"] + EPS) * w.double()
            r = torch.empty_like(y)
            for i in range(half):
                a = positions.double()[:, None] * math.exp(-2 * i / case["dim"] * math.log(THETA))
                r[:, :, i] = y[:, :, i] * torch.cos(a) - y[:, :, i + half] * torch.sin(a)
                r[:, :, i + half] = y[:, :, i + half] * torch.cos(a) + y[:, :, i] * torch.sin(a)
            out.append(r)
        return out
    held, parents = _tokens(case)
    n = len(held)
    starts = [sum(len(p) for p in parents[:i]) for i in range(n)]
    if case["kind"] == "verify":
        v = _verify_inputs(case, seed)
        tokens, u = v["tokens"].tolist(), v["uniforms"].tolist()
        path = torch.full((n, v["width"]), -1, dtype=torch.int32)
        kept, following = [], []
        for i, par in enumerate(parents):
            node, way = 0, [0]
            while True:
                p = v["target"][starts[i] + node].double()
                q = v["draft"][starts[i] + node].double() if case["drafts"] else None
                w, z, found = p.clone(), 1.0, None
                for c in range(len(par)):
                    if par[c] != node:
                        continue
                    x = tokens[starts[i] + c]
                    if u[starts[i] + c] * z * (float(q[x]) if q is not None else 1.0) < float(w[x]):
                        found = c
                        break
                    if q is not None:
                        w = torch.clamp(w - z * q, min=0)
                        z = float(w.sum())
                    else:
                        z -= float(w[x])
                        w[x] = 0
                if found is None:
                    break
                node = found
                way.append(node)
            if float(w.sum()) <= 0:
                w = p
            sums = torch.cumsum(w, 0)
            following.append(min(int((sums <= u[starts[i]] * sums[-1]).sum()), case["vocab"] - 1))
            path[i, :len(way)] = torch.tensor(way, dtype=torch.int32)
            kept.append(len(way))
        ints = {"dtype": torch.int32, "device": DEV}
        return {"path": path.to(DEV), "kept": torch.tensor(kept, **ints), "next": torch.tensor(following, **ints)}

    layers, q = _kv(case, seed)
    begins = [sum(held[:i]) for i in range(n)]

    def filled(x, i):
        r = _Request(held[i] + len(parents[i]), case)
        r.join(x[0][begins[i]:begins[i] + held[i]], 0)
        return r

    if case["kind"] == "keep":
        paths = _branches(parents, case["shape"])
        positions = [h + d for h, par in zip(held, parents) for d in _depths(par)] + [0] * case["pad"]
        values = []
        for kv in layers:
            values.append([])
            for x in kv:
                pages = []
                for i in range(n):
                    r = filled(x, i)
                    for _ in range(2):       # prepare() makes a pass, too
                        r.join(x[1][starts[i]:starts[i] + len(parents[i])], held[i])
                        r.keep(paths[i], held[i])
                    pages.append(r.values()[held[i] // case["page"]:(held[i] + len(paths[i]) - 1) // case["page"] + 1])
                values[-1].append(torch.cat(pages))
        ints = {"dtype": torch.int32, "device": DEV}
        return torch.tensor(positions, **ints), torch.tensor([h + len(p) for h, p in zip(held, paths)], **ints), values

    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    group = case["q_heads"] // case["kv_heads"]
    for i, par in enumerate(parents):
        kv = []
        for x in layers[0]:
            r = filled(x, i)
            r.join(x[1][starts[i]:starts[i] + len(par)], held[i])
            kv.append(r.values().flatten(0, 1)[:held[i] + len(par)])
        depths = torch.tensor(_depths(par), device=DEV)
        seen = torch.cat([torch.ones((len(par), held[i]), dtype=torch.bool, device=DEV), torch.tensor(_ancestors(par), device=DEV)], 1)
        if case["window"]:
            places = torch.cat([torch.arange(held[i], device=DEV), held[i] + depths])
            seen &= places[None] > held[i] + depths[:, None] - case["window"]
        rows = slice(starts[i], starts[i] + len(par))
        for h in range(case["q_heads"]):
            s = q[rows, h].double() @ kv[0][:, h // group].T / math.sqrt(case["dim"])
            s[~seen] = -math.inf
            lse[rows, h] = torch.logsumexp(s, 1)
            out[rows, h] = torch.softmax(s, 1) @ kv[1][:, h // group]
    return out, lse
