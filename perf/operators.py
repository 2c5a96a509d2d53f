"""The paged 8-bit KV cache as cases that can be timed and whose results can be compared.

Three kinds of pass, on one layer of a cache that requests share in pages:

  plan      new tokens are planned from their counts (block tables, slot map, positions, starts, lengths) and taken back
            again, as a decode loop that rolls rejected drafts back does
  append    the planned tokens' keys and values are written into the cache in 8 bits, with a scale for each page and head,
            and the pages that they went to are read back
  attend    causal attention of the planned tokens' queries over the cache: single tokens, drafts, prompts and chunks

Shapes are those of bench.py (Qwen2.5-7B- and 32B-shaped layers: 28 query heads on 4 KV heads and 40 on 8, of 128
dimensions, contexts of 4k to 128k tokens) and generic ones; draw() spreads over the same ranges.

The definitions.  A page holds `page` tokens.  Request i holds len_i tokens and gets c_i more; its pages grow to
ceil((len_i + c_i) / page), and the new ones come off the end of a stack of free pages, in the requests' order.  Token j of
the new ones has position len_i + j and slot page_of(position) * page + position % page.  Keys and values are held as whole
numbers of -127 .. 127 times a power of two for each page and head: the smallest with which the largest magnitude does not
round to more than 127 (and 2^-100 at least).  Tokens that join a page which holds older ones can make its scale larger, never
smaller; the older numbers are rounded again then.  The query of a token at position p sees positions max(0, p - window + 1)
.. p (all up to p without a window), with softmax(q . k / sqrt(dim)).
"""
import math
import random

import torch

own = False
DEV = "cuda"
OTHERS = 1000       # pages, at most, that requests outside the batch hold


def _heads(q, kv, dim):
    return {"q_heads": q, "kv_heads": kv, "dim": dim}


LAYER_7B, LAYER_32B = _heads(28, 4, 128), _heads(40, 8, 128)


def _case(kind, requests, chunked, new, context, page, layer, window=0, dtype="float16", pad=0, even=False, name=None, shape=1):
    """`requests` requests of up to `context` tokens, of which the first `chunked` get up to `new` tokens and the others one; `even`:
    all have as much as there can be, otherwise they are ragged; `pad`: rows behind the last request's, as a captured batch has."""
    c = {"kind": kind, "requests": requests, "chunked": chunked, "new": new, "context": context, "page": page, **layer,
         "window": window, "dtype": dtype, "pad": pad, "even": even, "shape": shape}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one user's decode step; the page that the token goes to is new
        _case("plan", 1, 0, 1, 4096, 64, LAYER_7B, even=True, name="plan_one"),
        # the decode step of a large served batch, captured with room for more rows
        _case("plan", 509, 0, 1, 8192, 64, LAYER_32B, pad=3, name="plan_decode_509"),
        # a batch of prompts of unequal lengths admitted at once, small pages
        _case("plan", 61, 61, 8192, 0, 16, LAYER_7B, name="plan_prompts"),
        # one token of one user
        _case("append", 1, 0, 1, 4096, 64, LAYER_7B, name="append_one"),
        # one token each of a served batch
        _case("append", 251, 0, 1, 1000, 64, LAYER_32B, name="append_decode_251"),
        # prompts of unequal lengths, from a layer that computes in fp32
        _case("append", 11, 11, 8192, 130, 32, LAYER_32B, dtype="float32", name="append_prompts"),
        # decode attention of one user
        _case("attend", 1, 0, 1, 4096, 64, LAYER_7B, name="attend_one"),
        # ... of a served batch of unequal contexts
        _case("attend", 32, 0, 1, 32768, 64, LAYER_32B, name="attend_decode_32"),
        # two long conversations
        _case("attend", 2, 0, 1, 131072, 128, LAYER_32B, name="attend_long_2"),
        # five drafted tokens each are verified, under a sliding window
        _case("attend", 16, 16, 5, 8192, 16, LAYER_7B, window=4096, name="attend_drafts_16"),
        # a prompt
        _case("attend", 1, 1, 8192, 0, 64, LAYER_7B, even=True, name="attend_prompt_8k"),
        # a chunk of one prompt beside the decode steps of others
        _case("attend", 8, 1, 512, 16384, 64, LAYER_7B, name="attend_chunk_and_decode"),
    ]


def _spread(rng, low, high):
    """A whole number, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    kv = rng.choice([1, 2, 4, 8])
    layer = _heads(kv * rng.choice([1, 2, 4, 5, 7, 8, 16]), kv, rng.choice([64, 128, 128]))
    shape, pad, even = rng.randrange(1 << 20), rng.choice([0, 0, 1, 5]), rng.random() < 0.2
    if kind == "plan":
        requests = _spread(rng, 1, 600)
        prompts = rng.random() < 0.4
        return _case(kind, requests, requests if prompts else 0, _spread(rng, 2, 8192 * 61 // max(61, requests)) if prompts else 1,
                     0 if prompts else _spread(rng, 1, 8192), page, layer, pad=pad, even=even, shape=shape)
    if kind == "append":
        requests = _spread(rng, 1, 300)
        prompts = rng.random() < 0.5
        new = _spread(rng, 2, max(3, 20000 // requests)) if prompts else 1
        return _case(kind, requests, requests if prompts else 0, new, _spread(rng, 1, max(2, 60000 // requests)), page, layer,
                     dtype=rng.choice(["float16", "float32"]), pad=pad, even=even, shape=shape)
    window = rng.choice([0, 0, 0, _spread(rng, 1, 8192)])
    form = rng.choice(["decode", "drafts", "prompts", "mixed"])
    if form == "decode":
        requests = _spread(rng, 1, 200)
        return _case(kind, requests, 0, 1, _spread(rng, 1, 600000 // requests // max(1, kv // 4)), page, layer, window, pad=pad, even=even, shape=shape)
    if form == "drafts":
        requests = _spread(rng, 1, 64)
        return _case(kind, requests, requests, rng.randrange(2, 12), _spread(rng, 1, 120000 // requests), page, layer, window, pad=pad, even=even, shape=shape)
    requests = _spread(rng, 1, 8)
    room = 6.0e8 / (requests * layer["q_heads"])        # padded (query, key) pairs that the plain form can hold
    new = _spread(rng, 2, int(min(4096, math.sqrt(room))))
    context = _spread(rng, 1, max(2, int(room / new) - new))
    return _case(kind, requests, requests if form == "prompts" else 1, new, context, page, layer, window, pad=pad, even=even, shape=shape)


def _sizes(case):
    """(tokens held, new tokens) of each request: by the case alone."""
    rng = random.Random(case["shape"])
    held, new = [], []
    for i in range(case["requests"]):
        top = case["context"]
        held.append(top if case["even"] or top == 0 else int(round(math.exp(rng.uniform(math.log(max(1, top / 8)), math.log(top))))))
        if i >= case["chunked"]:
            new.append(1)
        else:
            new.append(case["new"] if case["even"] else rng.randrange((case["new"] + 1) // 2, case["new"] + 1))
    return held, new


def work(case):
    held, new = _sizes(case)
    n, total, page, heads, dim = len(held), sum(new), case["page"], case["kv_heads"], case["dim"]
    after = [h + c for h, c in zip(held, new)]
    width = max(-(-a // page) for a in after)
    if case["kind"] == "plan":
        # counts and lengths read, starts, lengths, slots, positions and tables written; tables and the stack of the pages that change hands
        moved = sum(-(-a // page) - -(-h // page) for h, a in zip(held, after))
        return {"bytes": 4 * (3 * n + 2 * n + 1 + 2 * (total + case["pad"]) + n * width + sum(-(-a // page) for a in after) + 4 * moved), "flops": 0}
    if case["kind"] == "append":
        size = 4 if case["dtype"] == "float32" else 2
        pages = sum(-(-a // page) - h // page for h, a in zip(held, after))
        # keys and values read, written as bytes with the scales, the pages read as bytes and written as fp16
        return {"bytes": 2 * heads * (total * dim * (size + 1) + pages * (page * dim * 3 + 8)), "flops": 0}
    seen = pairs = 0
    for h, c in zip(held, new):
        first = max(0, h - case["window"] + 1) if case["window"] else 0
        seen += h + c - first
        if case["window"]:
            pairs += sum(min(case["window"], p + 1) for p in range(h, h + c))
        else:
            pairs += c * h + c * (c + 1) // 2
    return {"bytes": 2 * heads * seen * dim + total * case["q_heads"] * (dim * 4 + 4), "flops": 4 * dim * case["q_heads"] * pairs}


def _values(gen, tokens, case, gain):
    """Keys or values of `tokens` tokens: of unequal strength from channel to channel and from token to token, as a model's are."""
    shape = (tokens, case["kv_heads"], case["dim"])
    x = torch.randn(shape, generator=gen, device=DEV)
    x *= torch.exp(0.5 * torch.randn((tokens, 1, 1), generator=gen, device=DEV))
    return (x * gain).to(getattr(torch, case["dtype"]))


def _inputs(case, seed):
    """What the model gives: for each of two earlier rounds and the present one the counts, keys and values, and the present
    queries; the requests' rows; the pages that another request holds."""
    held, new = _sizes(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    first = [int(0.6 * h) for h in held]
    rounds = [first, [h - f for h, f in zip(held, first)], new]
    gains = [torch.exp(s * torch.randn((1, case["kv_heads"], case["dim"]), generator=gen, device=DEV)) for s in (0.4, 0.2)]
    kv = None
    if case["kind"] != "plan":
        kv = [tuple(_values(gen, sum(r) + (case["pad"] if r is new else 0), case, g) for g in gains) for r in rounds]
    q = None
    if case["kind"] == "attend":
        q = torch.randn((sum(new) + case["pad"], case["q_heads"], case["dim"]), generator=gen, device=DEV).half()
    order = list(range(len(held)))
    rng = random.Random(seed)
    rng.shuffle(order)                       # the requests' rows in the tables
    return rounds, kv, q, order, rng.randrange(OTHERS)


# ---- the plain form ---------------------------------------------------------------------------------------------------

def _plain_plan(s, counts, total, padded):
    """Counts of new tokens (a tensor) to starts, lengths, slots, positions and tables; s holds lengths, tables and the free stack."""
    page, rows = s["page"], s["rows"]
    old = s["lengths"][rows]
    new = old + counts
    before, after = (old + page - 1) // page, (new + page - 1) // page
    base = torch.cumsum(after - before, 0) - (after - before)
    column = torch.arange(s["tables"].shape[1], device=DEV)[None]
    mine = s["tables"][rows]
    fresh = (column >= before[:, None]) & (column < after[:, None])
    place = s["free"] - 1 - (base[:, None] + column - before[:, None])
    mine = torch.where(fresh, s["stack"][place.clamp(0, s["stack"].shape[0] - 1)], mine)
    s["tables"][rows] = mine
    s["free"] = s["free"] - (after - before).sum()
    s["lengths"][rows] = new
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), torch.cumsum(counts, 0)])
    request = torch.repeat_interleave(torch.arange(len(counts), device=DEV), counts, output_size=total)
    j = torch.arange(total, device=DEV) - starts[request]
    position = old[request] + j
    slot = mine[request, position // page] * page + position % page
    slots = torch.full((padded,), -1, dtype=torch.long, device=DEV)
    positions = torch.zeros(padded, dtype=torch.long, device=DEV)
    slots[:total], positions[:total] = slot, position
    tables = torch.where(column < after[:, None], mine, -1)
    return {"starts": starts, "lengths": new, "slots": slots, "positions": positions, "tables": tables, "request": request, "j": j}


def _plain_truncate(s, lengths):
    """Pages beyond `lengths` go back to the stack, so that the next plan takes them in the same order."""
    page, rows = s["page"], s["rows"]
    old = s["lengths"][rows]
    keep, had = (lengths + page - 1) // page, (old + page - 1) // page
    freed = had - keep
    base, total = torch.cumsum(freed, 0) - freed, freed.sum()
    column = torch.arange(s["tables"].shape[1], device=DEV)[None]
    gone = (column >= keep[:, None]) & (column < had[:, None])
    place = torch.where(gone, s["free"] + total - 1 - (base[:, None] + column - keep[:, None]), s["stack"].shape[0])
    padded = torch.cat([s["stack"], s["stack"][:1]])
    s["stack"] = padded.scatter(0, place.reshape(-1), s["tables"][rows].reshape(-1))[:-1]
    s["free"] = s["free"] + total
    s["lengths"][rows] = lengths


def _plain_scale(top):
    """The power of two for a largest magnitude."""
    m, x = torch.frexp(top)
    e = torch.where(m * 128 < 127.5, x - 7, x - 6)
    e = torch.where(top == 0, -100, e).clamp(min=-100)
    return ((e + 127) << 23).view(torch.float32)


def _plain_append(s, x, codes, scales):
    """x [tokens, heads, dim] into codes [pages, page, heads, dim] and scales [pages, heads], at the plan's slots."""
    pages, piece, first, slots = s["pages"], s["piece"], s["first"], s["slots"]
    x = x[:slots.shape[0]].float()
    top = torch.zeros((pages.shape[0], x.shape[1]), device=DEV).index_reduce_(0, piece, x.abs().amax(-1), "amax")
    held = scales[pages]
    scale = torch.where(first[:, None] == 0, _plain_scale(top), torch.maximum(held, _plain_scale(top)))
    old = codes[pages]
    older = (torch.arange(s["page"], device=DEV)[None] < first[:, None])[:, :, None, None]
    again = torch.round(old.float() * (held / scale)[:, None, :, None]).to(torch.int8)
    codes[pages] = torch.where(older, again, old)
    codes[pages[piece], slots % s["page"]] = torch.round(x / scale[piece][:, :, None]).to(torch.int8)
    scales[pages] = scale


def _plain_pieces(s, plan, total):
    """Which pages the plan's tokens go to, which of them each token, and what older tokens each page holds."""
    s["slots"] = plan["slots"][:total]
    s["pages"], s["piece"] = torch.unique_consecutive(s["slots"] // s["page"], return_inverse=True)
    s["first"] = torch.full(s["pages"].shape, s["page"], device=DEV).index_reduce_(0, s["piece"], s["slots"] % s["page"], "amin")


def _plain_attend(s):
    plan, q, page = s["plan"], s["q"], s["page"]
    n, heads, dim = plan["lengths"].shape[0], s["k"].shape[2], q.shape[2]
    group = q.shape[1] // heads
    tables = plan["tables"].clamp(min=0)
    tokens = tables.shape[1] * page
    k = (s["k"][tables].float() * s["k_scale"][tables][:, :, None, :, None]).reshape(n, tokens, heads, dim)
    v = (s["v"][tables].float() * s["v_scale"][tables][:, :, None, :, None]).reshape(n, tokens, heads, dim)
    most = s["most"]
    j = torch.arange(most, device=DEV)[None]
    rows = (plan["starts"][:-1, None] + j).clamp(max=q.shape[0] - 1)
    x = q[rows].float().reshape(n, most, heads, group, dim).permute(0, 2, 1, 3, 4).reshape(n, heads, most * group, dim)
    scores = torch.matmul(x, k.permute(0, 2, 3, 1)) * (1 / math.sqrt(dim))
    position = (plan["lengths"] - (plan["starts"][1:] - plan["starts"][:-1]))[:, None] + j
    t = torch.arange(tokens, device=DEV)
    seen = t[None, None] <= position[:, :, None]
    if s["window"]:
        seen &= t[None, None] > position[:, :, None] - s["window"]
    scores = scores.reshape(n, heads, most, group, tokens).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp_(scores.sub_(top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.reshape(n, heads, most * group, tokens), v.transpose(1, 2)).reshape(n, heads, most, group, dim) / total
    lse = (top + torch.log(total))[..., 0]
    result, sums = torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV)
    live = plan["request"].shape[0]
    result[:live] = out.permute(0, 2, 1, 3, 4).reshape(n, most, heads * group, dim)[plan["request"], plan["j"]].half()
    sums[:live] = lse.permute(0, 2, 1, 3).reshape(n, most, heads * group)[plan["request"], plan["j"]]
    return result, sums


# ---- both -------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    rounds, kv, q, order, others = _inputs(case, seed)
    held, new = _sizes(case)
    page, n, kind = case["page"], case["requests"], case["kind"]
    width = max(-(-(h + c) // page) for h, c in zip(held, new))
    num_pages = others + sum(-(-(h + c) // page) for h, c in zip(held, new)) + 7
    heads, dim = (1, 64) if kind == "plan" else (case["kv_heads"], case["dim"])
    rows = torch.tensor(order, device=DEV)
    padded = sum(new) + case["pad"]
    s = {"kind": kind, "window": case["window"], "counts": torch.tensor(new, device=DEV), "total": sum(new), "padded": padded,
         "most": max(new), "held": torch.tensor(held, device=DEV), "page": page}
    if own:
        import turboquant_mlx_core_b200 as tq
        cache = tq.PagedKVCache(1, heads, dim, num_pages, page, max_requests=n + 1, max_pages_per_request=max(width, others),
                                max_tokens=max(padded, others * page, *(sum(r) for r in rounds)))
        cache.plan(torch.tensor([others * page], device=DEV).int(), others * page, others * page, rows=torch.tensor([n], device=DEV).int())
        s |= {"cache": cache, "rows": rows.int(), "counts": s["counts"].int(), "held": s["held"].int()}
        for r, counts in enumerate(rounds):
            last = r == 2
            if (last and kind == "plan") or sum(counts) == 0:
                continue
            tokens = padded if last else sum(counts)
            s["slots"] = torch.empty(tokens, dtype=torch.int32, device=DEV)
            cache.plan(torch.tensor(counts, device=DEV).int(), tokens, max(counts), rows=s["rows"], slots=s["slots"])
            if kv is not None and not (last and kind == "append"):
                cache.append(0, *kv[r])
        if kind == "append":
            s["pages"] = torch.unique_consecutive(s["slots"][:s["total"]] // page).int()
            s["values"] = [torch.empty((s["pages"].shape[0], page, heads, dim), dtype=torch.float16, device=DEV) for _ in range(2)]
    else:
        s |= {"rows": rows, "lengths": torch.zeros(n, dtype=torch.long, device=DEV), "tables": torch.full((n, width), -1, device=DEV),
              "stack": torch.arange(num_pages - 1, -1, -1, device=DEV), "free": torch.tensor(num_pages - others, device=DEV)}
        for c in () if kind == "plan" else ("k", "v"):
            s[c] = torch.zeros((num_pages, page, heads, dim), dtype=torch.int8, device=DEV)
            s[c + "_scale"] = torch.full((num_pages, heads), 2.0 ** -100, device=DEV)
        for r, counts in enumerate(rounds):
            last = r == 2
            if (last and kind == "plan") or sum(counts) == 0:
                continue
            s["plan"] = _plain_plan(s, torch.tensor(counts, device=DEV), sum(counts), padded if last else sum(counts))
            _plain_pieces(s, s["plan"], sum(counts))
            if kv is not None and not (last and kind == "append"):
                _plain_append(s, kv[r][0], s["k"], s["k_scale"])
                _plain_append(s, kv[r][1], s["v"], s["v_scale"])
    if kind == "append":
        s["new_k"], s["new_v"] = kv[2]
    elif kind == "attend":
        s["q"] = q
        s["out"] = torch.zeros_like(q)
        s["lse"] = torch.zeros(q.shape[:2], device=DEV)
    else:
        ints = {"dtype": torch.int32, "device": DEV}
        s["outputs"] = {"starts": torch.empty(n + 1, **ints), "lengths": torch.empty(n, **ints), "slots": torch.empty(padded, **ints),
                        "positions": torch.empty(padded, **ints), "tables": torch.empty((n, width), **ints)}
    return s


def run(s):
    if s["kind"] == "plan":
        if own:
            s["cache"].plan(s["counts"], s["padded"], s["most"], rows=s["rows"], **s["outputs"])
            s["cache"].truncate(s["held"], rows=s["rows"])
            return s["outputs"]
        plan = _plain_plan(s, s["counts"], s["total"], s["padded"])
        _plain_truncate(s, s["held"])
        return {name: plan[name].int() for name in s["outputs"]}
    if s["kind"] == "append":
        if own:
            s["cache"].append(0, s["new_k"], s["new_v"])
            s["cache"].read_pages(0, s["pages"], *s["values"])
            return s["values"]
        _plain_append(s, s["new_k"], s["k"], s["k_scale"])
        _plain_append(s, s["new_v"], s["v"], s["v_scale"])
        return [(s[c][s["pages"]].float() * s[c + "_scale"][s["pages"]][:, None, :, None]).half() for c in ("k", "v")]
    if own:
        s["cache"].attention(0, s["q"], window=s["window"], out=s["out"], lse=s["lse"])
        return s["out"], s["lse"]
    return _plain_attend(s)


def exact(case, seed):
    """The definitions in 64 bits, request by request."""
    rounds, kv, q, _, others = _inputs(case, seed)
    held, new = _sizes(case)
    page, n = case["page"], len(held)
    up = lambda a: -(-a // page)                                                        # noqa: E731

    # pages are handed out in order, round by round
    tables, length, next_page = [[] for _ in range(n)], [0] * n, others
    for counts in rounds:
        for i in range(n):
            length[i] += counts[i]
            more = up(length[i]) - len(tables[i])
            tables[i] += range(next_page, next_page + more)
            next_page += more
    if case["kind"] == "plan":
        starts, slots, positions = [0], [], []
        for i in range(n):
            starts.append(starts[-1] + new[i])
            positions += range(held[i], held[i] + new[i])
        for i in range(n):
            slots += [tables[i][p // page] * page + p % page for p in range(held[i], held[i] + new[i])]
        width = max(map(len, tables))
        slots, positions = slots + [-1] * case["pad"], positions + [0] * case["pad"]
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)                 # noqa: E731
        return {"starts": ints(starts), "lengths": ints(length), "slots": ints(slots), "positions": ints(positions),
                "tables": ints([t + [-1] * (width - len(t)) for t in tables])}

    def power(e):
        """2^e by its bits: a library's power need not be exact."""
        return ((e + 1023) << 52).view(torch.float64)

    def exponent(top):
        """The smallest e with which top / 2^e rounds to 127 at most."""
        e = torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 127.5))
        e = torch.clamp(e, -900, 900).long()
        e = torch.where(top * power(-e) >= 127.5, e + 1, e)
        e = torch.where(top * power(1 - e) < 127.5, e - 1, e)
        return torch.clamp(e, min=-100)

    def stored(i, which):
        """Request i's keys or values as the cache holds them after the rounds: [pages, page, heads, dim]."""
        parts, at = [], 0
        for r, counts in enumerate(rounds):
            at = sum(counts[:i])
            parts.append(kv[r][which][at:at + counts[i]].double())
        x = torch.cat(parts)
        x = torch.cat([x, x.new_zeros((up(length[i]) * page - length[i], *x.shape[1:]))]).reshape(-1, page, *x.shape[1:])
        t = torch.arange(x.shape[0] * page, device=DEV).reshape(-1, page)
        codes, e, begin = torch.zeros_like(x), torch.full((x.shape[0], x.shape[2]), -100, device=DEV), 0
        for counts in rounds:
            end = begin + counts[i]
            if end > begin:
                now = (t >= begin) & (t < end)
                touched = now.any(1)
                joined = touched & (t[:, 0] < begin)
                mine = exponent((x.abs() * now[:, :, None, None]).amax((1, 3)))
                e1 = torch.where(joined[:, None], torch.maximum(e, mine), torch.where(touched[:, None], mine, e))
                codes = torch.where((t < begin)[:, :, None, None], torch.round(codes * power(e - e1)[:, None, :, None]), codes)
                codes = torch.where(now[:, :, None, None], torch.round(x * power(-e1)[:, None, :, None]), codes)
                e = e1
            begin = end
        return codes * power(e)[:, None, :, None]

    if case["kind"] == "append":
        return [torch.cat([stored(i, which)[held[i] // page:] for i in range(n)]) for which in (0, 1)]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    group, row = case["q_heads"] // case["kv_heads"], 0
    for i in range(n):
        k, v = (stored(i, which).flatten(0, 1)[:length[i]] for which in (0, 1))
        for begin in range(0, new[i], 512):
            end = min(new[i], begin + 512)
            p = torch.arange(held[i] + begin, held[i] + end, device=DEV)[:, None]
            t = torch.arange(length[i], device=DEV)[None]
            hidden = (t > p) | ((t <= p - case["window"]) if case["window"] else torch.zeros_like(t > p))
            for h in range(case["q_heads"]):
                s = q[row + begin:row + end, h].double() @ k[:, h // group].T / math.sqrt(case["dim"])
                s[hidden] = -math.inf
                lse[row + begin:row + end, h] = torch.logsumexp(s, 1)
                out[row + begin:row + end, h] = torch.softmax(s, 1) @ v[:, h // group]
        row += new[i]
    return out, lse
