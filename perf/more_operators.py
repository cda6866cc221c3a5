"""Operators of a cache whose pages are shared, moved and read in part, as cases to be timed.

Requests that fork from one prompt share its pages: copying gives a child its own
exact pages (``copy``), compaction moves the pages in use to the front of the pool
(``compact``), and attention reads a shared prefix once for all requests
(``prefix``).  Over a long history a token attends to the pages that bounds of
their keys pick out for it (``sparse``), and the bounds are taken from the key
codes as pages are completed (``bounds``).  Shapes are those of the package's own
configurations (32 query heads, 8 KV heads, head_dim 128, 16-token pages, exact
sidecars of prefix, suffix and ring pages) and the ranges around them.

``run`` computes an operator in plain torch, or where ``own`` is set calls the
package's.

INT8 pages: codes [pages, 16, Hkv, 128] and one FP16 scale per page and KV head,
K and V apart.  A value is code * scale; the V center of a request is added to
its output.
"""

import math
import random

import torch

own = False

DIM, PAGE = 128, 16
WORKSPACE_BYTES = 512 << 20
NO_PAGE = -1


def listed():
    return [
        # eight beams part after a token: each copies the one page that it goes on
        # writing, exact K and V of one layer: latency counts
        {"name": "copy_beams", "op": "copy", "layers": 1, "pool_pages": 96, "copies": 8, "kv_heads": 8},
        # a request forked into three: its sidecar of 180 exact pages (4 of the
        # prompt's start, 128 of its end, a ring of 48), K and V of 8 layers
        {"name": "copy_sidecars", "op": "copy", "layers": 8, "pool_pages": 720, "copies": 540, "kv_heads": 8},
        # a small pool after a few requests have left, one table of pages in use
        {"name": "compact_1k", "op": "compact", "pool_pages": 1021, "live": 0.8, "kv_heads": 8},
        # a serving pool half in use, its pages scattered by requests that came and went
        {"name": "compact_16k", "op": "compact", "pool_pages": 16384, "live": 0.5, "kv_heads": 8},
        # four samples of one short prompt, just started
        {"name": "prefix_b4", "op": "prefix", "kind": "int8", "requests": 4, "groups": 1, "common": 0,
         "prefix_low": 2000, "prefix_high": 2000, "own_low": 0, "own_high": 0, "tail_low": 17, "tail_high": 90,
         "q_heads": 32, "kv_heads": 8},
        # sixty requests of several prompts under one common instruction, uneven,
        # eight query heads per KV head, FP16 pages
        {"name": "prefix_uneven", "op": "prefix", "kind": "fp16", "requests": 61, "groups": 7, "common": 1531,
         "prefix_low": 37, "prefix_high": 6000, "own_low": 0, "own_high": 900, "tail_low": 1, "tail_high": 16,
         "q_heads": 32, "kv_heads": 4},
        # a full batch over one long document, each with its own turn and exact tail
        {"name": "prefix_b256", "op": "prefix", "kind": "int8", "requests": 256, "groups": 1, "common": 0,
         "prefix_low": 16384, "prefix_high": 16384, "own_low": 100, "own_high": 1000, "tail_low": 241,
         "tail_high": 256, "q_heads": 32, "kv_heads": 8},
        # the page that each of 32 requests completed in this step
        {"name": "bounds_step", "op": "bounds", "pool_pages": 4096, "pages": 32, "ragged": False, "kv_heads": 8},
        # a long prompt's pages after its prefill, the last one partial
        {"name": "bounds_prompt", "op": "bounds", "pool_pages": 8200, "pages": 8191, "ragged": True, "kv_heads": 8},
        # one request, 32K tokens, the best 64 pages of each KV head
        {"name": "sparse_b1", "op": "sparse", "requests": 1, "low": 32768, "high": 32768, "pages": 64, "first": 1,
         "last": 2, "tail_low": 250, "tail_high": 250, "q_heads": 32, "kv_heads": 8},
        # uneven requests of a serving batch, some shorter than what is picked
        {"name": "sparse_uneven", "op": "sparse", "requests": 45, "low": 500, "high": 30000, "pages": 96,
         "first": 2, "last": 0, "tail_low": 1, "tail_high": 256, "q_heads": 28, "kv_heads": 4},
        # eight requests of 128K tokens, 4096 tokens read for each
        {"name": "sparse_b8", "op": "sparse", "requests": 8, "low": 131072, "high": 131072, "pages": 256,
         "first": 4, "last": 4, "tail_low": 256, "tail_high": 256, "q_heads": 32, "kv_heads": 8},
    ]


def draw(rng):
    def spread(low, high):               # evenly over the logarithm
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    def sorted_pair(low, high):
        return sorted((spread(low, high), spread(low, high)))

    op = rng.choice(("copy", "compact", "prefix", "prefix", "bounds", "sparse", "sparse"))
    kv_heads = rng.choice((1, 2, 4, 8))
    if op == "copy":
        layers = rng.randint(1, 8)
        copies = spread(1, 500)
        return {"op": op, "layers": layers, "pool_pages": copies + rng.randint(1, 220), "copies": copies,
                "kv_heads": kv_heads}
    if op == "compact":
        return {"op": op, "pool_pages": spread(64, 16000), "live": round(rng.uniform(0.02, 0.99), 3),
                "kv_heads": kv_heads}
    if op == "bounds":
        pages = spread(1, 8000)
        return {"op": op, "pool_pages": pages + rng.randint(0, 200), "pages": pages,
                "ragged": rng.random() < 0.5, "kv_heads": kv_heads}
    tail = sorted((rng.randint(1, 256), rng.randint(1, 256)))
    q_heads = kv_heads * rng.choice((1, 2, 4, 4, 5, 7, 8, 16) if kv_heads < 8 else (1, 2, 4))
    if op == "prefix":
        requests = spread(1, 200)
        prefix, private = sorted_pair(16, 12000), sorted_pair(1, 900)
        return {"op": op, "kind": rng.choice(("int8", "int8", "fp16")), "requests": requests,
                "groups": min(requests, rng.choice((1, 1, 2, 3, 9))), "common": rng.choice((0, 0, rng.randint(1, 4000))),
                "prefix_low": prefix[0], "prefix_high": prefix[1], "own_low": private[0] - 1,
                "own_high": private[1] - 1, "tail_low": tail[0], "tail_high": tail[1], "q_heads": q_heads,
                "kv_heads": kv_heads}
    requests = spread(1, 48)
    tokens = sorted_pair(16, min(131072, 1000000 // requests))
    first, last = rng.choice((0, 1, 4)), rng.choice((0, 1, 4))
    return {"op": op, "requests": requests, "low": tokens[0], "high": tokens[1],
            "pages": max(spread(8, 256), first + last), "first": first, "last": last, "tail_low": tail[0],
            "tail_high": tail[1], "q_heads": q_heads, "kv_heads": kv_heads}


# ---------------------------------------------------------------------------
# Sizes of a case
# ---------------------------------------------------------------------------

def _between(low, high, count):
    """``count`` whole numbers in [low, high], uneven: the golden ratio's multiples."""
    return [low + int((high - low + 1) * ((i + 1) * 0.6180339887498949 % 1.0)) for i in range(count)] \
        if high > low else [low] * count


def _pages_of(tokens):
    return -(-tokens // PAGE)


def _segments(case):
    """(first request, end request, tokens) of the prefixes of a case."""
    requests, groups = case["requests"], case["groups"]
    cuts = [0]
    for g, w in enumerate(_between(1, 5, groups)):       # uneven groups, none empty
        left = requests - cuts[-1] - (groups - g - 1)
        cuts.append(requests if g == groups - 1 else cuts[-1] + max(1, min(left, w * requests // (3 * groups))))
    found = [(0, requests, case["common"])] if case["common"] else []
    lengths = _between(case["prefix_low"], case["prefix_high"], groups)
    return found + [(cuts[g], cuts[g + 1], lengths[g]) for g in range(groups)]


def work(case):
    op, heads = case["op"], case["kv_heads"]
    if op == "copy":
        return {"bytes": 2 * case["layers"] * case["copies"] * 2 * PAGE * heads * DIM * 2, "flops": 0}
    if op == "compact":
        live = _live_pages(case)
        count, limit = sum(live), case["pool_pages"]
        moved = sum(live[count:])
        page = 2 * heads * (PAGE * DIM + 2)
        return {"bytes": 2 * moved * page + 8 * limit + 2 * 4 * (limit // 2) + 2 * 4 * count, "flops": 0}
    if op == "bounds":
        return {"bytes": case["pages"] * heads * (PAGE * DIM + 2 * DIM), "flops": 0}
    requests, hq = case["requests"], case["q_heads"]
    tail = sum(_between(case["tail_low"], case["tail_high"], requests))
    exact_token, rows = 2 * heads * DIM * 2, requests * hq
    ends = requests * heads * DIM * 2 + rows * (2 * DIM * 2 + 4)       # centers; queries, outputs, lse
    if op == "prefix":
        token = heads * 2 * (DIM + 2 / PAGE) if case["kind"] == "int8" else exact_token
        held, scores = 0, 0
        for begin, end, tokens in _segments(case):
            held, scores = held + tokens, scores + (end - begin) * tokens
        private = sum(_between(case["own_low"], case["own_high"], requests))
        return {"bytes": int((held + private) * token) + tail * exact_token + ends,
                "flops": 4 * DIM * hq * (scores + private + tail)}
    lengths = _between(case["low"], case["high"], requests)
    pages = sum(_pages_of(n) for n in lengths)
    read = sum(min(_pages_of(n), case["pages"]) for n in lengths)
    return {"bytes": pages * heads * 2 * DIM + read * heads * 2 * (PAGE * DIM + 2) + tail * exact_token + ends
            + requests * heads * case["pages"] * 4,
            "flops": 4 * DIM * hq * pages + 4 * DIM * hq * (read * PAGE + tail)}


def _live_pages(case):
    """Which pages are in use: a fixed scatter of about ``live`` of them."""
    rng = random.Random(case["pool_pages"] * 1000 + int(case["live"] * 1000))
    return [int(rng.random() < case["live"]) for _ in range(case["pool_pages"])]


# ---------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------

def _codes(gen, pages, heads, spread):
    """Bell-shaped codes, with a part that a page's tokens share."""
    shape = (pages, PAGE, heads, DIM)
    draw8 = lambda size, top: torch.randint(-top, top + 1, size, generator=gen, device="cuda",  # noqa: E731
                                            dtype=torch.int8)
    codes = draw8((pages, 1, heads, DIM), spread).expand(shape).contiguous()
    top = (127 - spread) // 2
    for _ in range(2):
        codes += draw8(shape, top)
    return codes


def _scales(gen, pages, heads):
    return (torch.rand(pages, heads, generator=gen, device="cuda") * 0.02 + 0.01).half()


def _normal(gen, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).half()


def _shuffled(gen, count):
    return torch.randperm(count, generator=gen, device="cuda").int()


def _table(lengths):
    """(indptr, last page lengths) of token counts, on the host."""
    indptr = [0]
    for n in lengths:
        indptr.append(indptr[-1] + _pages_of(n))
    last = [(n - 1) % PAGE + 1 if n else 0 for n in lengths]
    return torch.tensor(indptr, dtype=torch.int32), torch.tensor(last, dtype=torch.int32)


def prepare(case, seed):
    """The inputs, and the handle that a program keeps."""
    state = _inputs(case, seed)
    if own and case["op"] == "compact":
        from pagegauge_amd import pages
        state["pool"] = pages.PagePool(case["pool_pages"], device="cuda")
        state["pool"].refs.copy_(state["refs"])
    if own and case["op"] in ("prefix", "sparse"):
        workspace = torch.empty(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
        own_table = state["indptr"], state["ids"], state["last"]
        tail_table = state["tail_indptr"], state["tail_ids"], state["tail_last"]
        heads = {"num_qo_heads": case["q_heads"], "num_kv_heads": case["kv_heads"]}
        if case["op"] == "prefix":
            from pagegauge_amd import prefix
            state["decode"] = prefix.SharedPrefixDecode(workspace)
            state["decode"].plan(state["segments"], state["prefix_indptr"], state["prefix_ids"],
                                 state["prefix_last"], *own_table, *tail_table, **heads,
                                 kv_data_type=torch.int8 if case["kind"] == "int8" else torch.float16)
        else:
            from pagegauge_amd import sparse
            state["decode"] = sparse.SelectedPagesDecode(workspace)
            state["decode"].plan(*own_table, *tail_table, **heads, pages=case["pages"],
                                 first_pages=case["first"], last_pages=case["last"])
    return state


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, heads = case["op"], case["kv_heads"]
    state = {"case": case}
    if op == "copy":
        shape = (case["layers"], case["pool_pages"], PAGE, heads, DIM)
        state["key"], state["value"] = _normal(gen, *shape), _normal(gen, *shape)
        order = _shuffled(gen, case["pool_pages"])
        spare = case["pool_pages"] - case["copies"]          # sources, copied several times where few
        state["target"] = order[spare:].contiguous()
        state["source"] = order[torch.arange(case["copies"], device="cuda") % spare].contiguous()
        return state
    if op == "compact":
        pages = case["pool_pages"]
        state["key"], state["value"] = _codes(gen, pages, heads, 40), _codes(gen, pages, heads, 20)
        state["key_scale"], state["value_scale"] = _scales(gen, pages, heads), _scales(gen, pages, heads)
        live = torch.tensor(_live_pages(case), dtype=torch.int32, device="cuda")
        # a page is used by one request or shared by a few
        refs = live * (1 + (torch.rand(pages, generator=gen, device="cuda") < 0.2).int() * 3)
        ids = live.nonzero().flatten().int()
        state["table"] = ids[torch.randperm(len(ids), generator=gen, device="cuda")].contiguous()
        state["refs"] = refs
        return state
    if op == "bounds":
        pool, pages = case["pool_pages"], case["pages"]
        state["key"] = _codes(gen, pool, heads, 40)
        state["ids"] = _shuffled(gen, pool)[:pages].contiguous()
        lengths = torch.full((pages,), PAGE, dtype=torch.int32, device="cuda")
        if case["ragged"]:
            lengths[-1:] = torch.randint(1, PAGE, (1,), generator=gen, device="cuda").int()
        state["lengths"] = lengths
        state["bounds"] = torch.zeros(pool, heads, 2, DIM, dtype=torch.int8, device="cuda")
        return state

    requests, hq = case["requests"], case["q_heads"]
    state["q"] = _normal(gen, requests, hq, DIM, scale=1.5)
    state["center"] = _normal(gen, requests, heads, DIM, scale=0.3)
    tails = _between(case["tail_low"], case["tail_high"], requests)
    state["tail_indptr"], tail_last = _table(tails)
    state["tail_last"] = tail_last.cuda()
    exact = int(state["tail_indptr"][-1])
    state["tail_ids"] = _shuffled(gen, exact)
    state["exact"] = _normal(gen, exact, PAGE, heads, DIM), _normal(gen, exact, PAGE, heads, DIM)
    if op == "prefix":
        segments = _segments(case)
        state["segments"] = torch.tensor([s[:2] for s in segments], dtype=torch.int32)
        state["prefix_indptr"], prefix_last = _table([s[2] for s in segments])
        state["indptr"], last = _table(_between(case["own_low"], case["own_high"], requests))
        state["prefix_last"], state["last"] = prefix_last.cuda(), last.cuda()
        shared = int(state["prefix_indptr"][-1])
        pool = shared + int(state["indptr"][-1])
        order = _shuffled(gen, pool)
        state["prefix_ids"], state["ids"] = order[:shared].contiguous(), order[shared:].contiguous()
    else:
        state["indptr"], last = _table(_between(case["low"], case["high"], requests))
        state["last"] = last.cuda()
        pool = int(state["indptr"][-1])
        state["ids"] = _shuffled(gen, pool)
    if op == "prefix" and case["kind"] == "fp16":
        state["cache"] = _normal(gen, pool, PAGE, heads, DIM, scale=0.7), _normal(gen, pool, PAGE, heads, DIM)
        state["scales"] = None, None
    else:
        state["cache"] = _codes(gen, pool, heads, 40), _codes(gen, pool, heads, 20)
        state["scales"] = _scales(gen, pool, heads), _scales(gen, pool, heads)
    if op == "sparse":
        state["bounds"] = torch.stack((state["cache"][0].amin(1), state["cache"][0].amax(1)), dim=2)
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    return (_own if own else _plain)[op](state)


def _own_copy(s):
    from pagegauge_amd import pages
    pages.copy_pages((s["key"], s["value"]), s["source"], s["target"], page_dim=1)
    return s["key"], s["value"]


def _own_compact(s):
    from pagegauge_amd import pages
    moves = s["pool"].stage_compaction()
    planes = s["key"], s["value"], s["key_scale"], s["value_scale"]
    pages.copy_pages(planes, moves.source, moves.target)
    table = pages.rewrite_ids(s["table"], moves.remap)
    return (*planes, moves.source, moves.target, moves.remap, moves.live, table)


def _own_prefix(s):
    return s["decode"].run(s["q"], s["cache"], *s["scales"], s["exact"], value_center=s["center"], return_lse=True)


def _own_bounds(s):
    from pagegauge_amd import sparse
    sparse.key_bounds(s["key"], s["bounds"], page_ids=s["ids"], lengths=s["lengths"])
    return s["bounds"]


def _own_sparse(s):
    selected = s["decode"].select(s["q"], s["bounds"], s["scales"][0])
    out, lse = s["decode"].run(s["q"], s["cache"], *s["scales"], selected, s["exact"], value_center=s["center"],
                               return_lse=True)
    return selected, out, lse


_own = {"copy": _own_copy, "compact": _own_compact, "prefix": _own_prefix, "bounds": _own_bounds,
        "sparse": _own_sparse}


def _plain_copy(s):
    source, target = s["source"].long(), s["target"].long()
    for plane in (s["key"], s["value"]):
        plane[:, target] = plane[:, source]
    return s["key"], s["value"]


def _plain_compact(s):
    live = s["refs"] > 0
    pages = live.numel()
    count = live.sum()
    page = torch.arange(pages, device="cuda")
    holes = (~live & (page < count)).nonzero().flatten()
    movers = (live & (page >= count)).nonzero().flatten()
    remap = torch.where(live, page, NO_PAGE)
    remap[movers] = holes
    planes = s["key"], s["value"], s["key_scale"], s["value_scale"]
    for plane in planes:
        plane[holes] = plane[movers]
    lists = torch.full((2, pages // 2), NO_PAGE, device="cuda")
    lists[0, :len(movers)], lists[1, :len(holes)] = movers, holes
    return (*planes, lists[0].int(), lists[1].int(), remap.int(), count.int().view(1),
            remap[s["table"].long()].int())


class _Sums:
    """Softmax sums of query rows [B, Hkv, G, 128] as tokens come in, base 2."""

    def __init__(self, q, heads):
        batch, hq, _ = q.shape
        self.q = q.float().view(batch, heads, hq // heads, DIM)
        shape = self.q.shape[:3] + (1,)
        self.top = torch.full(shape, -math.inf, device="cuda")
        self.total = torch.zeros(shape, device="cuda")
        self.out = torch.zeros_like(self.q)

    def add(self, begin, end, k, v, mask):
        """Rows of requests ``begin`` .. ``end`` see k, v [N or 1, Hkv, T, 128] where mask [N or 1, 1 or Hkv, 1, T]."""
        q = self.q[begin:end]
        if k.shape[0] == 1 and len(q) > 1:               # shared keys: rows of all requests in one product
            n, heads, group, _ = q.shape
            flat = q.transpose(0, 1).reshape(1, heads, n * group, DIM)
            score = (flat @ k.transpose(-1, -2)) * (DIM ** -0.5 * math.log2(math.e))
            score = torch.where(mask, score, -math.inf)
            top = score.amax(-1, keepdim=True)
            p = torch.exp2(score - torch.where(top == -math.inf, 0.0, top))
            parts = (top, p.sum(-1, keepdim=True), p @ v)
            top, total, out = (t.view(heads, n, group, -1).transpose(0, 1) for t in parts)
        else:
            score = (q @ k.transpose(-1, -2)) * (DIM ** -0.5 * math.log2(math.e))
            score = torch.where(mask, score, -math.inf)
            top = score.amax(-1, keepdim=True)
            p = torch.exp2(score - torch.where(top == -math.inf, 0.0, top))
            total, out = p.sum(-1, keepdim=True), p @ v
        old = self.top[begin:end]
        new = torch.maximum(old, top)
        base = torch.where(new == -math.inf, 0.0, new)
        a, b = torch.exp2(old - base), torch.exp2(top - base)
        self.total[begin:end] = self.total[begin:end] * a + total * b
        self.out[begin:end] = self.out[begin:end] * a + out * b
        self.top[begin:end] = new

    def finish(self, center):
        out = self.out / torch.where(self.total == 0, 1.0, self.total) + center.float().unsqueeze(2)
        lse = (torch.log2(self.total) + self.top).flatten(1)
        return out.half().flatten(1, 2), lse


def _values(cache, scale, ids):
    """float32 [..., T, Hkv, 128] of pages ids [..., P]."""
    x = cache[ids].float()
    if scale is not None:
        x = x * scale[ids].float()[..., None, :, None]
    return x.flatten(-4, -3)


def _add_padded(sums, cache, scales, indptr, ids, last):
    """Each request's own pages, padded to the longest; a few requests at a time."""
    indptr = indptr.cuda()
    counts = indptr[1:] - indptr[:-1]
    most = int(counts.max())
    if most == 0:
        return
    page = torch.arange(most, device="cuda")
    table = ids.long()[(indptr[:-1, None] + page).clamp(max=len(ids) - 1)]
    tokens = torch.where(counts > 0, (counts - 1) * PAGE + last, 0)
    mask = torch.arange(most * PAGE, device="cuda") < tokens[:, None]
    step = max(1, (1 << 22) // (most * PAGE * cache[0].shape[2]))
    for b in range(0, len(counts), step):
        part = slice(b, b + step)
        k = _values(cache[0], scales[0], table[part]).transpose(1, 2)
        v = _values(cache[1], scales[1], table[part]).transpose(1, 2)
        sums.add(b, min(b + step, len(counts)), k, v, mask[part, None, None])


def _plain_prefix(s):
    sums = _Sums(s["q"], s["case"]["kv_heads"])
    for i, (begin, end) in enumerate(s["segments"].tolist()):
        ids = s["prefix_ids"][int(s["prefix_indptr"][i]):int(s["prefix_indptr"][i + 1])].long()
        k, v = (_values(c, scale, ids).transpose(0, 1)[None] for c, scale in zip(s["cache"], s["scales"]))
        tokens = (len(ids) - 1) * PAGE + s["prefix_last"][i]
        sums.add(begin, end, k, v, (torch.arange(k.shape[2], device="cuda") < tokens)[None, None, None])
    _add_padded(sums, s["cache"], s["scales"], s["indptr"], s["ids"], s["last"])
    _add_padded(sums, s["exact"], (None, None), s["tail_indptr"], s["tail_ids"], s["tail_last"])
    return sums.finish(s["center"])


def _plain_bounds(s):
    ids = s["ids"].long()
    codes = s["key"][ids]
    seen = (torch.arange(PAGE, device="cuda") < s["lengths"][:, None])[:, :, None, None]
    s["bounds"][ids, :, 0] = torch.where(seen, codes, 127).amin(1)
    s["bounds"][ids, :, 1] = torch.where(seen, codes, -128).amax(1)
    return s["bounds"]


def _power_of_two(exponent):
    return ((exponent + 127) << 23).view(torch.float32)


def _plain_scores(q, bounds, scale, ids):
    """float32 [Hkv, pages] of one request's q [Hkv, G, 128]."""
    q = q.float()
    _, x = torch.frexp(q.abs().amax(-1, keepdim=True))
    steps = torch.clamp(torch.round(q * _power_of_two(7 - x.int())), -127, 127)
    unit = _power_of_two(x.int() - 7)                          # [Hkv, G, 1]
    b = bounds[ids].float().permute(1, 2, 3, 0)                # [Hkv, 2, 128, pages]
    # whole numbers below 2^22: exact in float32
    total = steps.clamp(min=0) @ b[:, 1] + steps.clamp(max=0) @ b[:, 0]
    return (total * scale[ids].float().t()[:, None] * unit).amax(1)


def _plain_selection(s):
    case, indptr = s["case"], s["indptr"].tolist()
    heads = case["kv_heads"]
    found = torch.full((case["requests"], heads, case["pages"]), NO_PAGE, dtype=torch.int32, device="cuda")
    q = s["q"].view(case["requests"], heads, -1, DIM)
    for b in range(case["requests"]):
        ids = s["ids"][indptr[b]:indptr[b + 1]].long()
        score = _plain_scores(q[b], s["bounds"], s["scales"][0], ids)
        score[:, :case["first"]] = math.inf
        score[:, max(0, len(ids) - case["last"]):] = math.inf
        best = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :case["pages"]]
        found[b, :, :best.shape[1]] = best.sort(dim=1).values.int()
    return found


def _plain_sparse(s):
    case = s["case"]
    heads, requests = case["kv_heads"], case["requests"]
    found = _plain_selection(s)
    sums = _Sums(s["q"], heads)
    indptr = s["indptr"].cuda()
    counts = (indptr[1:] - indptr[:-1])[:, None, None]
    page = s["ids"].long()[(indptr[:-1, None, None] + found.clamp(min=0)).clamp(max=len(s["ids"]) - 1)]
    visible = torch.where(found == counts - 1, s["last"][:, None, None], PAGE)
    visible = torch.where(found < 0, 0, visible)
    mask = torch.arange(PAGE, device="cuda") < visible[..., None]
    head = torch.arange(heads, device="cuda")[:, None]
    step = max(1, (1 << 22) // (heads * PAGE * case["pages"]))
    for b in range(0, requests, step):
        part = slice(b, b + step)
        k, v = ((c[page[part], :, head].float() * scale[page[part], head].float()[..., None, None]).flatten(2, 3)
                for c, scale in zip(s["cache"], s["scales"]))
        sums.add(b, min(b + step, requests), k, v, mask[part].flatten(2)[:, :, None])
    _add_padded(sums, s["exact"], (None, None), s["tail_indptr"], s["tail_ids"], s["tail_last"])
    return (found, *sums.finish(s["center"]))


_plain = {"copy": _plain_copy, "compact": _plain_compact, "prefix": _plain_prefix, "bounds": _plain_bounds,
          "sparse": _plain_sparse}


# ---------------------------------------------------------------------------
# From the definitions, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    """The outputs for these inputs, each request by itself."""
    state = _inputs(case, seed)
    return {"copy": _exact_copy, "compact": _exact_compact, "prefix": _exact_prefix, "bounds": _exact_bounds,
            "sparse": _exact_sparse}[case["op"]](state)


def _exact_copy(s):
    where = list(range(s["case"]["pool_pages"]))             # the page that each one holds afterwards
    for source, target in zip(s["source"].tolist(), s["target"].tolist()):
        where[target] = source
    where = torch.tensor(where, device="cuda")
    return s["key"].index_select(1, where), s["value"].index_select(1, where)


def _exact_compact(s):
    refs = s["refs"].tolist()
    total = sum(r > 0 for r in refs)
    holes = [p for p in range(total) if refs[p] <= 0]
    movers = [p for p in range(total, len(refs)) if refs[p] > 0]
    new = {p: p for p in range(len(refs)) if refs[p] > 0}
    new.update(zip(movers, holes))
    content = list(range(len(refs)))
    for target, source in zip(holes, movers):
        content[target] = source
    content = torch.tensor(content, device="cuda")
    planes = [s[name].index_select(0, content) for name in ("key", "value", "key_scale", "value_scale")]
    whole = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    pad = [NO_PAGE] * (len(refs) // 2 - len(movers))
    return (*planes, whole(movers + pad), whole(holes + pad), whole([new.get(p, NO_PAGE) for p in range(len(refs))]),
            whole([total]), whole([new[p] for p in s["table"].tolist()]))


def _exact_bounds(s):
    for page, n in zip(s["ids"].tolist(), s["lengths"].tolist()):
        low, high = torch.aminmax(s["key"][page, :n], dim=0)
        s["bounds"][page, :, 0], s["bounds"][page, :, 1] = low, high
    return s["bounds"]


def _rows64(cache, scales, ids, tokens, head):
    """K and V float64 [tokens, 128] of a head over pages in order."""
    rows = []
    for c, scale in zip(cache, scales):
        x = c[ids, :, head].double()
        if scale is not None:
            x = x * scale[ids, head].double()[:, None, None]
        rows.append(x.reshape(-1, DIM)[:tokens])
    return rows


def _tokens(indptr, last, i):
    pages = int(indptr[i + 1]) - int(indptr[i])
    return (pages - 1) * PAGE + int(last[i]) if pages else 0


def _softmax64(q, parts):
    """out [G, 128] and lse [G], base 2, of q [G, 128] over parts of (K, V)."""
    k, v = (torch.cat([part[i] for part in parts]) for i in range(2))
    if not len(k):
        return torch.zeros_like(q, dtype=torch.float64), torch.full((len(q),), -math.inf, dtype=torch.float64,
                                                                    device="cuda")
    score = torch.mm(q.double(), k.t().contiguous()) / math.sqrt(DIM)
    lse = torch.logsumexp(score, dim=1)
    return torch.mm(torch.exp(score - lse[:, None]), v), lse / math.log(2.0)


def _exact_attention(s, history):
    """``history(b, head)``: the parts of (K, V) before the exact tail."""
    case = s["case"]
    heads, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    out = torch.empty(case["requests"], case["q_heads"], DIM, dtype=torch.float64, device="cuda")
    lse = torch.empty(case["requests"], case["q_heads"], dtype=torch.float64, device="cuda")
    tail_last = s["tail_last"].tolist()
    for b in range(case["requests"]):
        tail = s["tail_ids"][int(s["tail_indptr"][b]):int(s["tail_indptr"][b + 1])].long()
        tokens = _tokens(s["tail_indptr"], tail_last, b)
        for h in range(heads):
            rows = slice(h * group, (h + 1) * group)
            parts = history(b, h) + [_rows64(s["exact"], (None, None), tail, tokens, h)]
            o, l = _softmax64(s["q"][b, rows], parts)
            out[b, rows], lse[b, rows] = o + s["center"][b, h].double(), l
    return out, lse


def _exact_prefix(s):
    segments, prefix_last, last = s["segments"].tolist(), s["prefix_last"].tolist(), s["last"].tolist()
    shared = {}

    def history(b, h):
        parts = []
        for i, (begin, end) in enumerate(segments):
            if begin <= b < end:
                if (i, h) not in shared:
                    ids = s["prefix_ids"][int(s["prefix_indptr"][i]):int(s["prefix_indptr"][i + 1])].long()
                    shared[i, h] = _rows64(s["cache"], s["scales"], ids, _tokens(s["prefix_indptr"], prefix_last, i), h)
                parts.append(shared[i, h])
        ids = s["ids"][int(s["indptr"][b]):int(s["indptr"][b + 1])].long()
        return parts + [_rows64(s["cache"], s["scales"], ids, _tokens(s["indptr"], last, b), h)]

    return _exact_attention(s, history)


def _exact_sparse(s):
    case, last = s["case"], s["last"].tolist()
    heads, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    found = torch.full((case["requests"], heads, case["pages"]), NO_PAGE, dtype=torch.int32, device="cuda")

    def pick(b, h):
        ids = s["ids"][int(s["indptr"][b]):int(s["indptr"][b + 1])].long()
        q = s["q"][b, h * group:(h + 1) * group].double()
        exponent = torch.floor(torch.log2(q.abs().amax(1, keepdim=True))) + 1
        steps = torch.clamp(torch.round(torch.ldexp(q, 7 - exponent)), -127, 127)
        low, high = s["bounds"][ids, h].double().unbind(1)
        total = torch.zeros(group, len(ids), dtype=torch.float64, device="cuda")
        for g in range(group):
            total[g] = torch.maximum(steps[g] * low, steps[g] * high).sum(1)
        # the definition rounds a page's product to float32; the unit is a power of two
        score = (total * s["scales"][0][ids, h].double()).float().double() * torch.ldexp(torch.ones_like(exponent), exponent - 7)
        score = score.amax(0)
        score[:case["first"]] = math.inf
        score[max(0, len(ids) - case["last"]):] = math.inf
        order = sorted(range(len(ids)), key=lambda p, values=score.tolist(): (-values[p], p))
        return ids, sorted(order[:case["pages"]])

    def history(b, h):
        ids, chosen = pick(b, h)
        found[b, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32, device="cuda")
        # a partial page is the last one in the table, and so in the selection
        cut = PAGE - last[b] if chosen and chosen[-1] == len(ids) - 1 else 0
        at = ids[torch.tensor(chosen, dtype=torch.long, device="cuda")]
        return [_rows64(s["cache"], s["scales"], at, len(chosen) * PAGE - cut, h)]

    out, lse = _exact_attention(s, history)
    return found, out, lse
