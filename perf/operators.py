"""Cases for the page operators and the tree attention over a paged KV cache.

A case names one operator (`op`) and the geometry of the cache that it works
on.  `run` with own = False computes it with elementary torch operations;
with own = True it calls demo_b200.pages.PagePool and
demo_b200.attention.TreeAttention.

The page state is what both sides share: table [rows, width], lens [rows],
refs [pages], free [pages] (a stack of free page ids) and count [1], all int32.
Row r holds the pages table[r, :ceil(lens[r] / block)].
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
ELT = {"bf16": 2, "fp16": 2, "e4m3": 1}
K_SCALE, V_SCALE = 0.75, 1.25          # dequantisation scales of the 8-bit caches


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # four pages copied on write while decoding: Llama-3-8B, 32 layers x 8 heads x 128, block 16
        {"name": "copy_on_write", "op": "copy", "order": "nhd", "layers": 32, "heads": 8, "dim": 128, "block": 16,
         "pages": 512, "n": 4, "partial": False},
        # a scheduler moving half of an MLA latent cache: 27 layers, K only, 576 wide, block 64
        {"name": "copy_mla", "op": "copy", "order": "k", "layers": 27, "heads": 1, "dim": 576, "block": 64,
         "pages": 1000, "n": 500, "partial": False},
        # eight continuations of one prompt (parallel sampling), Llama-3-8B
        {"name": "fork_samples", "op": "fork", "order": "nhd", "layers": 32, "heads": 8, "dim": 128, "block": 16,
         "pages": 1024, "parents": 1, "n": 8, "tokens": 2043, "width": 160},
        # beams of a batch, one KV head of an 80-layer model (Llama-3-70B, TP 8), head-major blocks
        {"name": "fork_beams", "op": "fork", "order": "hnd", "layers": 80, "heads": 1, "dim": 128, "block": 16,
         "pages": 5000, "parents": 64, "n": 256, "tokens": 1000, "width": 128},
        # a speculative step's accepted tokens: 64 requests of Llama-3-8B, 24 drafted tokens each, head-major blocks
        {"name": "compact_accepted", "op": "compact", "order": "hnd", "layers": 32, "heads": 8, "dim": 128, "block": 16,
         "pages": 1100, "n": 64, "tokens": 230, "drafted": 24, "kept": 5, "width": 20},
        # half of the tokens of four long requests evicted from the cache
        {"name": "compact_evicted", "op": "compact", "order": "nhd", "layers": 32, "heads": 8, "dim": 128, "block": 16,
         "pages": 1100, "n": 4, "tokens": 4093, "drafted": 4000, "kept": 2000, "width": 260},
        # a speculative step of 64 requests: some take a few pages, some give a few back
        {"name": "resize_step", "op": "resize", "block": 16, "pages": 16384, "n": 64, "low": 1900, "high": 2048,
         "width": 128},
        # a whole batch of long requests replaced by the next one
        {"name": "resize_batch", "op": "resize", "block": 16, "pages": 131072, "n": 256, "low": 1, "high": 8192,
         "width": 512},
        # one token of one request, the smallest call: Llama-3-8B, 2048 tokens cached
        {"name": "attend_one", "op": "attend", "order": "nhd", "type": "bf16", "q_heads": 32, "heads": 8, "dim": 128,
         "block": 16, "n": 1, "low": 2048, "high": 2048, "nodes_low": 1, "nodes_high": 1, "tree": False},
        # drafted trees of a batch of 64 requests, ragged, head-major blocks
        {"name": "attend_trees", "op": "attend", "order": "hnd", "type": "bf16", "q_heads": 32, "heads": 8, "dim": 128,
         "block": 16, "n": 64, "low": 500, "high": 2048, "nodes_low": 9, "nodes_high": 32, "tree": True},
        # long contexts on one KV head of Llama-3-70B (TP 8) with large trees
        {"name": "attend_long", "op": "attend", "order": "nhd", "type": "fp16", "q_heads": 8, "heads": 1, "dim": 128,
         "block": 16, "n": 8, "low": 32768, "high": 131072, "nodes_low": 64, "nodes_high": 64, "tree": True},
        # an 8-bit cache, head-major, a chain of drafted tokens per request
        {"name": "attend_8bit", "op": "attend", "order": "hnd", "type": "e4m3", "q_heads": 32, "heads": 8, "dim": 128,
         "block": 64, "n": 32, "low": 4000, "high": 8192, "nodes_low": 4, "nodes_high": 4, "tree": False},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["copy", "fork", "compact", "resize", "attend", "attend"])
    if op == "resize":
        n, high = _spread(rng, 1, 256), _spread(rng, 16, 8192)
        block = rng.choice([8, 16, 24, 64])
        width = -(-high // block)
        return {"op": op, "block": block, "pages": n * width + rng.randrange(1, 100), "n": n, "low": rng.choice([0, 1]),
                "high": high, "width": width}
    if op == "attend":
        q_heads, heads, dim = rng.choice([(32, 8, 128), (8, 1, 128), (8, 8, 64), (12, 2, 96), (8, 2, 256), (5, 1, 80)])
        nodes = _spread(rng, 1, 64)
        # cached tokens: at most 1 GiB of K and V at 16 bits, and the largest listed case's products
        room = min((1 << 30) // (heads * dim * 4), int(1.6e11 / (4 * q_heads * dim * nodes)))
        n = _spread(rng, 1, 64)
        high = _spread(rng, 64, max(65, min(65536, room // n)))
        return {"op": op, "order": rng.choice(["nhd", "hnd"]), "type": rng.choice(["bf16", "fp16", "e4m3"]),
                "q_heads": q_heads, "heads": heads, "dim": dim, "block": rng.choice([8, 16, 24, 32, 64]), "n": n,
                "low": max(1, high // rng.randrange(1, 9)), "high": high, "nodes_low": max(1, nodes // 2),
                "nodes_high": nodes, "tree": rng.random() < 0.6}
    order = rng.choice(["nhd", "hnd", "k"])
    heads, dim = (1, rng.choice([576, 320])) if order == "k" else rng.choice([(8, 128), (1, 128), (2, 64), (3, 40)])
    block = rng.choice([8, 16, 24, 64])
    layers = rng.randrange(1, 81)
    page = layers * (1 if order == "k" else 2) * block * heads * dim * 2
    pages = max(64, min(4096, (1 << 30) // page))
    case = {"op": op, "order": order, "layers": layers, "heads": heads, "dim": dim, "block": block, "pages": pages}
    if op == "copy":
        return {**case, "n": _spread(rng, 1, pages // 2), "partial": rng.random() < 0.5}
    if op == "fork":
        n = _spread(rng, 1, max(2, pages // 4))
        parents = rng.randrange(1, min(n, 16) + 1)
        tokens = _spread(rng, 1, max(2, (pages - n) // parents * block - 1))
        return {**case, "parents": parents, "n": n, "tokens": tokens, "width": -(-tokens // block) + rng.randrange(1, 9)}
    n = _spread(rng, 1, max(2, pages // 16))
    tokens = _spread(rng, 2, max(3, pages // n * block - block))
    drafted = _spread(rng, 1, tokens)
    return {**case, "n": n, "tokens": tokens, "drafted": drafted, "kept": _spread(rng, 1, drafted),
            "width": -(-tokens // block) + rng.randrange(0, 5)}


# --------------------------------------------------------------- the inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(low, high, size, g):
    """int32 in [low, high]"""
    return torch.randint(low, high + 1, (size,), generator=g, device="cuda", dtype=torch.int32)


def _cache(case, pages, g):
    """The cache's storage: token-major [layers, 2, pages, block, heads, dim]
    (all of K, then V), head-major [layers, pages, 2, heads, block, dim], K
    only [layers, pages, block, dim].  Page operators move bytes: int16."""
    L, H, D, bs = case["layers"], case["heads"], case["dim"], case["block"]
    shape = {"nhd": (L, 2, pages, bs, H, D), "hnd": (L, pages, 2, H, bs, D), "k": (L, pages, bs, D)}[case["order"]]
    return torch.randint(-30000, 30000, shape, generator=g, device="cuda", dtype=torch.int16)


def _view(cache, order):
    """[layers, 1 or 2, pages, block, heads, dim], whatever the storage"""
    if order == "nhd":
        return cache
    if order == "hnd":
        return cache.permute(0, 2, 1, 4, 3, 5)
    return cache[:, None, :, :, None]


def _layer_tensors(cache, order):
    """one tensor per layer in the form that engines hand over"""
    return list(cache.permute(0, 1, 2, 4, 3, 5) if order == "hnd" else cache)


def _state(lens, width, pages, block, g):
    """Tables of rows with `lens` tokens over distinct pages in random order."""
    rows = lens.numel()
    used = (lens + block - 1) // block
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    at = torch.arange(width, device="cuda")
    index = (torch.cumsum(used, 0) - used)[:, None] + at
    taken = at < used[:, None]
    table = torch.where(taken, order[index.clamp(max=pages - 1).long()], torch.full((), -1, device="cuda", dtype=torch.int32))
    total = int(used.sum())
    assert total <= pages, "the case's rows do not fit its pages"
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[order[total:].long()] = 0
    free = torch.zeros(pages, dtype=torch.int32, device="cuda")
    free[:pages - total] = order[total:]
    count = torch.full((1,), pages - total, dtype=torch.int32, device="cuda")
    return {"table": table.to(torch.int32).contiguous(), "lens": lens.clone(), "refs": refs, "free": free, "count": count,
            "block": block}


def _pool(s, cache, order):
    from demo_b200 import cache as cc
    from demo_b200.pages import PagePool

    layout, k, v = cc.layout_from_kv_tensors(_layer_tensors(cache, order),
                                             kv_layout={"nhd": "flash_attn", "hnd": "flashinfer", "k": None}[order])
    return PagePool(layout, k, v, s["table"], s["lens"], refs=s["refs"], free_list=s["free"], free_count=s["count"])


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "attend":
        return _prepare_attend(case, g)
    if op == "resize":
        # the tables alone are at work: one narrow layer stands for the cache
        n = case["n"]
        a, b = (_ints(case["low"], case["high"], n, g) for _ in range(2))
        s = _state(a, case["width"], case["pages"], case["block"], g)
        s["rows"] = torch.randperm(n, generator=g, device="cuda", dtype=torch.int32)
        s["to"], s["back"] = b[s["rows"].long()].contiguous(), a[s["rows"].long()].contiguous()
        s["cache"] = torch.zeros(1, 2, case["pages"], case["block"], 1, 8, dtype=torch.int16, device="cuda")
        order = "nhd"
    else:
        order = case["order"]
        pages = case["pages"]
        if op == "copy":
            s = _state(torch.zeros(1, dtype=torch.int32, device="cuda"), 1, pages, case["block"], g)
            ids = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
            n = case["n"]
            s["src"], s["dst"] = ids[:n].contiguous(), ids[n:2 * n].contiguous()
            s["tokens"] = _ints(0, case["block"], n, g) if case["partial"] else None
        elif op == "fork":
            p, n = case["parents"], case["n"]
            lens = torch.zeros(p + n, dtype=torch.int32, device="cuda")
            lens[:p] = _ints(max(1, case["tokens"] - 2 * case["block"]), case["tokens"], p, g)
            s = _state(lens, case["width"], pages, case["block"], g)
            s["parents"] = _ints(0, p - 1, n, g)
            s["children"] = torch.arange(p, p + n, dtype=torch.int32, device="cuda")
            s["zero"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        else:
            n, drafted, kept = case["n"], case["drafted"], case["kept"]
            tokens = _ints(max(drafted, case["tokens"] - case["block"]), case["tokens"], n, g)
            s = _state(tokens, case["width"], pages, case["block"], g)
            s["rows"] = torch.randperm(n, generator=g, device="cuda", dtype=torch.int32)
            s["full"] = tokens[s["rows"].long()].contiguous()
            s["start"] = (s["full"] - drafted).contiguous()
            many = _ints(max(0, kept // 2), kept, n, g)
            s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"),
                                      torch.cumsum(many, 0).to(torch.int32)])
            # `many` of the `drafted` tokens of each row, in ascending order
            pick = torch.rand(n, drafted, generator=g, device="cuda").argsort(1).argsort(1) < many[:, None]
            at = s["start"][:, None] + torch.arange(drafted, device="cuda", dtype=torch.int32)
            s["keep"] = at[pick].to(torch.int32).contiguous()
        s["cache"] = _cache(case, pages, g)
    s["op"], s["view"] = op, _view(s["cache"], order)
    s["pool"] = _pool(s, s["cache"], order) if own else None
    return s


def _prepare_attend(case, g):
    n, H, D, bs, Hq = case["n"], case["heads"], case["dim"], case["block"], case["q_heads"]
    # every count from nodes_low to nodes_high, dealt to the requests by the seed
    nodes = torch.linspace(case["nodes_low"], case["nodes_high"], n, device="cuda").round().to(torch.int32)
    nodes = nodes[torch.randperm(n, generator=g, device="cuda")]
    lens = _ints(case["low"], case["high"], n, g)
    lens[0] = case["high"]
    lens = lens + nodes
    longest, most = int(lens.max()), int(nodes.max())
    width = -(-longest // bs)
    pages = int(((lens + bs - 1) // bs).sum()) + 3
    s = _state(lens, width, pages, bs, g)
    t = DTYPES[case["type"]]
    shape = (1, 2, pages, bs, H, D) if case["order"] == "nhd" else (1, pages, 2, H, bs, D)
    cache = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16).to(t)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), torch.cumsum(nodes, 0).to(torch.int32)])
    total = int(offsets[-1])
    q = torch.randn(total, Hq, D, generator=g, device="cuda").to(torch.bfloat16 if t == torch.float8_e4m3fn else t)
    parents = None
    if case["tree"]:
        # a tree per request: each node under one of the nodes before it, or under the last cached token (-1)
        at = torch.cat([torch.arange(int(m), device="cuda") for m in nodes])
        parents = (torch.rand(total, generator=g, device="cuda") * (at + 1)).long().clamp(max=at) - 1
        parents = parents.to(torch.int32).contiguous()
    scales = (K_SCALE, V_SCALE) if case["type"] == "e4m3" else (1.0, 1.0)
    s.update(op="attend", cache=cache, kv=_view(cache, case["order"])[0], offsets=offsets, q=q, parents=parents,
             scales=scales, longest=longest, most=most, heads=H, attention=None)
    if own:
        from demo_b200 import cache as cc
        from demo_b200.attention import TreeAttention

        layout, k, v = cc.layout_from_kv_tensors(_layer_tensors(cache, case["order"]),
                                                 kv_layout="flash_attn" if case["order"] == "nhd" else "flashinfer")
        s["attention"] = TreeAttention(layout, k, v, num_heads=Hq, num_kv_heads=H, k_scale=scales[0], v_scale=scales[1])
    return s


# ------------------------------------------------------------ the operators
def _page_outputs(s, *status):
    return {"cache": s["cache"], "table": s["table"], "lens": s["lens"], "refs": s["refs"], "free": s["free"],
            "count": s["count"], "status": list(status)}


def run(s):
    op = s["op"]
    if op == "attend":
        if own:
            return s["attention"](0, s["q"], s["table"], s["lens"], s["offsets"], parents=s["parents"], return_lse=True)
        return _plain_attend(s, torch.float32)
    pool = s["pool"]
    if op == "copy":
        if own:
            pool.copy(s["src"], s["dst"], s["tokens"])
        else:
            _plain_copy(s, s["src"].long(), s["dst"].long(), s["tokens"])
        return s["cache"]
    if op == "resize":              # the batch goes to other lengths and back
        if own:
            return _page_outputs(s, pool.resize(s["rows"], s["to"]), pool.resize(s["rows"], s["back"]))
        return _page_outputs(s, _plain_resize(s, s["rows"], s["to"]), _plain_resize(s, s["rows"], s["back"]))
    if op == "fork":                # children forked, then dropped
        if own:
            return _page_outputs(s, pool.fork(s["parents"], s["children"]), pool.resize(s["children"], s["zero"]))
        return _page_outputs(s, _plain_fork(s), _plain_resize(s, s["children"], s["zero"]))
    # room for the drafted tokens, then the kept ones put in order
    if own:
        return _page_outputs(s, pool.resize(s["rows"], s["full"]),
                             pool.compact(s["rows"], s["start"], s["keep"], s["offsets"]))
    return _page_outputs(s, _plain_resize(s, s["rows"], s["full"]), _plain_compact(s))


def _plain_copy(s, src, dst, tokens):
    v = s["view"]
    new = v[:, :, src]
    if tokens is not None:
        within = torch.arange(v.shape[3], device="cuda") < tokens[:, None]
        new = torch.where(within[:, :, None, None], new, v[:, :, dst])
    v[:, :, dst] = new


def _plain_resize(s, rows, lens):
    table, seq, refs, free, count, bs = (s[k] for k in ("table", "lens", "refs", "free", "count", "block"))
    n, width, pages = rows.numel(), table.shape[1], refs.numel()
    r = rows.long()
    old, new = (seq[r].long() + bs - 1) // bs, (lens.long() + bs - 1) // bs
    at = torch.arange(width, device="cuda")
    mine = table[r].long()
    # entries given back, in the order of the call; page number `pages` stands for none
    drop = (at >= new[:, None]) & (at < old[:, None])
    page = torch.where(drop, mine, pages).reshape(-1)
    number = torch.arange(n * width, device="cuda")
    times = torch.zeros(pages + 1, dtype=torch.int64, device="cuda").scatter_add_(0, page, torch.ones_like(page))
    last = torch.full((pages + 1,), -1, device="cuda").scatter_reduce_(0, page, number, "amax")
    left = refs - times[:pages].to(torch.int32)
    gone = drop.reshape(-1) & (last[page] == number) & (torch.cat([left, left.new_ones(1)])[page] == 0)
    rank = torch.cumsum(gone, 0)
    stack = torch.cat([free, free.new_zeros(1)])
    stack.scatter_(0, torch.where(gone, count + rank - 1, pages), page.to(torch.int32))
    have = count + rank[-1:]
    # pages taken from the top of the stack, rows in the order of the call
    need = (new - old).clamp(min=0)
    upto = torch.cumsum(need, 0)
    fits = (need == 0) | (upto <= have)
    take = (at >= old[:, None]) & (at < new[:, None]) & fits[:, None]
    source = have - 1 - ((upto - need)[:, None] + at - old[:, None])
    fresh = stack[torch.where(take, source, pages)].long()
    table[r] = torch.where(take, fresh, mine).to(torch.int32)
    left = torch.cat([left, left.new_zeros(1)])
    left.scatter_(0, torch.where(take, fresh, pages).reshape(-1), torch.ones(n * width, dtype=torch.int32, device="cuda"))
    refs.copy_(left[:pages])
    free.copy_(stack[:pages])
    count.copy_(have - torch.where(fits, need, 0).sum())
    seq[r] = torch.where(fits, lens, seq[r])
    return torch.where(fits, 0, 1).to(torch.int32)


def _plain_fork(s):
    table, seq, refs, free, count, bs = (s[k] for k in ("table", "lens", "refs", "free", "count", "block"))
    pages = refs.numel()
    p, c = s["parents"].long(), s["children"].long()
    length = seq[p].long()
    full, tail = length // bs, length % bs
    need = (tail > 0).long()
    upto = torch.cumsum(need, 0)
    fits = (need == 0) | (upto <= count)
    copied = fits & (need > 0)
    at = torch.arange(table.shape[1], device="cuda")
    theirs = table[p].long()
    share = (at < full[:, None]) & fits[:, None]
    more = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    more.scatter_add_(0, torch.where(share, theirs, pages).reshape(-1), torch.ones(share.numel(), dtype=torch.int32, device="cuda"))
    fresh = free[torch.where(copied, count - upto, 0)].long()
    more.scatter_(0, torch.where(copied, fresh, pages), torch.ones_like(fresh, dtype=torch.int32))
    # a child that copies nothing rewrites the last page that it shares with what it holds
    source = torch.gather(theirs, 1, torch.where(copied, full, (full - 1).clamp(min=0))[:, None])[:, 0]
    _plain_copy(s, source, torch.where(copied, fresh, source), torch.where(copied, tail, 0))
    mine = torch.where((at == full[:, None]) & copied[:, None], fresh[:, None], table[c].long())
    table[c] = torch.where(share, theirs, mine).to(torch.int32)
    seq[c] = torch.where(fits, seq[p], seq[c])
    refs += more[:pages]
    count -= copied.sum().to(torch.int32)
    return torch.where(fits, 0, 1).to(torch.int32)


def _plain_compact(s):
    table, bs, keep, offsets = s["table"], s["block"], s["keep"].long(), s["offsets"].long()
    i = torch.arange(keep.numel(), device="cuda")
    of = torch.bucketize(i, offsets[1:], right=True)
    to = s["start"].long()[of] + i - offsets[of]
    row = s["rows"].long()[of]
    v = s["view"]
    v[:, :, table[row, to // bs].long(), to % bs] = v[:, :, table[row, keep // bs].long(), keep % bs]
    return _plain_resize(s, s["rows"], (s["start"] + (offsets[1:] - offsets[:-1])).to(torch.int32))


def _ancestors(parents, offsets, most):
    """[requests, most, most] truth values: node j sees node i (its ancestors
    and itself).  With one parent per node the sum of the parent matrix's
    powers, 1 / (1 - P), holds zeros and ones."""
    nodes = offsets[1:] - offsets[:-1]
    at = torch.arange(most, device="cuda")
    there = at < nodes[:, None]
    index = torch.where(there, offsets[:-1, None] + at, 0).long()
    up = torch.where(there, at - 1, -2) if parents is None else torch.where(there, parents[index], -2)
    step = (up[:, :, None] == at).float()
    eye = torch.eye(most, device="cuda")
    sees = torch.linalg.solve_triangular(eye - step, eye.expand(len(nodes), -1, -1), upper=False, unitriangular=True)
    return (sees > 0.5) & there[:, :, None], there, index


def _take(plane, page, slot, t):
    """[..., heads, dim] of the given pages and slots, in type t (8-bit caches
    are indexed as bytes)"""
    if plane.element_size() == 1:
        return plane.view(torch.uint8)[page, slot].view(plane.dtype).to(t)
    return plane[page, slot].to(t)


def _plain_attend(s, t):
    q, table, lens, offsets, bs, H = s["q"], s["table"], s["lens"].long(), s["offsets"].long(), s["block"], s["heads"]
    n, most, longest = lens.numel(), s["most"], s["longest"]
    Hq, D = q.shape[1:]
    sees, there, index = _ancestors(s["parents"], offsets, most)
    pos = torch.arange(longest, device="cuda")
    inside = pos < lens[:, None]
    page = torch.where(inside, table[:, pos // bs].long(), 0)
    k = _take(s["kv"][0], page, pos % bs, t) * s["scales"][0]                     # [n, longest, H, D]
    v = torch.where(inside[:, :, None, None], _take(s["kv"][1], page, pos % bs, t), 0.0) * s["scales"][1]
    x = q[index].to(t).reshape(n, most, H, Hq // H, D).permute(0, 2, 1, 3, 4).reshape(n, H, most * (Hq // H), D)
    score = (x @ k.permute(0, 2, 3, 1)).view(n, H, most, Hq // H, longest) * D ** -0.5
    node = pos - (lens - (offsets[1:] - offsets[:-1]))[:, None]                 # negative: cached before the drafts
    drafted = torch.gather(sees, 2, node.clamp(0, most - 1)[:, None].expand(-1, most, -1))
    seen = torch.where(node[:, None] < 0, there[:, :, None], drafted) & inside[:, None]
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(t).min)
    score = score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = score.view(n, H, most * (Hq // H), longest) @ v.permute(0, 2, 1, 3)
    out = out.view(n, H, most, Hq // H, D) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log())[..., 0]
    i = torch.arange(q.shape[0], device="cuda")
    of = torch.bucketize(i, offsets[1:], right=True)
    j = i - offsets[of]
    out = out.permute(0, 2, 1, 3, 4).reshape(n, most, Hq, D)[of, j]
    lse = lse.permute(0, 2, 1, 3).reshape(n, most, Hq)[of, j]
    return out.to(q.dtype), lse.to(torch.float32)


# ----------------------------------------------------------- what they cost
def _token_bytes(case):
    return case["layers"] * (1 if case["order"] == "k" else 2) * case["heads"] * case["dim"] * 2


def work(case):
    op, bs = case["op"], case.get("block")
    if op == "copy":
        tokens = case["n"] * bs // (2 if case["partial"] else 1)
        return {"bytes": 2 * tokens * _token_bytes(case) + 8 * case["n"], "flops": 0}
    if op == "fork":
        shared = case["n"] * (case["tokens"] // bs)
        tail = case["n"] * bs / 2 if case["parents"] > 1 else case["n"] * (bs // 2)
        return {"bytes": 2 * tail * _token_bytes(case) + 16 * shared + 24 * case["n"], "flops": 0}
    if op == "compact":
        moved = case["n"] * case["kept"] * 0.75
        return {"bytes": 2 * moved * _token_bytes(case) + 4 * moved, "flops": 0}
    if op == "resize":
        entries = 2 * case["n"] * (case["high"] - case["low"]) / bs / 3          # the mean change of two even draws, there and back
        return {"bytes": 2 * 12 * case["n"] + 20 * entries, "flops": 0}
    n, H, D, Hq = case["n"], case["heads"], case["dim"], case["q_heads"]
    cached = n * (case["low"] + case["high"]) / 2
    nodes = n * (case["nodes_low"] + case["nodes_high"]) / 2
    seen = (case["low"] + case["high"]) / 2 + 1
    return {"bytes": 2 * (cached + nodes) * H * D * ELT[case["type"]] + 2 * nodes * Hq * D * 2 + 4 * nodes * Hq,
            "flops": 4 * nodes * Hq * D * seen}


# --------------------------------------------------------- the definition
def exact(case, seed):
    """Attention in 64 bits, request by request and head by head, straight
    from the definition.  The page operators move bytes: nothing is computed."""
    if case["op"] != "attend":
        return None
    s = prepare(case, seed)
    q, kv, scales = s["q"], s["kv"], s["scales"]
    Hq, D = q.shape[1:]
    group = Hq // s["heads"]
    table, lens, offsets = s["table"].tolist(), s["lens"].tolist(), s["offsets"].tolist()
    parents = s["parents"].tolist() if s["parents"] is not None else None
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        first, nodes = offsets[b], offsets[b + 1] - offsets[b]
        before = length - nodes
        ids = torch.tensor(table[b][:-(-length // s["block"])], device="cuda")
        every = torch.arange(length, device="cuda")
        k, v = (_take(kv[i], ids[every // s["block"]], every % s["block"], torch.float64) * scales[i] for i in range(2))
        seen = torch.zeros(nodes, length, dtype=torch.bool)
        for j in range(nodes):
            up = j - 1 if parents is None else parents[first + j]
            seen[j, before + j] = True
            seen[j, :before] = True
            if up >= 0:
                seen[j, before:] |= seen[up, before:]
        seen = seen.cuda()
        for h in range(s["heads"]):
            x = q[first:first + nodes, h * group:(h + 1) * group].double()
            score = torch.einsum("jgd,pd->jgp", x, k[:, h]) / math.sqrt(D)
            score = score.masked_fill(~seen[:, None], -math.inf)
            whole = torch.logsumexp(score, -1)
            out[first:first + nodes, h * group:(h + 1) * group] = torch.einsum(
                "jgp,pd->jgd", (score - whole[..., None]).exp(), v[:, h])
            lse[first:first + nodes, h * group:(h + 1) * group] = whole
    return out, lse
