"""Operators of drafted tokens and of pages that requests copy, as cases that can be measured one by one.

A request whose next tokens were guessed brings several tokens in one step: a tree, whose first node is the last token that
is certain and whose other nodes continue their parents.  ``layout``: which nodes each node sees, and the nodes' positions.
``tree``: attention of the nodes over the cache and over one another.  ``keep``: the path that the model's own choices confirm,
whose entries move together behind the context in every layer.  ``copy``: pages, or the entries that they hold so far, copied in
every layer, as for a request that forks into several.

A cache is [pages, 2, kv heads, page, head size]; request r's entry e is row e % page of page table[r, e // page].  Head
counts, head sizes, page sizes and layers are those of the models that this repository measures and tests.

A case's keys: ``op``; ``dtype``; ``nh``, ``nkv``, ``d``, ``page``; ``requests`` of ``rows`` nodes behind ``context`` entries (layout, tree,
keep); ``layers`` (keep, copy); ``copies`` of pages that hold ``held`` entries (copy); ``shape``: "tree", or "chain" for one guess
after the other; ``ragged``: the numbers differ.
"""
import math

import numpy as np
import torch

own = False


def _case(op, dtype="bfloat16", nh=32, nkv=8, d=128, page=16, ragged=False, **sizes):
    return dict(op=op, dtype=dtype, nh=nh, nkv=nkv, d=d, page=page, ragged=ragged, **sizes)


def listed():
    return [
        # one request's small tree, between two steps
        dict(_case("layout", d=64, requests=1, rows=16, context=1024, shape="tree"), name="layout-1"),
        # a busy server with large trees, every request its own
        dict(_case("layout", ragged=True, requests=64, rows=256, context=4096, shape="tree"), name="layout-64"),
        # two requests of the smallest model in 32-bit
        dict(_case("tree", "float32", 3, 1, 32, 8, True, requests=2, rows=7, context=61, shape="tree"), name="tree-tiny-f32"),
        # one user, a small tree
        dict(_case("tree", d=64, requests=1, rows=16, context=1024, shape="tree"), name="tree-1"),
        # a few chats that guess four tokens ahead
        dict(_case("tree", nh=24, ragged=True, requests=8, rows=5, context=2000, shape="chain"), name="tree-chain"),
        # a busy server with long contexts, every request at its own length
        dict(_case("tree", ragged=True, requests=64, rows=16, context=4096, shape="tree"), name="tree-64"),
        # four users, wide trees
        dict(_case("tree", requests=4, rows=64, context=8192, shape="tree"), name="tree-wide"),
        # one very long document and all the guesses that there is time for
        dict(_case("tree", requests=1, rows=128, context=65536, shape="tree"), name="tree-long"),
        # one user: the confirmed path in the sixteen layers of a small model
        dict(_case("keep", d=64, requests=1, rows=16, context=40, layers=16, shape="tree"), name="keep-1"),
        # a busy server: the same in the thirty-two layers of a larger one
        dict(_case("keep", ragged=True, requests=64, rows=16, context=60, layers=32, shape="tree"), name="keep-64"),
        # a prompt forks into eight samples: the page that is being filled
        dict(_case("copy", d=64, copies=8, held=9, layers=16), name="copy-fork"),
        # requests of a whole batch copied, pages full or not
        dict(_case("copy", nh=24, ragged=True, copies=256, held=16, layers=28), name="copy-pages"),
    ]


# query heads, kv heads, head size, page of the models that this repository measures
_HEADS = [(32, 8, 64, 16), (24, 8, 128, 16), (32, 8, 128, 16), (16, 2, 128, 16), (32, 8, 128, 32)]
_TINY = [(3, 1, 32, 8), (4, 2, 16, 16), (4, 2, 64, 16)]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    op = rng.choice(["tree", "tree", "tree", "layout", "keep", "copy"])
    f32 = rng.random() < 0.2
    nh, nkv, d, page = rng.choice(_TINY if f32 else _HEADS)
    c = dict(dtype="float32" if f32 else "bfloat16", nh=nh, nkv=nkv, d=d, page=page, ragged=rng.random() < 0.6)
    shape = rng.choice(["tree", "tree", "chain"])
    if op == "layout":
        requests = size(1, 256)
        return _case(op, requests=requests, rows=size(1, min(512, int(math.sqrt(4_000_000 / requests)))), context=size(500, 65536), shape=shape, **c)
    if op == "tree":
        top = 64 if f32 else 1              # the 32-bit path serves small models: shorter by so much
        requests = size(1, 128 // min(top, 8))
        rows = size(1, min(128, 2048 // requests))
        context = size(1, min(65536 // top, 8_000_000 // (requests * rows), 131072 // requests))
        return _case(op, requests=requests, rows=rows, context=context, shape=shape, **c)
    entry = nkv * d * 2 * (4 if f32 else 2)
    layers = rng.choice([1, 2, 4]) if f32 else rng.choice([16, 28, 32])
    if op == "keep":
        requests = size(1, 128)
        rows = size(1, min(64, 2048 // requests))
        context = size(1, max(1, min(300, 500_000_000 // (requests * layers * entry) - rows - page)))
        return _case(op, requests=requests, rows=rows, context=context, layers=layers, shape=shape, **c)
    copies = size(1, min(512, 450_000_000 // (layers * entry * page)))
    return _case(op, copies=copies, held=rng.randint(1, page), layers=layers, **c)


# ---- what a user's program has in hand ------------------------------------------------------------------------------
def _lengths(n, top, ragged, least, gen):
    """n lengths, all ``top``, or between ``least`` and ``top`` with one of them ``top``."""
    if not ragged or n == 0:
        return [top] * n
    v = torch.randint(min(least, top), top + 1, (n,), generator=gen).tolist()
    v[int(torch.randint(0, n, (1,), generator=gen))] = top
    return v


def _spread(n, top, ragged, gen):
    """n numbers of rows, all ``top``, or from 1 to ``top`` in some order: their sum is the case's."""
    if not ragged or n == 1:
        return [top] * n
    v = torch.tensor([1 + (top - 1) * i // (n - 1) for i in range(n)])
    return v[torch.randperm(n, generator=gen)].tolist()


def _caches(c, pages, layers, gen):
    return [torch.randn(pages, 2, c["nkv"], c["page"], c["d"], generator=gen, device="cuda", dtype=getattr(torch, c["dtype"])) for _ in range(layers)]


def prepare(case, seed):
    c = dict(case)
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, nh, nkv, d, page = getattr(torch, c["dtype"]), c["nh"], c["nkv"], c["d"], c["page"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    s = dict(c, scale=d ** -0.5)
    if c["op"] == "copy":
        n = c["copies"]
        pages = torch.randperm(2 * n + 3, generator=host)
        sources = pages[:n][torch.randint(0, n, (n,), generator=host)]          # several copies of one page among them
        held = _lengths(n, c["held"], c["ragged"], 1, host)
        # what the allocator says: (from, to, entries)
        s["copies"] = torch.stack([sources, pages[n:2 * n], torch.tensor(held)], 1).to(torch.int32).numpy()
        s["caches"] = _caches(c, 2 * n + 3, c["layers"], gen)
        return s
    R = c["requests"]
    counts = _spread(R, c["rows"], c["ragged"], host)
    if c["op"] == "layout":                         # a text is seldom the same length twice
        starts = torch.randint(c["context"] // 2, c["context"] + 1, (R,), generator=host).tolist()
    else:
        starts = _lengths(R, c["context"], c["ragged"], c["context"] // 2, host)
    T, cu = sum(counts), [0]
    for n in counts:
        cu.append(cu[-1] + n)
    # a node's parent comes before it; later nodes are the likelier parents
    at = torch.cat([torch.arange(n) for n in counts])
    parents = at - 1
    if c["shape"] == "tree":
        parents = torch.where(at > 0, (torch.rand(T, generator=host).sqrt() * at).long().clamp(max=at - 1), parents)
    s.update(parents=parents.to(torch.int32).cuda(), cu_rows=i32(cu), starts=i32(starts), max_rows=max(counts))
    if c["op"] == "layout":
        return s
    lens = [a + n for a, n in zip(starts, counts)]
    need = [-(-n // page) for n in lens]
    total = R * -(-(c["context"] + c["rows"]) // page) + 3
    pages, table, used = torch.randperm(total, generator=host).to(torch.int32), torch.zeros(R, max(need), dtype=torch.int32), 0
    for r, n in enumerate(need):
        table[r, :n] = pages[used:used + n]
        used += n
    s.update(block_table=table.cuda(), max_context=max(lens))
    if c["op"] == "keep":
        # guesses, and the model's choices: mostly one of a node's children, if it has any
        tokens = torch.randint(0, 128256, (T,), generator=host)
        chosen = torch.randint(0, 128256, (T,), generator=host)
        first = torch.repeat_interleave(torch.tensor(cu[:-1]), torch.tensor(counts))
        children = (at > 0).nonzero()[:, 0]
        agrees = children[torch.rand(len(children), generator=host) < 0.7]
        chosen[(first + parents)[agrees]] = tokens[agrees]
        s.update(tokens=tokens.to(torch.int32).cuda(), chosen=chosen.to(torch.int32).cuda(), caches=_caches(c, total, c["layers"], gen))
        return s
    s["kv_cache"] = _caches(c, total, 1, gen)[0]
    # queries that look at some keys more than at others
    s["qkv"] = torch.randn(T, (nh + 2 * nkv) * d, generator=gen, device="cuda").mul_(1.5).to(dtype)
    # the tree's layout, made once for all layers: a word of 32 nodes for each 32
    s["masks"], s["positions"] = _plain_layout(s)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    if not own:
        return _PLAIN[s["op"]](s)
    from railgun_b200 import ops
    if s["op"] == "layout":
        return ops.draft_tree(s["parents"], s["cu_rows"], s["starts"], max_rows=s["max_rows"])
    if s["op"] == "tree":
        nh, d = s["nh"], s["d"]
        q = s["qkv"][:, :nh * d]                    # the queries' columns of the fused projection
        out = torch.empty(q.shape[0], nh * d, dtype=q.dtype, device=q.device)
        ops.tree_attention(q, out, s["kv_cache"], s["block_table"], s["cu_rows"], s["starts"], s["masks"], nh, s["nkv"], d, s["scale"],
                           max_rows=s["max_rows"], max_context=s["max_context"])
        return out
    if s["op"] == "keep":
        counts, path, tokens = ops.keep_drafts(s["caches"], s["block_table"], s["cu_rows"], s["starts"], s["parents"], s["tokens"], s["chosen"],
                                               max_rows=s["max_rows"])
        return s["caches"], counts, path, tokens
    ops.copy_pages(s["caches"], s["copies"])
    return s["caches"]


def _side_by_side(s, values, rest):
    """[T] -> [requests, most rows], ``rest`` where a request has no such row; and where it has one."""
    cu = s["cu_rows"].long()
    at = torch.arange(s["max_rows"], device=values.device)
    there = at < (cu[1:] - cu[:-1])[:, None]
    rows = (cu[:-1, None] + at).clamp(max=len(values) - 1)
    return torch.where(there, values[rows].long(), rest), there, rows


def _ancestors(parents):
    """[requests, n, n]: is node j node i or an ancestor of it?  By paths of 1, 3, 7, ... steps."""
    n = parents.shape[1]
    at = torch.arange(n, device=parents.device)
    step = (parents[..., None] == at).float()
    reach = step + (at[:, None] == at).float()
    steps = 1
    while steps < n:
        step = step @ step
        reach = ((reach + step @ reach) > 0).float()
        steps = 2 * steps + 1
    return reach > 0


def _plain_layout(s):
    parents, there, rows = _side_by_side(s, s["parents"], -1)
    seen = _ancestors(parents) & there[..., None]
    R, n, _ = seen.shape
    words = -(-n // 32)
    bits = torch.nn.functional.pad(seen.long(), (0, 32 * words - n)).reshape(R, n, words, 32)
    masks = (bits << torch.arange(32, device=bits.device)).sum(-1)
    masks = torch.where(masks >= 1 << 31, masks - (1 << 32), masks).to(torch.int32)
    positions = (s["starts"].long()[:, None] + seen.sum(-1) - 1).to(torch.int32)
    return masks[there], positions[there]


def _plain_tree(s):
    nh, nkv, d = s["nh"], s["nkv"], s["d"]
    R, n = s["starts"].numel(), s["max_rows"]
    q = s["qkv"][:, :nh * d]
    _, there, rows = _side_by_side(s, s["parents"], -1)
    cu, starts = s["cu_rows"].long(), s["starts"].long()
    kv = s["kv_cache"][s["block_table"].long()].float().permute(2, 0, 3, 1, 4, 5)       # 2, requests, heads, pages, page, d
    kv = kv.reshape(2, R, nkv, -1, d)
    entry = torch.arange(kv.shape[3], device=q.device)
    node = entry - starts[:, None]                                                       # requests, entries
    word = s["masks"][rows].long().gather(2, (node // 32).clamp(0, s["masks"].shape[1] - 1)[:, None].expand(-1, n, -1))
    bit = (word >> (node % 32)[:, None]) & 1
    of_tree = (node >= 0) & (node < (cu[1:] - cu[:-1])[:, None])
    seen = (node < 0)[:, None] | (of_tree[:, None] & (bit == 1))                         # requests, rows, entries
    side = q.float().reshape(-1, nkv, nh // nkv, d)[rows].permute(0, 2, 3, 1, 4)         # requests, kv heads, heads, rows, d
    scores = (side @ kv[0][:, :, None].transpose(-1, -2)) * s["scale"]
    scores = torch.where(seen[:, None, None], scores, float("-inf"))
    top = scores.max(-1, keepdim=True).values
    weights = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = weights @ kv[1][:, :, None] / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4)[there]
    return out.reshape(-1, nh * d).to(q.dtype)


def _plain_keep(s):
    parents, there, _ = _side_by_side(s, s["parents"], -1)
    tokens, _, _ = _side_by_side(s, s["tokens"], -1)
    chosen, _, _ = _side_by_side(s, s["chosen"], -2)
    R, n = parents.shape
    at = torch.arange(n, device=parents.device)
    up = parents.clamp(min=0)
    agrees = there & (at > 0) & (tokens == chosen.gather(1, up))
    # of several children that agree the first counts
    earlier = (parents[:, :, None] == parents[:, None, :]) & (at[:, None] > at) & agrees[:, None, :]
    agrees = (agrees & ~earlier.any(-1)) | (there & (at == 0))
    kept = there & ~(_ancestors(parents) & ~agrees[:, None, :]).any(-1)
    counts = kept.sum(1)
    path = torch.sort(torch.where(kept, at, n), 1).values
    inside = at < counts[:, None]
    path = torch.where(inside, path, -1)
    new = torch.where(inside, chosen.gather(1, path.clamp(min=0)), -1)
    r, k = inside.nonzero(as_tuple=True)
    table, page, starts = s["block_table"].long(), s["page"], s["starts"].long()
    to, back = starts[r] + k, starts[r] + path[r, k]
    for cache in s["caches"]:
        cache[table[r, to // page], :, :, to % page] = cache[table[r, back // page], :, :, back % page]
    return s["caches"], counts.to(torch.int32), path.to(torch.int32), new.to(torch.int32)


def _plain_copy(s):
    copies = torch.from_numpy(s["copies"]).cuda().long()
    held = (torch.arange(s["page"], device="cuda") < copies[:, 2, None])[:, None, None, :, None]
    for cache in s["caches"]:
        cache[copies[:, 1]] = torch.where(held, cache[copies[:, 0]], cache[copies[:, 1]])
    return s["caches"]


_PLAIN = dict(layout=_plain_layout, tree=_plain_tree, keep=_plain_keep, copy=_plain_copy)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "layout":
        return None                                   # whole numbers
    s = prepare(case, seed)
    page = s["page"]
    if s["op"] == "copy":
        caches = [x.double() for x in s["caches"]]
        for a, b, held in s["copies"].tolist():
            for cache in caches:
                cache[b, :, :, :held] = cache[a, :, :, :held]
        return caches
    cu, starts, parents = s["cu_rows"].tolist(), s["starts"].tolist(), s["parents"].tolist()
    if s["op"] == "keep":
        if len(starts) * s["max_rows"] * len(s["caches"]) > 40_000:
            return None
        caches = [x.double() for x in s["caches"]]
        tokens, chosen, table = s["tokens"].tolist(), s["chosen"].tolist(), s["block_table"].tolist()
        for r, start in enumerate(starts):
            node, kept, a, n = 0, [], cu[r], cu[r + 1] - cu[r]
            while node is not None:
                kept.append(node)
                node = next((c for c in range(node + 1, n) if parents[a + c] == node and tokens[a + c] == chosen[a + node]), None)
            for k, node in enumerate(kept):
                to, back = start + k, start + node
                if to != back:
                    for cache in caches:
                        cache[table[r][to // page], :, :, to % page] = cache[table[r][back // page], :, :, back % page]
        return caches, None, None, None
    nh, nkv, d = s["nh"], s["nkv"], s["d"]
    q = s["qkv"][:, :nh * d].double().view(-1, nh, d)
    out = torch.zeros_like(q)
    for r, start in enumerate(starts):
        a, n = cu[r], cu[r + 1] - cu[r]
        e = torch.arange(start + n, device="cuda")
        rows = s["kv_cache"][s["block_table"][r].long()[e // page], :, :, e % page].double()
        hidden = torch.zeros(n, start + n, dtype=torch.bool)
        for i in range(n):
            hidden[i, start:] = True
            j = i
            while j >= 0:
                hidden[i, start + j] = False
                j = parents[a + j]
        hidden = hidden.cuda()
        for h in range(nh):
            scores = (q[a:a + n, h] @ rows[:, 0, h * nkv // nh].T * s["scale"]).masked_fill_(hidden, -math.inf)
            scores = scores.sub_(scores.amax(1, keepdim=True)).exp_()
            out[a:a + n, h] = scores @ rows[:, 1, h * nkv // nh] / scores.sum(1, keepdim=True)
    return out.view(-1, nh * d)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    """Bytes and operations of the numbers that the case names (ragged ones counted at their mean)."""
    c, half = case, lambda top, least: (top + least) / 2 if case["ragged"] else top  # noqa: E731
    size = 2 if c["dtype"] == "bfloat16" else 4
    nh, nkv, d = c["nh"], c["nkv"], c["d"]
    entry = 2 * nkv * d * size
    if c["op"] == "copy":
        return dict(bytes=int(2 * c["layers"] * c["copies"] * half(c["held"], 1) * entry), flops=0)
    R, rows, context = c["requests"], half(c["rows"], 1), half(c["context"], c["context"] // 2)
    if c["op"] == "layout":
        return dict(bytes=int(R * (4 * rows + 8 + 4 * rows * (1 + -(-c["rows"] // 32)))), flops=int(R * rows))
    # nodes on a path of the tree, on average: some 2 ln(rows) where later nodes are likelier parents
    depth = (rows + 1) / 2 if c["shape"] == "chain" else 1 + 2 * math.log(max(1.0, rows))
    if c["op"] == "keep":
        moved = 0 if c["shape"] == "chain" else min(rows / 2, 2.0)
        return dict(bytes=int(R * (20 * rows + 4 + 2 * moved * c["layers"] * entry)), flops=int(R * rows))
    return dict(bytes=int(R * ((context + rows) * entry + 2 * rows * nh * d * size + 4 * rows * -(-c["rows"] // 32))),
                flops=int(4 * nh * d * R * rows * (context + depth)))
