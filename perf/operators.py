"""Operators over the paged cache that a server of long contexts runs, as cases that can be measured one by one.

``prefix``: attention of single tokens whose requests share a long prefix (a system prompt, a document that several
questions are asked about), computed once for all.  ``weigh``: attention of single tokens that adds up, for every cached
entry, the weight it receives.  ``prompt``: the same sums for portions of prompts, or for the last rows of prompts.
``evict``: the entries with the least of that weight leave the cache.

A cache is [pages, 2, kv heads, page, head size]; request r's entry e is row e % page of page table[r, e // page].  Head
counts, head sizes and page sizes are those of the models that this repository measures and tests.

A case's keys: ``op``; ``dtype``; ``nh``, ``nkv``, ``d``, ``page``; ``rows`` tokens in ``groups`` groups of one prefix of
``prefix`` entries each and ``own`` entries of their own (prefix); ``requests`` that hold ``context`` entries (weigh);
``requests`` with ``rows`` rows behind ``past`` entries (prompt); ``requests`` of ``length`` entries of which ``keep`` stay
(evict); ``ragged``: the lengths differ.
"""
import math

import torch

own = False


def _case(op, dtype="bfloat16", nh=32, nkv=8, d=128, page=16, ragged=False, **sizes):
    return dict(op=op, dtype=dtype, nh=nh, nkv=nkv, d=d, page=page, ragged=ragged, **sizes)


def listed():
    return [
        # two requests of the smallest model in 32-bit behind a short system prompt
        dict(_case("prefix", "float32", 3, 1, 32, 8, True, rows=2, groups=1, prefix=333, own=17), name="prefix-tiny-f32"),
        # a few chats behind one system prompt of a thousand tokens
        dict(_case("prefix", d=64, rows=8, groups=1, prefix=1024, own=128), name="prefix-8"),
        # a busy server: three system prompts, every request at its own length
        dict(_case("prefix", nh=24, ragged=True, rows=96, groups=3, prefix=2500, own=700), name="prefix-groups"),
        # sixty-four questions about one document
        dict(_case("prefix", ragged=True, rows=64, groups=1, prefix=8192, own=512), name="prefix-64"),
        # many samples of answers to one very long prompt
        dict(_case("prefix", rows=128, groups=1, prefix=65536, own=256), name="prefix-long"),
        # three requests of the smallest model in 32-bit
        dict(_case("weigh", "float32", 3, 1, 32, 8, True, requests=3, context=63), name="weigh-tiny-f32"),
        # one user waiting for the next token
        dict(_case("weigh", d=64, requests=1, context=1024), name="weigh-1"),
        # a busy server with long contexts, every request at its own length
        dict(_case("weigh", ragged=True, requests=64, context=4096), name="weigh-64"),
        # a long prompt, all of its rows
        dict(_case("prompt", requests=1, rows=2048, past=0), name="prompt-2048"),
        # the last rows of a batch of long prompts, which say what their answers will look at
        dict(_case("prompt", d=64, ragged=True, requests=8, rows=33, past=6000), name="prompt-window"),
        # every request has grown by a page over its budget
        dict(_case("evict", d=64, requests=64, length=1040, keep=1024), name="evict-step"),
        # long prompts shrink to their budget
        dict(_case("evict", ragged=True, requests=8, length=16384, keep=2048), name="evict-prompts"),
    ]


# query heads, kv heads, head size, page of the models that this repository measures
_HEADS = [(32, 8, 64, 16), (24, 8, 128, 16), (32, 8, 128, 16), (16, 2, 128, 16), (32, 8, 128, 32)]
_TINY = [(3, 1, 32, 8), (4, 2, 16, 16), (4, 2, 64, 16)]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    op = rng.choice(["prefix", "prefix", "weigh", "prompt", "evict"])
    f32 = rng.random() < 0.2
    nh, nkv, d, page = rng.choice(_TINY if f32 else _HEADS)
    c = dict(dtype="float32" if f32 else "bfloat16", nh=nh, nkv=nkv, d=d, page=page, ragged=rng.random() < 0.6)
    top = 64 if f32 else 1                  # the 32-bit path serves small models: shorter by so much
    if op == "prefix":
        rows = size(1, 256 // min(top, 8))
        return _case(op, rows=rows, groups=min(rows, rng.choice([1, 1, 2, 3, 5])), prefix=size(1, min(65536 // top, 8_000_000 // rows)),
                     own=size(1, min(2048 // min(top, 8), 131072 // rows)), **c)
    if op == "weigh":
        requests = size(1, 256 // min(top, 8))
        return _case(op, requests=requests, context=size(1, min(32768 // top, 262144 // requests)), **c)
    if op == "prompt":
        requests = size(1, 16)
        rows = size(1, min(2048 // min(top, 8), 4096 // requests))
        return _case(op, requests=requests, rows=rows, past=size(1, min(16384 // top, 8_000_000 // (requests * rows))), **c)
    requests = size(1, 64 // min(top, 8))
    length = size(2, min(32768 // top, 131072 // requests))
    return _case(op, requests=requests, length=length, keep=size(1, length), **c)


# ---- what a user's program has in hand ------------------------------------------------------------------------------
def _lengths(n, top, ragged, least, gen):
    """n lengths, all ``top``, or between ``least`` and ``top`` with one of them ``top``."""
    if not ragged or n == 0:
        return [top] * n
    v = torch.randint(min(least, top), top + 1, (n,), generator=gen).tolist()
    v[int(torch.randint(0, n, (1,), generator=gen))] = top
    return v


def _tables(pages, lists, width):
    """int32 [len(lists), width]: each list's pages, the rest 0."""
    flat, at = torch.zeros(len(lists), width, dtype=torch.int32), 0
    for i, n in enumerate(lists):
        flat[i, :n] = pages[at:at + n]
        at += n
    return flat.cuda()


def prepare(case, seed):
    c = dict(case)
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, nh, nkv, d, page = getattr(torch, c["dtype"]), c["nh"], c["nkv"], c["d"], c["page"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    pages_of = lambda n: -(-n // page)  # noqa: E731
    s = dict(c, scale=d ** -0.5)
    if c["op"] == "prefix":
        T, NG = c["rows"], c["groups"]
        first = [i * T // NG for i in range(NG + 1)]
        prefix = _lengths(NG, c["prefix"], c["ragged"], c["prefix"] // 2, host)
        have = _lengths(T, c["own"], c["ragged"], 0, host)           # a request may bring nothing of its own yet
        need = [pages_of(n) for n in prefix] + [pages_of(n) for n in have]
        pages = torch.randperm(sum(need) + 3, generator=host).to(torch.int32)
        width, deep = max(need[NG:] + [1]), max(need[:NG])
        tables = _tables(pages, need, max(width, deep))
        s.update(prefix_table=tables[:NG, :deep].contiguous(), block_table=tables[NG:, :width].contiguous(),
                 groups=i32([[first[g], first[g + 1] - first[g], prefix[g]] for g in range(NG)]), positions=i32([n - 1 for n in have]),
                 max_rows=max(first[g + 1] - first[g] for g in range(NG)), max_prefix=max(prefix), max_own=max(have))
        total, rows = sum(need) + 3, T
    else:
        R = c["requests"]
        if c["op"] == "weigh":
            lens = _lengths(R, c["context"], c["ragged"], 1, host)
            rows = R
        elif c["op"] == "prompt":
            counts = _lengths(R, c["rows"], c["ragged"], 1, host)
            past = _lengths(R, c["past"], c["ragged"], c["past"] // 2, host)
            lens = [n + p for n, p in zip(counts, past)]
            rows = sum(counts)
            cu = [0]
            for n in counts:
                cu.append(cu[-1] + n)
            # rows of a portion bring their own entries; the earlier ones' sums go on
            s.update(cu_rows=i32(cu), starts=i32(past), fresh=i32(past), max_rows=max(counts))
        else:
            lens = _lengths(R, c["length"], c["ragged"], c["length"] // 2, host)
            rows = 0
        need = [pages_of(n) for n in lens]
        total = R * pages_of(max(lens)) + 3
        s["block_table"] = _tables(torch.randperm(total, generator=host).to(torch.int32), need, max(need))
        slots = torch.randperm(R + 2, generator=host)[:R].tolist()
        longest = max(lens)
        s.update(slots=i32(slots), max_context=longest, positions=i32([n - 1 for n in lens]))
        # sums of some dozen steps' weights: heavy-tailed
        shape = (R + 2, nkv, -(-(c["rows"] + c["past"] if c["op"] == "prompt" else longest) // 64) * 64)
        s["weights"] = torch.empty(shape, device="cuda").exponential_(generator=gen).square_().mul_(32.0 * nh / nkv / longest)
        if c["op"] == "evict":
            # entries stand in the order in which they came, but for some that earlier evictions have moved
            places = torch.arange(shape[2], device="cuda", dtype=torch.int32).expand(shape).contiguous()
            moved = torch.randperm(max(1, longest // 2), generator=gen, device="cuda")[:longest // 4]
            places[:, :, moved] = moved.flip(0).to(torch.int32)
            s.update(places=places, weights_out=torch.zeros(shape, device="cuda"), places_out=torch.zeros_like(places), lens=i32(lens),
                     keeps=i32([c["keep"]] * R), protect_first=4, protect_last=c["keep"] // 8)
    # queries that look at some keys more than at others
    s["qkv"] = torch.randn(rows, (nh + 2 * nkv) * d, generator=gen, device="cuda").mul_(1.5).to(dtype)
    s["kv_cache"] = torch.randn(total, 2, nkv, page, d, generator=gen, device="cuda", dtype=dtype)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    nh, nkv, d = s["nh"], s["nkv"], s["d"]
    q = s["qkv"][:, :nh * d]                        # the queries' columns of the fused projection
    if not own:
        return _PLAIN[s["op"]](s, q, nh, nkv, nh // nkv, d)
    from railgun_b200 import ops
    if s["op"] == "prefix":
        out = torch.empty(q.shape[0], nh * d, dtype=q.dtype, device=q.device)
        ops.prefix_attention(q, out, s["kv_cache"], s["prefix_table"], s["groups"], s["block_table"], s["positions"], nh, nkv, d,
                             s["scale"], max_rows=s["max_rows"], max_prefix=s["max_prefix"], max_own=s["max_own"])
        return out
    if s["op"] == "weigh":
        out = torch.empty(q.shape[0], nh * d, dtype=q.dtype, device=q.device)
        ops.weighed_attention(q, out, s["kv_cache"], s["weights"], s["slots"], s["block_table"], s["positions"], nh, nkv, d, s["scale"],
                              max_context=s["max_context"], decay=0.99)
        return out, s["weights"]
    if s["op"] == "prompt":
        ops.prompt_key_weights(q, s["kv_cache"], s["weights"], s["slots"], s["block_table"], s["cu_rows"], s["starts"], s["fresh"],
                               nh, nkv, d, s["scale"], max_rows=s["max_rows"], max_context=s["max_context"])
        return s["weights"]
    lens = ops.evict_entries(s["kv_cache"], s["weights"], s["places"], s["weights_out"], s["places_out"], s["slots"], s["block_table"],
                             s["lens"], s["keeps"], s["positions"], nkv, d, s["protect_first"], s["protect_last"],
                             max_context=s["max_context"])
    return s["kv_cache"], s["weights_out"], s["places_out"], lens


def _entries(cache, table):
    """Keys and values of the tables' entries in 32 bits, each [tables, kv heads, entries, d]."""
    rows = cache[table.long()].float().permute(2, 0, 3, 1, 4, 5)       # 2, tables, heads, pages, page, d
    return rows.reshape(2, table.shape[0], rows.shape[2], -1, rows.shape[5])


def _partial(q, kv, seen, scale):
    """Attention without its division: (largest score, sum of weights, weighted sum of values) of queries [.., m, d] over keys
    and values [2, .., n, d], of which ``seen`` [.., m, n] are looked at."""
    scores = (q @ kv[0].transpose(-1, -2)) * scale
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.max(-1, keepdim=True).values
    weights = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    return top, weights.sum(-1, keepdim=True), weights @ kv[1]


def _plain_prefix(s, q, nh, nkv, G, d):
    T, groups = q.shape[0], s["groups"].long()
    q = q.float().reshape(T, nkv, G, d)
    # the rows of a group side by side: [groups, most rows]
    at = torch.arange(s["max_rows"], device=q.device)
    rows = (groups[:, :1] + at).clamp(max=T - 1)
    side = q[rows].permute(0, 2, 1, 3, 4).reshape(len(groups), nkv, -1, d)
    kv = _entries(s["kv_cache"], s["prefix_table"])
    seen = torch.arange(kv.shape[3], device=q.device) < groups[:, 2, None]
    part = [x.reshape(len(groups), nkv, s["max_rows"], G, -1).permute(0, 2, 1, 3, 4)
            for x in _partial(side, kv, seen[:, None, None, :], s["scale"])]
    row = torch.arange(T, device=q.device)
    group = (row[:, None] >= groups[:, 0]).sum(1) - 1
    top1, sum1, out1 = (x[group, row - groups[group, 0]] for x in part)
    kv = _entries(s["kv_cache"], s["block_table"])
    seen = torch.arange(kv.shape[3], device=q.device) <= s["positions"][:, None]
    top2, sum2, out2 = _partial(q, kv, seen[:, None, None, :], s["scale"])
    top = torch.maximum(top1, top2)
    top = torch.where(top == float("-inf"), 0.0, top)
    a, b = torch.exp(top1 - top), torch.exp(top2 - top)
    total = a * sum1 + b * sum2
    out = torch.where(total > 0, (a * out1 + b * out2) / total, 0.0)
    return out.reshape(T, nh * d).to(s["qkv"].dtype)


def _plain_weigh(s, q, nh, nkv, G, d):
    R = q.shape[0]
    kv = _entries(s["kv_cache"], s["block_table"])
    entry = torch.arange(kv.shape[3], device=q.device)
    position = s["positions"].long()[:, None]
    scores = (q.float().reshape(R, nkv, G, d) @ kv[0].transpose(-1, -2)) * s["scale"]
    scores = torch.where((entry <= position)[:, None, None, :], scores, float("-inf"))
    weights = torch.exp(scores - scores.max(-1, keepdim=True).values)
    weights = weights / weights.sum(-1, keepdim=True)
    out = (weights @ kv[1]).reshape(R, nh * d).to(s["qkv"].dtype)
    n = s["max_context"]
    slots, entry = s["slots"].long(), entry[:n]
    before = s["weights"][slots, :, :n]
    added = torch.where((entry < position)[:, None, :], 0.99 * before, 0.0) + weights.sum(2)[..., :n]
    s["weights"][slots, :, :n] = torch.where((entry <= position)[:, None, :], added, before)
    return out, s["weights"]


def _plain_prompt(s, q, nh, nkv, G, d):
    R, n = s["slots"].numel(), s["max_context"]
    kv = _entries(s["kv_cache"], s["block_table"])
    entry, at = torch.arange(kv.shape[3], device=q.device), torch.arange(s["max_rows"], device=q.device)
    cu, starts = s["cu_rows"].long(), s["starts"].long()
    count = cu[1:] - cu[:-1]
    rows = (cu[:-1, None] + at).clamp(max=q.shape[0] - 1)
    side = q.float().reshape(-1, nkv, G, d)[rows].permute(0, 2, 3, 1, 4)                # requests, kv heads, heads, rows, d
    scores = (side @ kv[0][:, :, None].transpose(-1, -2)) * s["scale"]
    seen = (entry <= (starts[:, None] + at)[..., None])[:, None, None]
    scores = torch.where(seen, scores, float("-inf"))
    weights = torch.exp(scores - scores.max(-1, keepdim=True).values)
    weights = weights / weights.sum(-1, keepdim=True)
    there = (at < count[:, None])[:, None, None, :, None]
    added = torch.where(there, weights, 0.0).sum((2, 3))[..., :n]
    slots, entry = s["slots"].long(), entry[:n]
    before = s["weights"][slots, :, :n]
    after = torch.where((entry < s["fresh"].long()[:, None])[:, None, :], before, 0.0) + added
    s["weights"][slots, :, :n] = torch.where((entry < (starts + count)[:, None])[:, None, :], after, before)
    return s["weights"]


def _plain_evict(s, q, nh, nkv, G, d):
    cache, page = s["kv_cache"], s["page"]
    R, n = s["slots"].numel(), s["max_context"]
    slots, lens, keeps = s["slots"].long(), s["lens"].long(), s["keeps"].long()
    entry = torch.arange(n, device=cache.device)
    weights, places = s["weights"][slots, :, :n], s["places"][slots, :, :n]
    there = (entry < lens[:, None])[:, None, :].expand(R, nkv, n)
    safe = (places < s["protect_first"]) | (places > (s["positions"] - s["protect_last"])[:, None, None]) | weights.isnan()
    rank = torch.where(there, torch.where(safe, float("inf"), weights), float("-inf"))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    new = torch.minimum(lens, keeps)
    stays = torch.zeros(R, nkv, n, dtype=torch.bool, device=cache.device)
    stays.scatter_(2, order, (entry < new[:, None])[:, None, :].expand(R, nkv, n))
    front = (entry < new[:, None])[:, None, :]
    # the i-th entry behind the new length that stays goes into the i-th place before it that got free
    free, late = front & ~stays, stays & ~front
    r, h, to = free.nonzero(as_tuple=True)
    _, _, back = late.nonzero(as_tuple=True)
    table = s["block_table"].long()
    cache[table[r, to // page], :, h, to % page] = cache[table[r, back // page], :, h, back % page]
    for new_values, values in ((s["weights_out"], weights), (s["places_out"], places)):
        values = values.clone()
        values[r, h, to] = values[r, h, back]
        new_values[slots, :, :n] = torch.where(front, values, new_values[slots, :, :n])
    return cache, s["weights_out"], s["places_out"], new.to(torch.int32)


_PLAIN = dict(prefix=_plain_prefix, weigh=_plain_weigh, prompt=_plain_prompt, evict=_plain_evict)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    nh, nkv, d, page = s["nh"], s["nkv"], s["d"], s["page"]
    G, cache = nh // nkv, s["kv_cache"]
    q = s["qkv"][:, :nh * d].double().view(-1, nh, d)

    def entries(table, n):
        """keys, values [kv heads, n, d] of a table's first n entries"""
        e = torch.arange(n, device="cuda")
        rows = cache[table.long()[e // page], :, :, e % page].double()
        return rows[:, 0].transpose(0, 1), rows[:, 1].transpose(0, 1)

    def softmax(x):
        x = (x - x.amax(-1, keepdim=True)).exp_()
        return x.div_(x.sum(-1, keepdim=True))

    if s["op"] == "prefix":
        out = torch.zeros(len(q), nh, d, dtype=torch.float64, device="cuda")
        positions = s["positions"].tolist()
        for g, (first, n, P) in enumerate(s["groups"].tolist()):
            Kp, Vp = entries(s["prefix_table"][g], P)
            for t in range(first, first + n):
                Ko, Vo = entries(s["block_table"][t], positions[t] + 1)
                for k in range(nkv):
                    mine = q[t, k * G:(k + 1) * G] * s["scale"]
                    p = softmax(torch.cat([mine @ Kp[k].T, mine @ Ko[k].T], 1))
                    out[t, k * G:(k + 1) * G] = p[:, :P] @ Vp[k] + p[:, P:] @ Vo[k]
        return out.view(len(q), nh * d)
    weights = s["weights"].double()
    slots = s["slots"].tolist()
    if s["op"] == "weigh":
        out = torch.zeros(len(q), nh, d, dtype=torch.float64, device="cuda")
        for r, p in enumerate(s["positions"].tolist()):
            K, V = entries(s["block_table"][r], p + 1)
            a = softmax(q[r].view(nkv, G, d) @ K.transpose(1, 2) * s["scale"])
            out[r] = (a @ V).view(nh, d)
            mine = weights[slots[r], :, :p + 1]
            mine *= 0.99
            mine[:, p] = 0.0
            mine += a.sum(1)
        return out.view(len(q), nh * d), weights
    if s["op"] == "prompt":
        cu = s["cu_rows"].tolist()
        for r, (start, fresh) in enumerate(zip(s["starts"].tolist(), s["fresh"].tolist())):
            n = cu[r + 1] - cu[r]
            K, _ = entries(s["block_table"][r], start + n)
            later = torch.arange(start + n, device="cuda") > torch.arange(start, start + n, device="cuda")[:, None]
            mine = weights[slots[r], :, :start + n]
            mine[:, fresh:] = 0.0
            for h in range(nh):
                scores = q[cu[r]:cu[r + 1], h] @ K[h // G].T * s["scale"]
                mine[h // G] += softmax(scores.masked_fill_(later, float("-inf"))).sum(0)
        return weights
    # evict: one row at a time, by counting how many entries come before each
    if cache.numel() > 1 << 28 or sum(s["lens"].tolist()) * nkv > 1 << 20:
        return None
    cache = cache.double()
    weights_out, places_out = s["weights_out"].double(), s["places_out"].clone()
    new = s["lens"].clone()
    for r, (n, keep, newest) in enumerate(zip(s["lens"].tolist(), s["keeps"].tolist(), s["positions"].tolist())):
        k = min(n, keep)
        new[r] = k
        table = s["block_table"][r].long().cpu()
        for h in range(nkv):
            w, pl = weights[slots[r], h, :n].cpu(), s["places"][slots[r], h, :n].cpu()
            w = torch.where((pl < s["protect_first"]) | (pl > newest - s["protect_last"]), math.inf, w)
            best = sorted(range(n), key=lambda e: (-float(w[e]), e))[:k]
            stays = set(best)
            holes = [e for e in range(k) if e not in stays]
            late = sorted(e for e in best if e >= k)
            source = list(range(k))
            for a, b in zip(holes, late):
                source[a] = b
            a, b = torch.tensor(holes, dtype=torch.long), torch.tensor(late, dtype=torch.long)
            cache[table[a // page].cuda(), :, h, (a % page).cuda()] = cache[table[b // page].cuda(), :, h, (b % page).cuda()]
            source = torch.tensor(source, dtype=torch.long).cuda()
            weights_out[slots[r], h, :k] = weights[slots[r], h][source]
            places_out[slots[r], h, :k] = s["places"][slots[r], h][source]
    return cache, weights_out, places_out, new


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    """Bytes and operations of the lengths that the case names (ragged lengths counted at their mean)."""
    c, half = case, lambda top, least: (top + least) / 2 if case["ragged"] else top  # noqa: E731
    size = 2 if c["dtype"] == "bfloat16" else 4
    nh, nkv, d = c["nh"], c["nkv"], c["d"]
    entry = 2 * nkv * d * size
    if c["op"] == "prefix":
        prefix, mine = half(c["prefix"], c["prefix"] // 2), half(c["own"], 0)
        return dict(bytes=int(c["groups"] * prefix * entry + c["rows"] * mine * entry + 2 * c["rows"] * nh * d * size),
                    flops=int(4 * nh * d * c["rows"] * (prefix + mine)))
    if c["op"] == "weigh":
        n = half(c["context"], 1)
        return dict(bytes=int(c["requests"] * (n * entry + 2 * n * nkv * 4 + 2 * nh * d * size)), flops=int(4 * nh * d * c["requests"] * n))
    if c["op"] == "prompt":
        rows, past = half(c["rows"], 1), half(c["past"], c["past"] // 2)
        return dict(bytes=int(c["requests"] * (rows * nh * d * size + (rows + past) * (entry / 2 + 2 * nkv * 4))),
                    flops=int(2 * nh * d * c["requests"] * rows * (past + (rows + 1) / 2)))
    n = half(c["length"], c["length"] // 2)
    k = min(n, c["keep"])
    moved = k * (n - k) / max(n, 1)                # of entries with unordered weights that many stand behind the new length
    return dict(bytes=int(c["requests"] * nkv * (8 * n + 8 * k + moved * 4 * d * size)), flops=int(c["requests"] * nkv * n))
