"""Operators over the paged cache against the formulas in 64 bits: attention behind shared prefixes, attention that adds up
the weights its entries receive, the same sums for portions of prompts, and eviction by them.

Rows of the cache that no table names, and those behind the last entry of a page, hold NaN: none of them may have a say.
"""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24                                   # half a unit in the last place of a 32-bit number at 1


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    from railgun_b200 import ops
    ops.tc_gemm_check()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Cache:
    """Pages of NaN, and lists of entries with numbers in them."""

    def __init__(self, lens, nkv, d, page, dtype, g, spare=2, width=1):
        self.page, need = page, [-(-n // page) for n in lens]
        total = sum(need) + spare
        pages = torch.randperm(total, device=DEV, generator=g)
        self.kv = torch.full((total, 2, nkv, page, d), float("nan"), dtype=dtype, device=DEV)
        self.table = torch.randint(0, total, (len(lens), max(need + [width])), device=DEV, generator=g).to(torch.int32)
        at = 0
        for i, n in enumerate(lens):
            self.table[i, :need[i]] = pages[at:at + need[i]].to(torch.int32)
            at += need[i]
            e = torch.arange(n, device=DEV)
            self.kv[self.table[i].long()[e // page], :, :, e % page] = torch.randn(n, 2, nkv, d, device=DEV, generator=g).to(dtype)

    def entries(self, i, n):
        """keys and values [nkv, n, d] of list i in 64 bits"""
        e = torch.arange(n, device=DEV)
        rows = self.kv[self.table[i].long()[e // self.page], :, :, e % self.page].double()
        return rows[:, 0].transpose(0, 1), rows[:, 1].transpose(0, 1)


def queries(T, nh, d, dtype, g, more=8):
    """Rows further apart than their width."""
    return torch.randn(T, nh * d + more, device=DEV, generator=g).mul_(1.5).to(dtype)[:, :nh * d]


def out_view(T, n, dtype):
    return torch.full((T, n + 8), 7.0, dtype=dtype, device=DEV)[:, :n]


def score_error(q, K, scale, dtype):
    """How far a score may be off: d terms added in 32 bits (a tensor core's sums are cut, not rounded: twice that)."""
    G = q.shape[0] // K.shape[0]
    size = (q.double().abs().view(K.shape[0], G, -1) @ K.abs().transpose(1, 2)).max().item() * scale if K.shape[1] else 0.0
    return (q.shape[1] + 4) * (2 * U if dtype == torch.bfloat16 else U) * size


def weight_error(q, K, n, scale, dtype):
    """The relative error of a softmax weight: its score's and the sum's, 2^x good to 2 units in the last place (and what the
    argument of 2^x, up to some 40, loses), sums of n terms."""
    return 4 * score_error(q, K, scale, dtype) + (2 * n + 400) * U


def softmax(x):
    if x.shape[-1] == 0:
        return x
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return x / x.sum(-1, keepdim=True)


def out_error(q, K, V, n, scale, dtype):
    """An output is a mean of values under weights that are off by weight_error (in bfloat16 also rounded, 2^-9), added up in 32
    bits and rounded to its type."""
    if n == 0:
        return 0.0
    top = V.abs().max().item()
    return top * (weight_error(q, K, n, scale, dtype) + (2 * n + 8) * U + (2.0 ** -8 + 2.0 ** -9 if dtype == torch.bfloat16 else 2 * U))


HEADS = [(3, 1, 32, 8), (4, 4, 64, 16), (8, 2, 128, 32), (32, 8, 64, 16), (20, 1, 16, 7), (12, 1, 128, 64), (6, 2, 24, 5), (2, 1, 256, 16),
         (5, 5, 80, 16), (40, 1, 64, 128)]
TYPES = [torch.float32, torch.bfloat16]


# ---- attention behind shared prefixes ---------------------------------------------------------------------------------
# groups of (rows, prefix entries), own entries of every row; the second number of a scenario is how many rows belong to no group
SCENES = {
    "one row": ([(1, 1)], 0, [0]),
    "nothing at all": ([(2, 0)], 1, [0, 0, 0]),
    "no prefix": ([(3, 0)], 0, [1, 64, 65]),
    "no group": ([], 4, [0, 1, 300, 17]),
    "nothing of their own": ([(9, 130)], 0, [0] * 9),
    "three groups": ([(2, 65), (1, 0), (7, 201)], 2, [3, 0, 9, 31, 0, 64, 63, 129, 1, 16, 0, 5]),
    "many rows": ([(70, 77), (3, 640)], 1, [i * 7 % 40 for i in range(74)]),
    "long": ([(5, 3001)], 0, [700, 0, 1, 128, 333]),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scene", SCENES)
@pytest.mark.parametrize("nh,nkv,d,page", HEADS)
def test_prefix_attention(nh, nkv, d, page, scene, dtype):
    from railgun_b200 import ops
    groups, alone, own = SCENES[scene]
    g = torch.Generator(device=DEV).manual_seed(len(scene) * nh + d)
    T, prefixes = len(own), [p for _, p in groups]
    assert sum(n for n, _ in groups) + alone == T
    cache = Cache(prefixes + own, nkv, d, page, dtype, g)
    q, scale, G = queries(T, nh, d, dtype, g), d ** -0.5, nh // nkv
    first, table = 0, []
    for n, p in groups:
        table.append([first, n, p])
        first += n
    out = out_view(T, nh * d, dtype)
    args = (cache.kv, cache.table[:len(groups)].contiguous(), i32(table).view(-1, 3), cache.table[len(groups):].contiguous(),
            i32([n - 1 for n in own]), nh, nkv, d, scale)
    sizes = dict(max_rows=max([n for n, _ in groups] + [0]), max_prefix=max(prefixes + [0]), max_own=max(own))
    ops.prefix_attention(q, out, *args, **sizes)
    of = {t: i for i, (a, n, _) in enumerate(table) for t in range(a, a + n)}
    for t in range(T):
        i = of.get(t)
        P = prefixes[i] if i is not None else 0
        Kp, Vp = cache.entries(i or 0, P)
        Ko, Vo = cache.entries(len(groups) + t, own[t])
        K, V = torch.cat([Kp, Ko], 1), torch.cat([Vp, Vo], 1)
        mine = q[t].reshape(nh, d)
        want = softmax(mine.double().view(nkv, G, d) @ K.transpose(1, 2) * scale) @ V
        off = (out[t].double().view(nkv, G, d) - want).abs().max().item()
        assert off <= out_error(mine, K, V, P + own[t], scale, dtype), (t, off)
    again = torch.empty(T, nh * d, dtype=dtype, device=DEV)
    # more room than there is need for, on another stream: the sums may be cut elsewhere, the result is the same to their rounding
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.prefix_attention(q, again, *args, **{k: v + 100 for k, v in sizes.items()})
        twice = torch.empty_like(again)
        ops.prefix_attention(q, twice, *args, **{k: v + 100 for k, v in sizes.items()})
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(again, twice)
    assert (again.double() - out.double()).abs().max() <= (2.0 ** -6 if dtype == torch.bfloat16 else 1e-5) * max(1.0, out.double().abs().max().item())


# ---- weights that entries receive from single tokens -----------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1], [0, 5], [64, 63, 65, 1, 0, 200], [2049, 3, 700]])
@pytest.mark.parametrize("nh,nkv,d,page", HEADS)
def test_weighed_attention(nh, nkv, d, page, lens, dtype):
    from railgun_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(len(lens) * nh + d)
    R, most, G, scale = len(lens), max(lens), nh // nkv, d ** -0.5
    cache = Cache(lens, nkv, d, page, dtype, g)
    q, out = queries(R, nh, d, dtype, g), out_view(R, nh * d, dtype)
    slots = list(range(R + 1, 1, -1))
    if R > 2:
        slots[2] = -1                                                 # nobody keeps this row's weights
    weights = torch.rand(R + 3, nkv, most + 3, device=DEV, generator=g)
    for r, n in enumerate(lens):
        weights[slots[r], :, max(n - 1, 0)] = float("nan")             # the newest entry has no weight yet
    before, first = weights.clone(), weights.clone()
    args = (cache.kv, weights, i32(slots), cache.table, i32([n - 1 for n in lens]), nh, nkv, d, scale)
    ops.weighed_attention(q, out, *args, max_context=most, decay=0.75)
    want_w = before.double()
    for r, n in enumerate(lens):
        K, V = cache.entries(r, n)
        mine = q[r].reshape(nh, d)
        p = softmax(mine.double().view(nkv, G, d) @ K.transpose(1, 2) * scale)
        assert (out[r].double().view(nkv, G, d) - p @ V).abs().max().item() <= out_error(mine, K, V, n, scale, dtype)
        if slots[r] < 0 or n == 0:
            continue
        want = p.sum(1)
        want[:, :-1] += 0.75 * before[slots[r], :, :n - 1].double()
        off = (weights[slots[r], :, :n].double() - want).abs() / want.clamp(min=1e-30)
        assert off.max().item() <= weight_error(mine, K, n, scale, dtype) + (G + 3) * U
        want_w[slots[r], :, :n] = weights[slots[r], :, :n].double()
    assert torch.equal(torch.nan_to_num(weights.double(), nan=-1.0), torch.nan_to_num(want_w, nan=-1.0))      # the rest is as it was
    second = torch.empty(R, nh * d, dtype=dtype, device=DEV)
    ops.weighed_attention(q, second, cache.kv, first, *args[2:], max_context=most, decay=0.75)
    assert torch.equal(second, out) and torch.equal(torch.nan_to_num(first, nan=-1.0), torch.nan_to_num(weights, nan=-1.0))


# ---- weights that entries receive from portions ----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,starts,fresh", [([1], [0], [0]), ([3, 0, 1], [0, 5, 64], [0, 5, 64]), ([70, 129, 2], [0, 300, 63], [0, 300, 0]),
                                               ([33, 64], [1000, 191], [2000, 0]), ([260], [0], [0])])
@pytest.mark.parametrize("nh,nkv,d,page", HEADS)
def test_prompt_key_weights(nh, nkv, d, page, rows, starts, fresh, dtype):
    from railgun_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(sum(rows) * nh + d)
    R, lens, G, scale = len(rows), [n + s for n, s in zip(rows, starts)], nh // nkv, d ** -0.5
    cache = Cache(lens, nkv, d, page, dtype, g)
    q = queries(sum(rows), nh, d, dtype, g)
    slots = list(range(R, 0, -1))
    if R > 2:
        slots[2] = -1
    most = max(lens)
    weights = torch.rand(R + 2, nkv, most + 5, device=DEV, generator=g)
    for r in range(R):
        weights[slots[r], :, fresh[r]:lens[r]] = float("nan")
    before, cu = weights.clone(), [0, *itertools.accumulate(rows)]
    args = (i32(slots), cache.table, i32(cu), i32(starts), i32(fresh), nh, nkv, d, scale)
    sizes = dict(max_rows=max(rows), max_context=most)
    ops.prompt_key_weights(q, cache.kv, weights, *args, **sizes)
    want_w = before.double()
    for r in range(R):
        n = lens[r]
        if slots[r] < 0 or rows[r] == 0:
            continue
        K, _ = cache.entries(r, n)
        mine = q[cu[r]:cu[r + 1]].reshape(rows[r], nkv, G, d).permute(1, 2, 0, 3)
        s = mine.double() @ K[:, None].transpose(2, 3) * scale
        later = torch.arange(n, device=DEV) > torch.arange(starts[r], n, device=DEV)[:, None]
        p = softmax(s.masked_fill(later, float("-inf"))).sum((1, 2))
        want = p.clone()
        want[:, :fresh[r]] += before[slots[r], :, :min(fresh[r], n)].double()
        off = (weights[slots[r], :, :n].double() - want).abs() / want
        flat = q[cu[r]:cu[r + 1]].reshape(rows[r], nkv, G, d).transpose(0, 1).reshape(-1, d)
        assert off.max().item() <= weight_error(flat, K, n, scale, dtype) + (rows[r] * G + 3) * U
        want_w[slots[r], :, :n] = weights[slots[r], :, :n].double()
    assert torch.equal(torch.nan_to_num(weights.double(), nan=-1.0), torch.nan_to_num(want_w, nan=-1.0))
    again = before.clone()
    ops.prompt_key_weights(q, cache.kv, again, *args, **sizes)
    assert torch.equal(torch.nan_to_num(again, nan=-1.0), torch.nan_to_num(weights, nan=-1.0))


def test_portions_and_single_tokens_agree():
    """Rows one at a time, each with the weights of the single tokens' operator, and all at once."""
    from railgun_b200 import ops
    nh, nkv, d, page, n, past = 8, 2, 64, 16, 9, 100
    g = torch.Generator(device=DEV).manual_seed(1)
    for dtype in TYPES:
        cache = Cache([past + n], nkv, d, page, dtype, g)
        q, slots = queries(n, nh, d, dtype, g), i32([0])
        start = torch.rand(1, nkv, past + n, device=DEV, generator=g)
        one, all_ = start.clone(), start.clone()
        out = torch.empty(1, nh * d, dtype=dtype, device=DEV)
        for i in range(n):
            ops.weighed_attention(q[i:i + 1], out, cache.kv, one, slots, cache.table, i32([past + i]), nh, nkv, d, d ** -0.5,
                                  max_context=past + n)
        ops.prompt_key_weights(q, cache.kv, all_, slots, cache.table, i32([0, n]), i32([past]), i32([past]), nh, nkv, d, d ** -0.5,
                               max_rows=n, max_context=past + n)
        K, _ = cache.entries(0, past + n)
        bound = 2 * weight_error(q.reshape(n, nkv, 4, d).transpose(0, 1).reshape(-1, d), K, past + n, d ** -0.5, dtype) + 2 * n * 8 * U
        assert ((one - all_).abs() / all_).max() <= bound


# ---- eviction --------------------------------------------------------------------------------------------------------
def plain_evict(cache, weights, places, slots, lens, keep, newest, first, last):
    """(cache, weights, places, lens) after it, one head at a time, by sorting."""
    kv, new = cache.kv.clone(), []
    w_out, p_out = weights.clone(), places.clone()
    for r, n in enumerate(lens):
        k = min(n, keep[r])
        new.append(k if slots[r] >= 0 else n)
        if slots[r] < 0:
            continue
        table = cache.table[r].tolist()
        for h in range(kv.shape[2]):
            w, p = weights[slots[r], h, :n].tolist(), places[slots[r], h, :n].tolist()
            rank = [math.inf if p[e] < first or p[e] > newest[r] - last or math.isnan(w[e]) else w[e] for e in range(n)]
            stay = sorted(sorted(range(n), key=lambda e: (-rank[e], e))[:k])
            free = [e for e in range(k) if e not in set(stay)]
            late = [e for e in stay if e >= k]
            assert len(free) == len(late)
            w_out[slots[r], h, :k], p_out[slots[r], h, :k] = weights[slots[r], h, :k], places[slots[r], h, :k]
            for a, b in zip(free, late):
                pa, pb = table[a // cache.page], table[b // cache.page]
                kv[pa, :, h, a % cache.page] = cache.kv[pb, :, h, b % cache.page]
                w_out[slots[r], h, a], p_out[slots[r], h, a] = weights[slots[r], h, b], places[slots[r], h, b]
    return kv, w_out, p_out, new


def same(a, b):
    """The same bits but for which NaN it is."""
    return torch.equal(torch.nan_to_num(a.float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nkv,d,page", [(1, 32, 8), (2, 64, 16), (3, 5, 7), (8, 128, 32), (1, 24, 5)])
@pytest.mark.parametrize("lens,keep", [([1, 0, 2], [1, 3, 1]), ([100, 33, 64, 65], [50, 33, 0, 64]), ([700], [699]), ([1500, 1499], [1, 400]),
                                       ([4000, 17, 2600], [1000, 90, 2599])])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evict_entries(nkv, d, page, lens, keep, kind, dtype):
    from railgun_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(sum(lens) + d)
    R, most = len(lens), max(lens)
    cache = Cache(lens, nkv, d, page, dtype, g)
    shape = (R + 2, nkv, most + 4)
    weights = torch.empty(shape, device=DEV).exponential_(generator=g)
    if kind == "ties":
        weights = (weights * 2).floor() / 4                            # a handful of values, zeros of both signs
        weights[:, :, ::3] *= -1.0
    if kind == "odd":
        flat = weights.view(-1)
        at = torch.randperm(flat.numel(), device=DEV, generator=g)
        for j, v in enumerate([float("nan"), float("inf"), float("-inf"), -3.0, 1e-42, 3e38, 0.0, -0.0]):
            flat[at[j::23]] = v
    places = torch.randint(0, 2 * most + 1, shape, device=DEV, generator=g, dtype=torch.int32)
    slots = list(range(R, 0, -1))
    if R == 4:
        slots[1] = -1
    newest = [2 * most - r for r in range(R)]
    first, last = (3, 40) if kind != "ties" else (0, 0)
    want = plain_evict(cache, weights, places, slots, lens, keep, newest, first, last)
    w_out, p_out, before = weights.clone(), places.clone(), cache.kv.clone()
    new = ops.evict_entries(cache.kv, weights, places, w_out, p_out, i32(slots), cache.table, i32(lens), i32(keep), i32(newest), nkv, d,
                            first, last, max_context=most)
    assert new.tolist() == want[3]
    assert same(w_out, want[1]) and torch.equal(p_out, want[2])
    assert same(cache.kv, want[0])
    # in place: the same but for what lies behind the new lengths, which stays as it was
    cache.kv.copy_(before)
    ops.evict_entries(cache.kv, weights, places, weights, places, i32(slots), cache.table, i32(lens), i32(keep), i32(newest), nkv, d,
                      first, last, max_context=most)
    assert same(weights, want[1]) and torch.equal(places, want[2]) and same(cache.kv, want[0])


@pytest.mark.parametrize("n,keep", [(70000, 30000), (420000, 1234)])
def test_evict_long(n, keep):
    """More entries than one block, and than eight blocks, keep in their shared memory."""
    from railgun_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(n)
    nkv, d, page = 1, 8, 64
    cache = Cache([n], nkv, d, page, torch.bfloat16, g)
    weights = torch.empty(1, nkv, n, device=DEV).exponential_(generator=g)
    weights[:, :, ::5] = 0.5                                           # many ties around the border
    places = torch.arange(n, device=DEV, dtype=torch.int32).view(1, 1, n).contiguous()
    rank = torch.where((places < 4) | (places > n - 1 - 64), float("inf"), weights)[0, 0]
    stay = torch.zeros(n, dtype=torch.bool, device=DEV)
    stay[torch.sort(rank, descending=True, stable=True).indices[:keep]] = True
    free, late = (~stay[:keep]).nonzero()[:, 0], stay[keep:].nonzero()[:, 0] + keep
    source = torch.arange(keep, device=DEV)
    source[free] = late
    table, before = cache.table[0].long(), cache.kv.clone()
    w_out, p_out = torch.zeros_like(weights), torch.zeros_like(places)
    new = ops.evict_entries(cache.kv, weights, places, w_out, p_out, i32([0]), cache.table, i32([n]), i32([keep]), i32([n - 1]), nkv, d, 4, 64,
                            max_context=n)
    assert new.tolist() == [keep]
    assert torch.equal(w_out[0, 0, :keep], weights[0, 0, source]) and torch.equal(p_out[0, 0, :keep], places[0, 0, source])
    e = torch.arange(keep, device=DEV)
    assert torch.equal(cache.kv[table[e // page], :, 0, e % page], before[table[source // page], :, 0, source % page])
    e = torch.arange(keep, n, device=DEV)
    assert torch.equal(cache.kv[table[e // page], :, 0, e % page], before[table[e // page], :, 0, e % page])


# ---- together, far addresses, refusals --------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
def test_far_pages(dtype):
    """Pages more than 2^31 elements into the cache."""
    from railgun_b200 import ops
    nh, nkv, d, page, n = 4, 2, 64, 16, 90
    per = 2 * nkv * page * d
    total = (1 << 31) // per + 40
    g = torch.Generator(device=DEV).manual_seed(3)
    small = Cache([n], nkv, d, page, dtype, g, spare=0)
    kv = torch.empty(total, 2, nkv, page, d, dtype=dtype, device=DEV)
    kv[-small.kv.shape[0]:] = small.kv
    table = small.table + (total - small.kv.shape[0])
    q, none, zero = queries(1, nh, d, dtype, g), i32([-1]), i32([0])
    rows = {}
    for name, c, tb in (("near", small.kv, small.table), ("far", kv, table)):
        a, b = (torch.empty(1, nh * d, dtype=dtype, device=DEV) for _ in range(2))
        w, w2 = (torch.zeros(1, nkv, n, device=DEV) for _ in range(2))
        ops.prefix_attention(q, a, c, tb, i32([[0, 1, n]]), tb, none, nh, nkv, d, 0.125, max_rows=1, max_prefix=n, max_own=0)
        ops.weighed_attention(q, b, c, w, zero, tb, i32([n - 1]), nh, nkv, d, 0.125, max_context=n)
        ops.prompt_key_weights(q, c, w2, zero, tb, i32([0, 1]), i32([n - 1]), zero, nh, nkv, d, 0.125, max_rows=1, max_context=n)
        places = torch.arange(n, device=DEV, dtype=torch.int32).expand(1, nkv, n).contiguous()
        wo, po = torch.zeros_like(w), torch.zeros_like(places)
        ops.evict_entries(c, w, places, wo, po, zero, tb, i32([n]), i32([30]), i32([n - 1]), nkv, d, 2, 5, max_context=n)
        rows[name] = (a, b, w, w2, wo, po, c[tb[0].long()])
    for x, y in zip(rows["near"], rows["far"]):
        assert same(x, y)


def _good(dtype=torch.bfloat16, nh=4, nkv=2, d=64, page=16, R=2, n=40):
    g = torch.Generator(device=DEV).manual_seed(0)
    c = Cache([n] * R, nkv, d, page, dtype, g)
    z = torch.zeros(R, nkv, n, device=DEV)
    return dict(q=queries(R, nh, d, dtype, g), out=torch.empty(R, nh * d, dtype=dtype, device=DEV), kv=c.kv, table=c.table, pos=i32([n - 1] * R),
                slots=i32([0, 1]), w=z, w2=z.clone(), p=z.int(), p2=z.int(), lens=i32([n] * R), keep=i32([8] * R), groups=i32([[0, 2, 8]]),
                ptable=c.table[:1].contiguous(), cu=i32([0, 1, 2]), nh=nh, nkv=nkv, d=d, n=n)


def _prefix(ops, a):
    ops.prefix_attention(a["q"], a["out"], a["kv"], a["ptable"], a["groups"], a["table"], a["pos"], a["nh"], a["nkv"], a["d"], 0.125,
                         max_rows=2, max_prefix=8, max_own=a["n"])


def _weigh(ops, a):
    ops.weighed_attention(a["q"], a["out"], a["kv"], a["w"], a["slots"], a["table"], a["pos"], a["nh"], a["nkv"], a["d"], 0.125,
                          max_context=a["n"])


def _prompt(ops, a):
    ops.prompt_key_weights(a["q"], a["kv"], a["w"], a["slots"], a["table"], a["cu"], a["pos"], a["pos"], a["nh"], a["nkv"], a["d"], 0.125,
                           max_rows=1, max_context=a["n"])


def _evict(ops, a):
    ops.evict_entries(a["kv"], a["w"], a["p"], a["w2"], a["p2"], a["slots"], a["table"], a["lens"], a["keep"], a["pos"], a["nkv"], a["d"], 1, 1,
                      max_context=a["n"])


BAD = [("q", lambda a: a["q"].cpu(), "pwk"), ("q", lambda a: a["q"].half(), "pwk"), ("q", lambda a: a["q"].float(), "pwk"),
       ("q", lambda a: a["q"][:, :100], "pwk"), ("q", lambda a: a["q"].t().contiguous().t(), "pwk"), ("out", lambda a: a["out"].float(), "pw"),
       ("out", lambda a: a["out"][:1], "pw"), ("kv", lambda a: a["kv"][:, :, :1], "pwke"), ("kv", lambda a: a["kv"].cpu(), "pwke"),
       ("kv", lambda a: a["kv"].half(), "pwke"), ("kv", lambda a: a["kv"].transpose(0, 3), "pwke"), ("table", lambda a: a["table"].long(), "pwke"),
       ("table", lambda a: a["table"][:1], "pwke"), ("pos", lambda a: a["pos"][:1], "pwke"), ("pos", lambda a: a["pos"].float(), "pwke"),
       ("groups", lambda a: a["groups"][:, :2].contiguous(), "p"), ("ptable", lambda a: a["table"], "p"), ("slots", lambda a: a["slots"][:1], "wke"),
       ("w", lambda a: a["w"].double(), "wke"), ("w", lambda a: a["w"][:, :, :30].contiguous(), "wke"), ("w", lambda a: a["w"][:, :1].contiguous(), "wke"),
       ("w2", lambda a: a["w2"][:, :, :30].contiguous(), "e"), ("p2", lambda a: a["p2"].float(), "e"), ("p", lambda a: a["p"].float(), "e"), ("keep", lambda a: a["keep"][:1], "e"),
       ("lens", lambda a: a["lens"].long(), "e"), ("cu", lambda a: a["cu"][:2], "k"), ("nh", lambda a: 3, "pwk"), ("nkv", lambda a: 0, "pwk"),
       ("n", lambda a: -1, "pwke")]


@pytest.mark.parametrize("call,letter", [(_prefix, "p"), (_weigh, "w"), (_prompt, "k"), (_evict, "e")])
@pytest.mark.parametrize("i", range(len(BAD)))
def test_refusals(call, letter, i):
    from railgun_b200 import ops
    a = _good()
    call(ops, a)                                                       # as it is, it runs
    key, change, who = BAD[i]
    if letter not in who:
        return
    a[key] = change(a)
    with pytest.raises(ops.KernelError):
        call(ops, a)
    assert torch.cuda.current_stream().query() in (True, False)        # the context is in order


def test_no_rows():
    from railgun_b200 import ops
    a = _good()
    none, table = torch.empty(0, 4 * 64, dtype=torch.bfloat16, device=DEV), a["table"][:0]
    ops.prefix_attention(none, none, a["kv"], a["ptable"], i32([[0, 0, 8]]), table, a["pos"][:0], 4, 2, 64, 0.125, max_rows=0, max_prefix=8, max_own=9)
    ops.weighed_attention(none, none, a["kv"], a["w"], a["slots"][:0], table, a["pos"][:0], 4, 2, 64, 0.125, max_context=40)
    ops.prompt_key_weights(none, a["kv"], a["w"], a["slots"][:0], table, i32([0]), a["pos"][:0], a["pos"][:0], 4, 2, 64, 0.125, max_rows=0,
                           max_context=40)
    new = ops.evict_entries(a["kv"], a["w"], a["p"], a["w2"], a["p2"], a["slots"][:0], table, a["lens"][:0], a["keep"][:0], a["pos"][:0], 2, 64, 1, 1,
                            max_context=40)
    assert new.shape == (0,) and not a["w"].any()


def test_in_a_captured_graph():
    """Lengths stay on the device: a captured step runs again with others."""
    from railgun_b200 import ops
    nh, nkv, d, page = 8, 2, 64, 16
    g = torch.Generator(device=DEV).manual_seed(2)
    cache = Cache([300, 90, 90, 90], nkv, d, page, torch.bfloat16, g)
    q = queries(3, nh, d, torch.bfloat16, g)
    groups, pos, slots = i32([[0, 3, 300]]), i32([3, 50, 0]), i32([0, 1, 2])
    weights = torch.zeros(3, nkv, 90, device=DEV)

    def step(out1, out2, w):
        ops.prefix_attention(q, out1, cache.kv, cache.table[:1].contiguous(), groups, own_table, pos, nh, nkv, d, 0.125, max_rows=3,
                             max_prefix=300, max_own=90)
        ops.weighed_attention(q, out2, cache.kv, w, slots, own_table, pos, nh, nkv, d, 0.125, max_context=90)

    own_table = cache.table[1:].contiguous()
    outs = [torch.empty(3, nh * d, dtype=torch.bfloat16, device=DEV) for _ in range(4)]
    step(outs[0], outs[1], weights.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(outs[0], outs[1], weights)
    for values, prefix in (([3, 50, 0], 300), ([89, -1, 64], 17)):
        pos.copy_(i32(values))
        groups[0, 2] = prefix
        weights.zero_()
        graph.replay()
        w = torch.zeros_like(weights)
        step(outs[2], outs[3], w)
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]) and torch.equal(w, weights)


# ---- at the edges of what a call says -----------------------------------------------------------------------------------
@pytest.mark.parametrize("most", [2500, 20000])
def test_evict_leaves_requests_alone_in_long_contexts(most):
    """Requests without entries or without a slot, next to one that has both, where another kernel makes the moves."""
    from railgun_b200 import ops
    nkv, d, page, lens, slots = 2, 64, 16, [0, 2400, 300, 2500], [3, -1, 5, 0]
    g = torch.Generator(device=DEV).manual_seed(most)
    cache = Cache(lens, nkv, d, page, torch.bfloat16, g, width=-(-most // page))
    weights = torch.empty(5, nkv, most, device=DEV).exponential_(generator=g)
    places = torch.arange(most, device=DEV, dtype=torch.int32).expand(5, nkv, most).contiguous()
    w_out, p_out = weights.clone(), places.clone()               # there are slots 0 .. 4
    want = plain_evict(cache, weights, places, [s if 0 <= s < 5 else -1 for s in slots], lens, [100] * 4, lens, 4, 8)
    new = ops.evict_entries(cache.kv, weights, places, w_out, p_out, i32(slots), cache.table, i32(lens), i32([100] * 4), i32(lens), nkv, d, 4, 8,
                            max_context=most)
    assert new.tolist() == want[3] == [0, 2400, 300, 100]
    assert same(w_out, want[1]) and torch.equal(p_out, want[2]) and same(cache.kv, want[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows(dtype):
    """More rows than a grid has blocks in its second and third dimension."""
    from railgun_b200 import ops
    T, nh, nkv, d, page = 66000, 2, 1, 64, 8
    g = torch.Generator(device=DEV).manual_seed(5)
    kv = torch.randn(3, 2, nkv, page, d, device=DEV, generator=g).to(dtype)
    q = queries(T, nh, d, dtype, g)
    table = torch.randint(0, 3, (T, 1), device=DEV, generator=g, dtype=torch.int32)
    n = torch.randint(0, page + 1, (T,), device=DEV, generator=g)
    outs = [torch.empty(T, nh * d, dtype=dtype, device=DEV) for _ in range(2)]
    weights, slots = torch.zeros(T, nkv, page, device=DEV), torch.arange(T, device=DEV, dtype=torch.int32)
    pos = (n - 1).to(torch.int32)
    ops.weighed_attention(q, outs[0], kv, weights, slots, table, pos, nh, nkv, d, 0.125, max_context=page)
    ops.prefix_attention(q, outs[1], kv, table[:0], i32([]).view(0, 3), table, pos, nh, nkv, d, 0.125, max_rows=0, max_prefix=0, max_own=page)
    K, V = (kv[table[:, 0].long(), i, 0].double() for i in range(2))
    s = q.double().view(T, nh, d) @ K.transpose(1, 2) * 0.125
    p = torch.nan_to_num(torch.softmax(s.masked_fill(torch.arange(page, device=DEV) >= n[:, None, None], float("-inf")), -1))
    bound = out_error(q.reshape(-1, d), kv[:, 0, 0].reshape(1, -1, d).double(), V, page, 0.125, dtype)
    for out in outs:
        assert (out.double().view(T, nh, d) - p @ V).abs().max().item() <= bound
    w_bound = 2 * (weight_error(q.reshape(-1, d), kv[:, 0, 0].reshape(1, -1, d).double(), page, 0.125, dtype) + (nh + 3) * U)
    assert (weights[:, 0].double() - p.sum(1)).abs().max().item() <= w_bound


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,prefix,own", [(40, 700, 900), (5, 70, 40)])
def test_rows_beyond_what_a_call_says_are_not_seen(rows, prefix, own, dtype):
    from railgun_b200 import ops
    nh, nkv, d, page, most = 8, 2, 64, 16, rows - 2
    g = torch.Generator(device=DEV).manual_seed(rows)
    cache = Cache([prefix, prefix] + [own] * rows, nkv, d, page, dtype, g)
    q, tables, pos = queries(rows, nh, d, dtype, g), cache.table[:2].contiguous(), i32([own - 1] * rows)
    own_table = cache.table[2:].contiguous()

    def run(groups, max_rows):
        out = torch.empty(rows, nh * d, dtype=dtype, device=DEV)
        ops.prefix_attention(q, out, cache.kv, tables, i32(groups), own_table, pos, nh, nkv, d, 0.125, max_rows=max_rows, max_prefix=prefix, max_own=own)
        return out
    want = run([[0, most, prefix], [rows, 0, 0]], most)
    assert torch.equal(run([[0, rows, prefix], [-1, 5, prefix]], most), want)      # more rows than max_rows; no such first row
    # portions: the third request's rows come to more than max_rows
    few, outs = min(2, rows - 1), []
    for last in (1 + few, rows):
        w = torch.zeros(3, nkv, own + 8, device=DEV)
        ops.prompt_key_weights(q, cache.kv, w, i32([0, 1, 2]), cache.table[2:5].contiguous(), i32([0, 1, 1, last]), i32([5, 0, own // 2]),
                               i32([0, 0, 0]), nh, nkv, d, 0.125, max_rows=few, max_context=own)
        outs.append(w)
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [40, 700, 5000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_score_that_is_no_number_is_seen(bad, n, dtype):
    """An entry that a row sees and whose score is no number, or infinite: the row's results for its kv head are no numbers, as a
    softmax gives them; other heads, rows and requests are none the worse."""
    from railgun_b200 import ops
    nh, nkv, d, page, R = 8, 2, 64, 16, 3
    g = torch.Generator(device=DEV).manual_seed(n)
    cache = Cache([n] * R, nkv, d, page, dtype, g)
    q, pos, slots = queries(R, nh, d, dtype, g).abs(), i32([n - 1] * R), i32([0, 1, 2])
    args = (nh, nkv, d, 0.125)

    def run():
        outs = [torch.empty(R, nh * d, dtype=dtype, device=DEV) for _ in range(2)]
        w1, w2 = (torch.zeros(R, nkv, n, device=DEV) for _ in range(2))
        ops.prefix_attention(q, outs[0], cache.kv, cache.table[:1].contiguous(), i32([[0, 0, 0]]), cache.table, pos, *args, max_rows=0, max_prefix=0,
                             max_own=n)
        ops.weighed_attention(q, outs[1], cache.kv, w1, slots, cache.table, pos, *args, max_context=n)
        ops.prompt_key_weights(q, cache.kv, w2, slots, cache.table, i32([0, 1, 2, 3]), pos, i32([0, 0, 0]), *args, max_rows=1, max_context=n)
        return [o.view(R, nkv, -1) for o in outs] + [w1, w2]
    before = run()
    cache.kv[cache.table[1, 25 // page].long(), 0, 1, 25 % page, 3] = bad
    for x, y in zip(before, run()):
        hit = torch.zeros(R, nkv, dtype=torch.bool, device=DEV)
        hit[1, 1] = True
        assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], x[~hit])


# ---- head sizes that are no multiples of four, queries on odd addresses --------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,d,page", [(4, 2, 5, 7), (3, 1, 33, 16), (2, 1, 130, 8), (6, 3, 255, 4), (9, 1, 1, 3)])
def test_odd_head_sizes(nh, nkv, d, page, dtype):
    for scene in ("three groups", "long"):
        test_prefix_attention(nh, nkv, d, page, scene, dtype)
    test_weighed_attention(nh, nkv, d, page, [64, 63, 65, 1, 0, 200], dtype)
    test_prompt_key_weights(nh, nkv, d, page, [70, 129, 2], [0, 300, 63], [0, 300, 0], dtype)
    test_prompt_key_weights(nh, nkv, d, page, [3, 0, 1], [0, 5, 64], [0, 5, 64], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,d", [(8, 2, 64), (8, 2, 128), (4, 1, 48)])
def test_queries_on_odd_addresses(nh, nkv, d, dtype):
    """The same numbers one column further on, where no wide load can read them: the same results but for their rounding."""
    from railgun_b200 import ops
    R, n, P, page = 5, 150, 90, 16
    g = torch.Generator(device=DEV).manual_seed(d)
    cache = Cache([P] + [n] * R, nkv, d, page, dtype, g)
    q = torch.randn(R, nh * d, device=DEV, generator=g).to(dtype)
    odd = torch.empty(R, nh * d + 9, dtype=dtype, device=DEV)[:, 1:nh * d + 1]
    odd.copy_(q)
    tables, table, pos, slots = cache.table[:1].contiguous(), cache.table[1:].contiguous(), i32([n - 1] * R), i32(list(range(R)))
    args, outs = (nh, nkv, d, d ** -0.5), []
    for x in (q, odd):
        a, b = (out_view(R, nh * d, dtype) for _ in range(2))
        w1, w2 = (torch.zeros(R, nkv, n, device=DEV) for _ in range(2))
        ops.prefix_attention(x, a, cache.kv, tables, i32([[0, R, P]]), table, pos, *args, max_rows=R, max_prefix=P, max_own=n)
        ops.weighed_attention(x, b, cache.kv, w1, slots, table, pos, *args, max_context=n)
        ops.prompt_key_weights(x, cache.kv, w2, slots, table, i32(list(range(R + 1))), pos, i32([0] * R), *args, max_rows=1, max_context=n)
        outs.append((a, b, w1, w2))
    for r in range(R):
        K, V = cache.entries(1 + r, n)
        Kp, Vp = cache.entries(0, P)
        mine = q[r].reshape(nh, d)
        both = torch.cat([Kp, K], 1), torch.cat([Vp, V], 1)
        assert (outs[0][0][r].double() - outs[1][0][r].double()).abs().max() <= 2 * out_error(mine, *both, P + n, d ** -0.5, dtype)
        assert (outs[0][1][r].double() - outs[1][1][r].double()).abs().max() <= 2 * out_error(mine, K, V, n, d ** -0.5, dtype)
        for i in (2, 3):
            x, y = outs[0][i][r].double(), outs[1][i][r].double()
            assert ((x - y).abs() / y).max() <= 2 * (weight_error(mine, K, n, d ** -0.5, dtype) + (nh + 3) * U)


@pytest.mark.parametrize("nh,nkv,d,page", [(8, 2, 128, 256), (4, 4, 64, 512), (128, 1, 64, 16), (160, 1, 64, 16), (96, 1, 128, 32), (130, 2, 128, 8)])
def test_large_pages_and_many_heads(nh, nkv, d, page):
    """Pages longer than a tile, and as many query heads on a kv head as a tile has rows, or more."""
    for scene in ("three groups", "many rows", "long"):
        test_prefix_attention(nh, nkv, d, page, scene, torch.bfloat16)
    test_weighed_attention(nh, nkv, d, page, [2049, 3, 700], torch.bfloat16)
    test_prompt_key_weights(nh, nkv, d, page, [70, 129, 2], [0, 300, 63], [0, 300, 0], torch.bfloat16)
    test_prompt_key_weights(nh, nkv, d, page, [33, 64], [1000, 191], [2000, 0], torch.bfloat16)
