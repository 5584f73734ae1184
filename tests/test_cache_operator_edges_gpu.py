"""Operators over the cache at the edges of their sizes: odd head sizes in parts, lists longer than a call's counts, many groups,
and outputs held to bounds of their own size."""
import pytest
import torch

from test_cache_operators_gpu import (DEV, HEADS, TYPES, U, Cache, i32, no_wait_gave_up, out_view, plain_evict, queries, same, softmax,  # noqa: F401
                                      weight_error)

pytestmark = pytest.mark.gpu


def attended(q, K, V, scale, dtype):
    """One row's softmax weights [nkv, G, n] and output [nkv, G, d] in 64 bits, and how far each number of the kernels' output may be
    off: the weights by ``weight_error`` and, where the tensor cores multiply them (bfloat16, head sizes in 64s), by their rounding; sums of
    n products in 32 bits; the output's own rounding.  A rounding to bfloat16, of 8 significant bits, is at most 2^-8 of a number
    (1 + 2^-8 lies half way between 1 and 1 + 2^-7)."""
    nkv, n = K.shape[0], K.shape[1]
    nh, d = q.shape
    p = softmax(q.double().view(nkv, nh // nkv, d) @ K.transpose(1, 2) * scale)
    out = p @ V
    if n == 0:
        return p, out, torch.zeros_like(out)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else U
    rounded = half if dtype == torch.bfloat16 and d % 64 == 0 else 0.0
    off = (p @ V.abs()) * (weight_error(q, K, n, scale, dtype) + (2 * n + 8) * U + rounded)
    return p, out, off + half * (out.abs() + off)


def run_weighed(lens, nh, nkv, d, page, dtype, seed):
    from railgun_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(seed)
    R, most, G, scale = len(lens), max(lens), nh // nkv, d ** -0.5
    cache = Cache(lens, nkv, d, page, dtype, g)
    q, out, slots = queries(R, nh, d, dtype, g), out_view(R, nh * d, dtype), torch.randperm(R, device=DEV, generator=g)
    weights = torch.rand(R, nkv, most, device=DEV, generator=g)
    before = weights.clone()
    ops.weighed_attention(q, out, cache.kv, weights, slots.int(), cache.table, i32([n - 1 for n in lens]), nh, nkv, d, scale, max_context=most,
                          decay=0.75)
    for r, n in enumerate(lens):
        K, V = cache.entries(r, n)
        mine, s = q[r].reshape(nh, d), int(slots[r])
        p, want, off = attended(mine, K, V, scale, dtype)
        assert ((out[r].double().view(nkv, G, d) - want).abs() <= off).all(), r
        if n:
            w = p.sum(1)
            w[:, :-1] += 0.75 * before[s, :, :n - 1].double()
            assert ((weights[s, :, :n].double() - w).abs() <= w * (weight_error(mine, K, n, scale, dtype) + (G + 3) * U)).all(), r
        assert torch.equal(weights[s, :, n:], before[s, :, n:])


def run_prefix(groups, own, nh, nkv, d, page, dtype, seed):
    """groups: (rows, prefix entries); rows behind them belong to none."""
    from railgun_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(seed)
    T, G, scale, prefixes = len(own), nh // nkv, d ** -0.5, [p for _, p in groups]
    cache = Cache(prefixes + own, nkv, d, page, dtype, g)
    q, out, first, table, of = queries(T, nh, d, dtype, g), out_view(T, nh * d, dtype), 0, [], {}
    for i, (n, p) in enumerate(groups):
        table.append([first, n, p])
        of.update({t: i for t in range(first, first + n)})
        first += n
    ops.prefix_attention(q, out, cache.kv, cache.table[:len(groups)].contiguous(), i32(table).view(-1, 3), cache.table[len(groups):].contiguous(),
                         i32([n - 1 for n in own]), nh, nkv, d, scale, max_rows=max(n for n, _ in groups), max_prefix=max(prefixes),
                         max_own=max(own))
    lists = {}
    for t in range(T):
        i = of.get(t)
        if i not in lists:
            lists[i] = cache.entries(i or 0, prefixes[i] if i is not None else 0)
        K, V = (torch.cat(x, 1) for x in zip(lists[i], cache.entries(len(groups) + t, own[t])))
        _, want, off = attended(q[t].reshape(nh, d), K, V, scale, dtype)
        assert ((out[t].double().view(nkv, G, d) - want).abs() <= off).all(), t


# ---- odd numbers of rows, heads, parts and columns: parts whose (m, l) start behind an odd number of numbers -------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,nh,nkv,d,most", [(201, 3, 3, 5, 450), (601, 1, 1, 5, 500), (199, 3, 1, 33, 450), (593, 1, 1, 255, 300)])
def test_odd_parts_of_weighed_attention(R, nh, nkv, d, most, dtype):
    run_weighed([most - 7 * i % most for i in range(R)], nh, nkv, d, 16, dtype, R + d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,nh,nkv,d,prefix,own", [(199, 3, 1, 33, 600, 100), (199, 3, 1, 33, 500, 100), (601, 1, 1, 5, 700, 40)])
def test_odd_parts_of_prefix_attention(T, nh, nkv, d, prefix, own, dtype):
    run_prefix([(T - 2, prefix)], [7 * i % (own + 1) for i in range(T)], nh, nkv, d, 16, dtype, T + d)


# ---- lists longer than a call's counts ---------------------------------------------------------------------------------------
# which kernels: few and many rows in 32-bit, few and many in bfloat16, more heads on one than a cluster's block takes
WEIGHED = [(torch.float32, 8, 2, 64, 3, 90), (torch.float32, 8, 2, 64, 3, 5000), (torch.bfloat16, 8, 2, 64, 2, 700),
           (torch.bfloat16, 8, 2, 128, 40, 2000), (torch.bfloat16, 40, 1, 64, 2, 300), (torch.float32, 20, 1, 24, 2, 130)]


@pytest.mark.parametrize("dtype,nh,nkv,d,R,most", WEIGHED)
@pytest.mark.parametrize("cut", ["max_context", "table"])
def test_an_entry_is_new_by_its_position(dtype, nh, nkv, d, R, most, cut):
    """The last entry that a call has room for is not new where the row's position lies behind it: its weight goes on."""
    from railgun_b200 import ops
    page, G, scale, decay = 16, nh // nkv, d ** -0.5, 0.5
    most = -(-most // page) * page                                    # whole pages: a table of so many has room for no more
    g = torch.Generator(device=DEV).manual_seed(most)
    cache = Cache([most + page] * R, nkv, d, page, dtype, g)
    table = cache.table if cut == "max_context" else cache.table[:, :most // page].contiguous()
    q, out = queries(R, nh, d, dtype, g), out_view(R, nh * d, dtype)
    positions = [most - 1 + (1, 0, 2)[r % 3] for r in range(R)]       # the last one that is seen, or behind it
    weights = 1.0 + torch.rand(R, nkv, most + page, device=DEV, generator=g)
    before = weights.clone()
    ops.weighed_attention(q, out, cache.kv, weights, i32(list(range(R))), table, i32(positions), nh, nkv, d, scale,
                          max_context=most if cut == "max_context" else most + page, decay=decay)
    for r, at in enumerate(positions):
        K, V = cache.entries(r, most)
        mine = q[r].reshape(nh, d)
        p, want, off = attended(mine, K, V, scale, dtype)
        assert ((out[r].double().view(nkv, G, d) - want).abs() <= off).all(), r
        w = p.sum(1) + decay * before[r, :, :most].double()
        if at == most - 1:
            w[:, -1] = p.sum(1)[:, -1]
        assert ((weights[r, :, :most].double() - w).abs() <= w * (weight_error(mine, K, most, scale, dtype) + (G + 3) * U)).all(), r
        assert torch.equal(weights[r, :, most:], before[r, :, most:])


# few rows and many in 32-bit and bfloat16; groups of many rows, whose prefixes the tensor cores take, with one or two parts a block
PREFIXED = [(torch.float32, 4, 2, 64, 3), (torch.float32, 8, 2, 32, 150), (torch.bfloat16, 8, 2, 64, 4), (torch.bfloat16, 20, 1, 256, 2),
            (torch.bfloat16, 8, 2, 192, 170), (torch.bfloat16, 32, 8, 128, 150), (torch.bfloat16, 32, 8, 64, 60), (torch.bfloat16, 8, 2, 128, 40)]


@pytest.mark.parametrize("dtype,nh,nkv,d,T", PREFIXED)
@pytest.mark.parametrize("max_prefix,max_own", [(0, 0), (0, 70), (130, 0), (1000, 100), (300, 333), (1, 1), (2500, 17)])
def test_entries_beyond_what_a_call_says_are_not_seen(max_prefix, max_own, dtype, nh, nkv, d, T):
    """Prefixes and own lists that are longer than a call says: the results are those of lists that end there."""
    from railgun_b200 import ops
    page, more = 16, 150
    g = torch.Generator(device=DEV).manual_seed(max_prefix + T)
    cache = Cache([max_prefix + more] * 2 + [max_own + more] * T, nkv, d, page, dtype, g)
    q, tables, own_table = queries(T, nh, d, dtype, g), cache.table[:2].contiguous(), cache.table[2:].contiguous()
    first = T // 2

    def run(prefix, own):
        out = out_view(T, nh * d, dtype)
        ops.prefix_attention(q, out, cache.kv, tables, i32([[0, first, prefix[0]], [first, T - first, prefix[1]]]), own_table, i32(own), nh, nkv,
                             d, d ** -0.5, max_rows=T - first, max_prefix=max_prefix, max_own=max_own)
        return out
    lens = [(max_own + more - 1) * (r % 4) // 3 for r in range(T)]       # positions, some behind what the call says
    over = run([max_prefix + more, max_prefix + 1], lens)
    assert torch.equal(over, run([max_prefix, max_prefix], [min(n, max_own - 1) for n in lens]))
    if max_prefix + max_own == 0:
        assert not over.any()


@pytest.mark.parametrize("most", [0, 1, 90, 2048, 2500, 20000])
def test_evict_leaves_longer_requests_alone(most):
    """A request with more entries than a call has room for: choosing among some of them could drop those that are protected."""
    from railgun_b200 import ops
    nkv, d, page = 2, 64, 16
    lens = [most, most + 1, most + 40, max(0, most - 1)]
    keep = [max(1, n // 3) for n in lens]
    g = torch.Generator(device=DEV).manual_seed(most)
    cache = Cache(lens, nkv, d, page, torch.bfloat16, g, width=1)
    weights = torch.empty(4, nkv, most + 40, device=DEV).exponential_(generator=g)
    places = torch.arange(most + 40, device=DEV, dtype=torch.int32).expand(4, nkv, most + 40).contiguous()
    want = plain_evict(cache, weights, places, [0, -1, -1, 3], lens, keep, [n - 1 for n in lens], 2, 5)
    got = weights.clone(), places.clone()
    new = ops.evict_entries(cache.kv, weights, places, *got, i32([0, 1, 2, 3]), cache.table, i32(lens), i32(keep), i32([n - 1 for n in lens]),
                            nkv, d, 2, 5, max_context=most)
    assert new.tolist() == [min(most, keep[0]), most + 1, most + 40, min(lens[3], keep[3])]
    assert same(got[0], want[1]) and torch.equal(got[1], want[2]) and same(cache.kv, want[0])
    # the table has room for fewer entries than the call
    if most >= 90:
        narrow = cache.table[:, :2].contiguous()
        kv, w, p = cache.kv.clone(), weights.clone(), places.clone()
        new = ops.evict_entries(cache.kv, weights, places, weights, places, i32([0, 1, 2, 3]), narrow, i32([33, 32, most, 34]), i32([8] * 4),
                                i32([32, 31, most - 1, 33]), nkv, d, 2, 5, max_context=most)
        assert new.tolist() == [33, 8, most, 34]
        for r in (0, 2, 3):
            assert torch.equal(weights[r], w[r]) and torch.equal(places[r], p[r])
            mine = cache.table[r, :-(-lens[r] // page)].long()
            assert same(cache.kv[mine], kv[mine])


# ---- many groups ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_groups,nh,nkv,d,prefix,own", [(48, 8, 2, 64, 300, 40), (70, 4, 2, 32, 90, 20), (33, 32, 8, 128, 700, 60), (130, 2, 1, 64, 40, 5)])
def test_many_groups(n_groups, nh, nkv, d, prefix, own, dtype):
    """Parallel samples: dozens of groups of a few rows, some without rows or entries, rows of no group behind them."""
    groups = [((i * 5 + 3) % 9, 0 if i % 11 == 4 else prefix - 7 * i % prefix) for i in range(n_groups)]
    T = sum(n for n, _ in groups) + 3
    run_prefix(groups, [3 * i % (own + 1) for i in range(T)], nh, nkv, d, 16, dtype, n_groups + d)


# ---- outputs to their own size ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,d,page", HEADS)
def test_outputs_are_as_near_as_their_roundings(nh, nkv, d, page, dtype):
    """A mean over thousands of entries is small: held to what its own weights and values allow, not to the largest value."""
    run_prefix([(2, 65), (1, 0), (7, 201)], [3, 0, 9, 31, 0, 64, 63, 129, 1, 16, 0, 5], nh, nkv, d, page, dtype, nh + d)
    run_prefix([(20, 4999), (3, 640)], [i * 37 % 140 for i in range(24)], nh, nkv, d, page, dtype, nh + d + 1)
    run_prefix([(5, 3001)], [700, 0, 1, 128, 333], nh, nkv, d, page, dtype, nh + d + 2)
    run_weighed([64, 63, 65, 1, 0, 200], nh, nkv, d, page, dtype, nh + d + 3)
    run_weighed([5000, 2049, 3, 700], nh, nkv, d, page, dtype, nh + d + 4)
    run_weighed([i * 53 % 1500 for i in range(70)], nh, nkv, d, page, dtype, nh + d + 5)
