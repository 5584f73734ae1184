"""Trees of drafted tokens over the paged cache against their definitions in 64 bits: which nodes a node sees, attention of the nodes,
what is kept of a tree, and copies of pages.

Rows of the cache that no table names, and those behind a request's last entry, hold NaN: none of them may have a say.
"""
import random

import numpy as np
import pytest
import torch

from test_cache_operators_gpu import DEV, TYPES, U, Cache, i32, no_wait_gave_up, out_view, queries, weight_error  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- trees ------------------------------------------------------------------------------------------------------------
def tree(n, kind, rng):
    """Parents of n nodes, node 0 the root."""
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return ([-1] + [0] * (n - 1))[:n]
    if kind == "forest":
        return [-1 if i == 0 or rng.random() < 0.3 else rng.randrange(i) for i in range(n)]
    return [-1 if i == 0 else rng.randrange(max(0, i - 5), i) for i in range(n)]


def ancestors(parents):
    """Of every node: itself, its parent, ... up to its root."""
    lines = []
    for i, p in enumerate(parents):
        lines.append([i] + (lines[p] if 0 <= p < i else []))
    return lines


def mask_words(rows, words):
    """int32 words of lists of nodes."""
    m = np.zeros((len(rows), words), dtype=np.uint32)
    for i, nodes in enumerate(rows):
        for j in nodes:
            m[i, j // 32] |= np.uint32(1 << (j % 32))
    return torch.from_numpy(m.view(np.int32)).to(DEV)


def ends(counts, first=0):
    out = [first]
    for n in counts:
        out.append(out[-1] + n)
    return out


# ---- layout -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["chain", "star", "tree", "forest"])
@pytest.mark.parametrize("counts", [[1], [0, 3], [32, 33, 31, 0, 64, 65, 1], [300, 5], [1] * 70])
def test_draft_tree(counts, kind):
    from railgun_b200 import ops
    rng = random.Random(len(counts) + sum(counts))
    first, behind, most = 2, 3, max(counts)                             # rows of no request in front and behind
    cu = ends(counts, first)
    T = cu[-1] + behind
    trees = [tree(n, kind, rng) for n in counts]
    parents = [7] * first + sum(trees, []) + [0] * behind
    starts = [rng.randrange(1 << 20) for _ in counts]
    masks, positions = ops.draft_tree(i32(parents), i32(cu), i32(starts), max_rows=most)
    words = -(-most // 32)
    want, where = [[]] * first, [0] * first
    for t, s in zip(trees, starts):
        lines = ancestors(t)
        want += lines
        where += [s + len(x) - 1 for x in lines]
    want, where = want + [[]] * behind, where + [0] * behind
    assert masks.shape == (T, words) and torch.equal(masks, mask_words(want, words))
    assert positions.tolist() == where
    # fewer rows than there are: what is left of the layout is the same, the others see nothing
    few = max(1, most // 2)
    masks, positions = ops.draft_tree(i32(parents), i32(cu), i32(starts), max_rows=few)
    for r, n in enumerate(counts):
        for i in range(n):
            t = cu[r] + i
            assert positions[t].item() == (where[t] if i < few else 0)
            assert torch.equal(masks[t].cpu(), mask_words([want[t] if i < few else []], masks.shape[1])[0].cpu())


def test_draft_tree_of_odd_parents():
    """A parent that does not come before its node, and a request that is left out."""
    from railgun_b200 import ops
    masks, positions = ops.draft_tree(i32([-1, 5, 1, 2, -9, 0, 0]), i32([0, 5, 7]), i32([10, -1]), max_rows=5)
    assert masks[:, 0].tolist() == [1, 2, 6, 14, 16, 0, 0] and positions.tolist() == [10, 10, 11, 12, 10, 0, 0]


# ---- attention --------------------------------------------------------------------------------------------------------
def attend(q, K, V, seen, scale):
    """Weights [nkv, G n, entries] and outputs of rows [n, nh, d] that see [n, entries] in 64 bits."""
    n, nh, d = q.shape
    nkv = K.shape[0]
    G = nh // nkv
    scores = q.double().view(n, nkv, G, d).permute(1, 0, 2, 3).reshape(nkv, n * G, d) @ K.transpose(1, 2) * scale
    hidden = ~seen.repeat_interleave(G, 0)
    scores = scores.masked_fill(hidden, float("-inf"))
    top = scores.amax(-1, keepdim=True) if scores.shape[-1] else scores.sum(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, 1.0)


def held_to(out, q, K, V, seen, scale, dtype):
    """Is every number of ``out`` [n, nh, d] as near to the formula as its roundings allow?  The weights by weight_error (scores, 2^x,
    the sum) and, where the tensor cores multiply them (bfloat16), by their rounding, at most 2^-8 of each; sums of N products in 32 bits;
    the output's own rounding, at most 2^-8 of it in bfloat16."""
    n, nh, d = q.shape
    nkv, N = K.shape[0], K.shape[1]
    if n == 0:
        return
    p = attend(q, K, V, seen, scale)
    want = p @ V
    half = 2.0 ** -8 if dtype == torch.bfloat16 else U
    w = max(weight_error(q[i], K, N, scale, dtype) for i in range(n)) if N else 0.0
    off = (p @ V.abs()) * (w + (2 * N + 8) * U + (half if dtype == torch.bfloat16 else 0.0))
    off = off + half * (want.abs() + off)
    got = out.double().view(n, nkv, nh // nkv, d).permute(1, 0, 2, 3).reshape(nkv, -1, d)
    worst = ((got - want).abs() - off).max().item()
    assert worst <= 0, worst


def run_tree(counts, starts, nh, nkv, d, page, dtype, seed, choose="tree", more=0, first=1, behind=2):
    """One call, every row held to the formula, and rows of no request as they were.  ``choose``: the masks, of trees or of
    nodes drawn at will.  Returns what a second look needs."""
    from railgun_b200 import ops
    g, rng = torch.Generator(device=DEV).manual_seed(seed), random.Random(seed)
    R, scale = len(counts), d ** -0.5
    lens = [n + s for n, s in zip(counts, starts)]
    cache = Cache(lens, nkv, d, page, dtype, g)
    cu = ends(counts, first)
    T = cu[-1] + behind
    q, out = queries(T, nh, d, dtype, g), out_view(T, nh * d, dtype)
    most = max(counts)
    rows = [[]] * first
    for n in counts:
        rows += ancestors(tree(n, "tree", rng)) if choose == "tree" else [[j for j in range(n) if rng.random() < choose] for _ in range(n)]
    rows += [[]] * behind
    masks = mask_words(rows, -(-most // 32))
    if n_bits := most % 32:                                              # bits behind the last node say nothing
        masks[:, -1] |= torch.tensor(-(1 << n_bits), dtype=torch.int32, device=DEV)
    args = (cache.kv, cache.table, i32(cu), i32(starts), masks, nh, nkv, d, scale)
    ops.tree_attention(q, out, *args, max_rows=most + more, max_context=max(lens) + more)
    for r, n in enumerate(counts):
        K, V = cache.entries(r, lens[r])
        seen = torch.zeros(n, lens[r], dtype=torch.bool)
        seen[:, :starts[r]] = True
        for i in range(n):
            for j in rows[cu[r] + i]:
                seen[i, starts[r] + j] = True
        mine = q[cu[r]:cu[r + 1]].reshape(n, nh, d)
        held_to(out[cu[r]:cu[r + 1]].reshape(n, nh, d), mine, K, V, seen.to(DEV), scale, dtype)
    assert (out[:first] == 7).all() and (out[cu[-1]:] == 7).all()
    return q, out, args, dict(max_rows=most + more, max_context=max(lens) + more)


HEADS = [(3, 1, 32, 8), (4, 4, 64, 16), (8, 2, 128, 32), (32, 8, 64, 16), (24, 8, 128, 16), (20, 1, 16, 7), (12, 1, 128, 64), (6, 2, 24, 5),
         (2, 1, 256, 16), (5, 5, 80, 16), (40, 1, 64, 128), (4, 1, 128, 8)]
SCENES = {
    "one token": ([1], [0]),
    "one node": ([1], [200]),
    "no context": ([5, 1], [0, 0]),
    "no rows": ([0, 3, 0], [7, 64, 0]),
    "ends of tiles": ([16, 8, 1, 3, 64], [48, 120, 127, 126, 64]),
    "many nodes": ([70, 33], [100, 0]),
    "longer": ([4, 9], [1500, 333]),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scene", SCENES)
@pytest.mark.parametrize("nh,nkv,d,page", HEADS)
def test_tree_attention(nh, nkv, d, page, scene, dtype):
    from railgun_b200 import ops
    counts, starts = SCENES[scene]
    q, out, args, sizes = run_tree(counts, starts, nh, nkv, d, page, dtype, nh * d + len(scene))
    # the same again, on another stream: the same bits
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = torch.full_like(out, 7.0)
        ops.tree_attention(q, again, *args, **sizes)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cluster", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("scene", SCENES)
@pytest.mark.parametrize("nh,nkv,d,page", [(3, 1, 32, 8), (8, 2, 128, 32), (24, 8, 64, 16), (20, 1, 16, 7), (8, 1, 192, 16), (2, 1, 256, 16), (40, 1, 64, 128)])
def test_each_way_to_split_the_work(monkeypatch, nh, nkv, d, page, scene, cluster, dtype):
    """Stretches and clusters, whichever the sizes would have chosen."""
    from railgun_b200 import ops
    monkeypatch.setattr(ops, "tree_cluster", lambda *a: cluster)
    run_tree(*SCENES[scene], nh, nkv, d, page, dtype, nh + d + len(scene))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cluster", [None, 0, 1, 2, 8])
@pytest.mark.parametrize("nh,nkv,d,page", [(8, 2, 64, 16), (3, 1, 33, 16), (4, 2, 128, 4)])
def test_calls_at_the_limits(monkeypatch, nh, nkv, d, page, cluster, dtype):
    """Scales of any sign, operands on any address, room for more rows than there can be, and calls that say that nothing is seen."""
    from railgun_b200 import ops
    if cluster is not None:
        monkeypatch.setattr(ops, "tree_cluster", lambda *a: cluster)
    counts, starts = [5, 20], [100, 0]
    q, out, args, sizes = run_tree(counts, starts, nh, nkv, d, page, dtype, 17)
    T, scale = q.shape[0], args[-1]
    wide = torch.zeros(T * (nh * d + 3) + 1, dtype=dtype, device=DEV)
    odd = wide[1:].view(T, nh * d + 3)
    odd[:, :nh * d] = q
    to = torch.full((T * (nh * d + 1) + 1,), 7.0, dtype=dtype, device=DEV)[1:].view(T, nh * d + 1)
    mine = to[:, :nh * d]
    seen = torch.zeros(5, 105, dtype=torch.bool, device=DEV)
    seen[:, :100] = True
    seen[:, 100:] = (args[4][1:6, :1] >> torch.arange(5, device=DEV)) & 1 == 1
    cache = args[0]
    K, V = [cache[args[1][0, :-(-105 // page)].long()][:, j].double().permute(1, 0, 2, 3).reshape(nkv, -1, d)[:, :105] for j in (0, 1)]
    for s in (scale, -scale, 0.0):
        ops.tree_attention(odd, mine, *args[:-1], s, **{**sizes, "max_rows": 1 << 30})
        assert (to[:, nh * d] == 7).all() and (mine[0] == 7).all() and (mine[-2:] == 7).all()
        p = attend(q[1:6].view(5, nh, d), K, V, seen, s)
        want = (p @ V).view(nkv, 5, nh // nkv, d).permute(1, 0, 2, 3).reshape(5, nh * d)
        # weights that are off by w of themselves, and their rounding and the output's in bfloat16
        w = max(weight_error(q[1 + i].view(nh, d), K, 105, abs(s), dtype) for i in range(5)) + 218 * U + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
        off = w * V.abs().max() + (2.0 ** -8 if dtype == torch.bfloat16 else U) * (want.abs() + w * V.abs().max())
        assert ((mine[1:6].double() - want).abs() <= off).all()
    ops.tree_attention(q, out, *args, max_rows=20, max_context=0)
    assert not out[1:26].any() and (out[0] == 7).all() and (out[26:] == 7).all()
    ops.tree_attention(q, out, cache, args[1][:, :0].contiguous(), *args[2:], **sizes)           # a table without columns
    assert not out[1:26].any()
    ops.tc_gemm_check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cluster", [0, 1, 2, 8])
@pytest.mark.parametrize("nh,nkv,d,page", [(8, 2, 64, 16), (8, 2, 80, 16)])
def test_pages_that_are_not_there(monkeypatch, nh, nkv, d, page, cluster, dtype):
    """Reported, and read nowhere; entries behind a request's last one may be on any page, and the next call is right again."""
    from railgun_b200 import ops
    monkeypatch.setattr(ops, "tree_cluster", lambda *a: cluster)
    q, out, args, sizes = run_tree([5, 20, 3], [100, 40, 0], nh, nkv, d, page, dtype, 3)
    ops.tc_gemm_check()
    want, table = out.clone(), args[1]
    behind = table.clone()
    behind[0, 7:], behind[1, 4:], behind[2, 1:] = -5, 1 << 30, 999999   # 105, 60 and 3 entries
    ops.tree_attention(q, out, args[0], behind, *args[2:], **sizes)
    ops.tc_gemm_check()
    assert torch.equal(out, want)
    for page_id in (-1, args[0].shape[0], 2 ** 31 - 1):
        bad = table.clone()
        bad[1, 2] = page_id
        ops.tree_attention(q, out, args[0], bad, *args[2:], **sizes)
        with pytest.raises(ops.KernelError, match="page"):
            ops.tc_gemm_check()
    ops.tree_attention(q, out, *args, **sizes)
    ops.tc_gemm_check()
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("share", [0.0, 0.03, 0.5])
def test_masks_that_are_no_trees(share, dtype):
    """Any nodes may be seen, or none: rows without context then give 0."""
    _, out, _, _ = run_tree([40, 3, 64], [0, 5, 129], 8, 2, 64, 16, dtype, 5, choose=share)
    if share == 0:
        assert (out[1:41] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_more_room_than_there_is_need_for(dtype):
    run_tree([3, 1, 20], [70, 0, 400], 8, 2, 128, 16, dtype, 11, more=500)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,d,page", [(4, 2, 5, 7), (3, 1, 33, 16), (2, 1, 130, 8), (6, 3, 255, 4), (9, 1, 1, 3), (160, 1, 64, 16),
                                           (96, 1, 128, 32), (8, 2, 128, 256), (4, 1, 192, 16), (130, 2, 128, 8)])
def test_odd_sizes(nh, nkv, d, page, dtype):
    run_tree([5, 18, 1], [130, 7, 64], nh, nkv, d, page, dtype, d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,d,page", [(8, 2, 64, 16), (24, 8, 128, 16), (5, 5, 24, 4), (80, 2, 128, 32), (4, 1, 256, 16)])
@pytest.mark.parametrize("seed", range(4))
def test_stretches_that_begin_and_end_anywhere(monkeypatch, seed, nh, nkv, d, page, dtype):
    """Requests of all lengths, so that stretches begin and end in the middle of items, between them, and where there is little or nothing."""
    from railgun_b200 import ops
    monkeypatch.setattr(ops, "tree_cluster", lambda *a: 0)
    rng = random.Random(seed)
    n = rng.choice([1, 3, 17, 60])
    most, longest = rng.choice([1, 4, 20, 50]), rng.choice([0, 30, 300, 1500])
    run_tree([rng.randrange(most + 1) for _ in range(n - 1)] + [most], [rng.randrange(longest + 1) for _ in range(n)], nh, nkv, d, page, dtype, seed)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cluster", [None, 0])
@pytest.mark.parametrize("nh,nkv,d,page", [(8, 8, 8, 16), (8, 8, 1, 16), (8, 8, 4, 4), (6, 6, 5, 7), (16, 8, 3, 16), (8, 8, 9, 16), (8, 4, 32, 8)])
def test_small_heads_in_stretches(monkeypatch, nh, nkv, d, page, cluster, dtype):
    """More items of a tile or two than there are workers, so that stretches go on behind an item's end while the next item's first tile is
    there: sums of groups of threads that share columns have room of their own."""
    from railgun_b200 import ops
    if cluster is not None:
        monkeypatch.setattr(ops, "tree_cluster", lambda *a: cluster)
    rng = random.Random(d)
    n = 256
    run_tree([rng.choice([1, 1, 1, 2]) for _ in range(n)], [rng.choice([63, 62, 64, 20, 130]) for _ in range(n)], nh, nkv, d, page, dtype, d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cluster", [None, 0])
def test_many_requests(monkeypatch, cluster, dtype):
    """More requests than a block has threads, most of them short."""
    from railgun_b200 import ops
    if cluster is not None:
        monkeypatch.setattr(ops, "tree_cluster", lambda *a: cluster)
    rng = random.Random(3)
    n = 700
    run_tree([rng.choice([0, 1, 1, 2, 5]) for _ in range(n)], [rng.choice([0, 1, 9, 40]) for _ in range(n)], 4, 2, 64, 16, dtype, 8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("cluster", [None, 0, 2])
@pytest.mark.parametrize("counts,starts", [([6, 5], [70, 9]), ([40, 33], [500, 0])])
def test_what_is_not_seen_has_no_say(monkeypatch, counts, starts, cluster, bad, dtype):
    """A node whose key and value are no numbers: rows that see it show it, the others are what they were to their last bit but one
    rounding."""
    from railgun_b200 import ops
    if cluster is not None:
        monkeypatch.setattr(ops, "tree_cluster", lambda *a: cluster)
    nh, nkv, d, page, scale = 8, 2, 64, 16, 0.125
    g = torch.Generator(device=DEV).manual_seed(1)
    lens = [n + s for n, s in zip(counts, starts)]
    cache = Cache(lens, nkv, d, page, dtype, g)
    cu, most = ends(counts), max(counts)
    T = cu[-1]
    q = queries(T, nh, d, dtype, g)
    lines = sum([ancestors(tree(n, "tree", random.Random(2))) for n in counts], [])
    masks = mask_words(lines, -(-most // 32))

    def run():
        out = torch.empty(T, nh * d, dtype=dtype, device=DEV)
        ops.tree_attention(q, out, cache.kv, cache.table, i32(cu), i32(starts), masks, nh, nkv, d, scale, max_rows=most, max_context=max(lens))
        return out
    before = run()
    node = 3
    e = starts[0] + node
    where = (cache.table[0, e // page].long(), slice(None), 1, e % page)
    cache.kv[where] = bad
    after = run()
    for t in range(T):
        sees = t < counts[0] and node in lines[t]
        x, y = before[t].view(nkv, -1).double(), after[t].view(nkv, -1).double()
        assert torch.equal(x[0], y[0])                                   # the other kv head
        if sees:
            assert not torch.isfinite(y[1]).any()
        else:
            assert torch.isfinite(y[1]).all() and (x[1] - y[1]).abs().max() <= 2.0 ** (-6 if dtype == torch.bfloat16 else -17) * max(1.0, x[1].abs().max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cluster", [None, 0, 2])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_queries_that_are_no_numbers(monkeypatch, bad, cluster, dtype):
    """Their rows and heads are no numbers, quickly, and nobody else's: long contexts, where entry by entry would take its time."""
    from railgun_b200 import ops
    if cluster is not None:
        monkeypatch.setattr(ops, "tree_cluster", lambda *a: cluster)
    nh, nkv, d = 8, 2, 64
    q, out, args, sizes = run_tree([20, 40], [3000, 100], nh, nkv, d, 16, dtype, 23)
    hurt = q.clone()
    hurt[3, :d] = bad                                                    # a head of a row
    hurt[25:41] = bad                                                    # rows of the other request
    after = torch.full_like(out, 7.0)
    ops.tree_attention(hurt, after, *args, **sizes)
    no = torch.zeros(after.shape, dtype=torch.bool, device=DEV)
    no[3, :d] = True
    no[25:41] = True
    assert not torch.isfinite(after[no]).any() and torch.equal(after[~no], out[~no])
    # and values: of the first request's first entry and kv head
    cache, table = args[0].clone(), args[1]
    cache[table[0, 0].long(), 1, 0, 0] = bad
    ops.tree_attention(q, after, cache, table, *args[2:], **sizes)
    no[:] = False
    no[1:21, :nh // nkv * d] = True
    assert not torch.isfinite(after[no]).any() and torch.equal(after[~no], out[~no])


@pytest.mark.parametrize("dtype", TYPES)
def test_what_a_call_says_is_what_is_seen(dtype):
    """Rows beyond max_rows are left as they were, nodes beyond them and entries beyond max_context are not seen; a request with a
    negative start is left out."""
    from railgun_b200 import ops
    nh, nkv, d, page, scale = 8, 2, 64, 16, 0.125
    g = torch.Generator(device=DEV).manual_seed(4)
    cache = Cache([60, 40, 30], nkv, d, page, dtype, g)
    q = queries(20, nh, d, dtype, g)
    cu, starts = [0, 10, 15, 20], [50, -1, 25]
    masks = torch.full((20, 1), -1, dtype=torch.int32, device=DEV)
    out = torch.full((20, nh * d), 7.0, dtype=dtype, device=DEV)
    ops.tree_attention(q, out, cache.kv, cache.table, i32(cu), i32(starts), masks, nh, nkv, d, scale, max_rows=4, max_context=53)
    assert (out[4:15] == 7).all() and (out[19:] == 7).all()
    for r, n, most in ((0, 4, 53), (2, 4, 29)):
        K, V = cache.entries(r, most)
        mine = q[cu[r]:cu[r] + n].reshape(n, nh, d)
        held_to(out[cu[r]:cu[r] + n].reshape(n, nh, d), mine, K, V, torch.ones(n, most, dtype=torch.bool, device=DEV), scale, dtype)
    # nodes that the masks have no word for are not seen
    ops.tree_attention(q, out, cache.kv, cache.table, i32([0, 10, 10, 10]), i32(starts), masks[:, :0].contiguous(), nh, nkv, d, scale, max_rows=10,
                       max_context=60)
    K, V = cache.entries(0, 60)
    seen = torch.zeros(10, 60, dtype=torch.bool, device=DEV)
    seen[:, :50] = True
    held_to(out[:10].reshape(10, nh, d), q[:10].reshape(10, nh, d), K, V, seen, scale, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_chain_is_a_portion(dtype):
    """One guess after the other: what attention of a prompt's portion gives."""
    from railgun_b200 import ops
    nh, nkv, d, page, n, start = 8, 2, 64, 16, 12, 77
    g = torch.Generator(device=DEV).manual_seed(9)
    cache = Cache([start + n], nkv, d, page, dtype, g)
    q = queries(n, nh, d, dtype, g, more=0)
    masks, positions = ops.draft_tree(i32([i - 1 for i in range(n)]), i32([0, n]), i32([start]), max_rows=n)
    assert positions.tolist() == list(range(start, start + n))
    out = torch.empty(n, nh * d, dtype=dtype, device=DEV)
    ops.tree_attention(q, out, cache.kv, cache.table, i32([0, n]), i32([start]), masks, nh, nkv, d, 0.125, max_rows=n, max_context=start + n)
    portion = ops.paged_attention_general(q, nh * d, cache.kv, cache.table, i32([0] * n), positions, nh, nkv, d, 0, 0.125)
    assert (out.double() - portion.double()).abs().max() <= (2.0 ** -6 if dtype == torch.bfloat16 else 1e-5) * portion.double().abs().max()


@pytest.mark.parametrize("dtype", TYPES)
def test_trees_in_a_captured_graph(dtype):
    """Captured once, replayed with other lengths, masks and tables; two graphs in turn."""
    from railgun_b200 import ops
    nh, nkv, d, page, R, most = 8, 2, 128, 16, 4, 6
    g = torch.Generator(device=DEV).manual_seed(2)
    q = queries(R * most, nh, d, dtype, g)
    graphs = []
    for _ in range(2):
        s = dict(kv=torch.zeros(64, 2, nkv, page, d, dtype=dtype, device=DEV), table=torch.zeros(R, 14, dtype=torch.int32, device=DEV),
                 cu=torch.zeros(R + 1, dtype=torch.int32, device=DEV), starts=torch.zeros(R, dtype=torch.int32, device=DEV),
                 masks=torch.zeros(R * most, 1, dtype=torch.int32, device=DEV), out=torch.zeros(R * most, nh * d, dtype=dtype, device=DEV))

        def call(s=s):
            ops.tree_attention(q, s["out"], s["kv"], s["table"], s["cu"], s["starts"], s["masks"], nh, nkv, d, 0.09, max_rows=most, max_context=200)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append((graph, s))
    for counts, starts in (([6, 0, 3, 1], [100, 5, 0, 190]), ([1, 1, 1, 1], [0, 1, 2, 3]), ([0, 0, 6, 6], [7, 8, 60, 111])):
        scenes = []
        for k, (graph, s) in enumerate(graphs):
            cache = Cache([n + a for n, a in zip(counts, starts)], nkv, d, page, dtype, g, width=14)
            s["kv"][:cache.kv.shape[0]] = cache.kv
            s["table"].copy_(cache.table[:, :14])
            s["cu"].copy_(i32(ends(counts)))
            s["starts"].copy_(i32(starts))
            lines = sum([ancestors(tree(n, "chain" if k else "tree", random.Random(1))) for n in counts], [])
            s["masks"][:len(lines)] = mask_words(lines, 1)
            s["out"].fill_(7)
            scenes.append((cache, lines))
            graph.replay()
        for (graph, s), (cache, lines) in zip(graphs, scenes):
            cu = ends(counts)
            for r, n in enumerate(counts):
                N = n + starts[r]
                K, V = cache.entries(r, N)
                seen = torch.zeros(n, N, dtype=torch.bool)
                seen[:, :starts[r]] = True
                for i in range(n):
                    seen[i, [starts[r] + j for j in lines[cu[r] + i]]] = True
                held_to(s["out"][cu[r]:cu[r + 1]].reshape(n, nh, d), q[cu[r]:cu[r + 1]].reshape(n, nh, d), K, V, seen.to(DEV), 0.09, dtype)
            assert (s["out"][cu[-1]:] == 7).all()


@pytest.mark.parametrize("cluster", [0, 2])
def test_a_replayed_graph_reports_pages_that_are_not_there(monkeypatch, cluster):
    """Once who replays it has said so: a replay is no call that could be seen from here."""
    from railgun_b200 import ops
    monkeypatch.setattr(ops, "tree_cluster", lambda *a: cluster)
    q, out, args, sizes = run_tree([5, 20], [100, 40], 8, 2, 64, 16, torch.bfloat16, 3)
    ops.tc_gemm_check()
    want, table = out.clone(), args[1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.tree_attention(q, out, *args, **sizes)
    ops.tc_gemm_check()
    args[1][1, 2] = -1
    graph.replay()
    ops.mark_tc_unchecked()
    with pytest.raises(ops.KernelError, match="page"):
        ops.tc_gemm_check()
    args[1].copy_(table)
    graph.replay()
    ops.mark_tc_unchecked()
    ops.tc_gemm_check()
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_pages_beyond_two_to_the_31_elements(dtype):
    from railgun_b200 import ops
    nh, nkv, d, page = 8, 8, 128, 16
    pages = (1 << 31) // (2 * nkv * page * d) + 40                       # elements of the cache pass 2^31
    kv = torch.empty(pages, 2, nkv, page, d, dtype=dtype, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    starts, n = [100], 5
    table = torch.arange(pages - 7, pages, dtype=torch.int32, device=DEV)[None].contiguous()
    kv[pages - 7:] = torch.randn(7, 2, nkv, page, d, device=DEV, generator=g).to(dtype)
    q, out = queries(n, nh, d, dtype, g), out_view(n, nh * d, dtype)
    masks = mask_words(ancestors([-1, 0, 0, 1, 2]), 1)
    ops.tree_attention(q, out, kv, table, i32([0, n]), i32(starts), masks, nh, nkv, d, 0.09, max_rows=n, max_context=105)
    rows = kv[pages - 7:].double().permute(1, 2, 0, 3, 4).reshape(2, nkv, -1, d)[:, :, :105]
    seen = torch.ones(n, 105, dtype=torch.bool, device=DEV)
    seen[:, 100:] = torch.tensor([[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 1, 0, 1, 0], [1, 0, 1, 0, 1]], device=DEV) == 1
    held_to(out.reshape(n, nh, d), q.reshape(n, nh, d), rows[0], rows[1], seen, 0.09, dtype)


# ---- what is kept -----------------------------------------------------------------------------------------------------
def kept(parents, tokens, chosen):
    path, node = [], 0 if parents else None
    while node is not None:
        path.append(node)
        node = next((c for c in range(node + 1, len(parents)) if parents[c] == node and tokens[c] == chosen[node]), None)
    return path


@pytest.mark.parametrize("dtype", TYPES + [torch.uint8])
@pytest.mark.parametrize("layers,shape", [(1, (2, 2, 16, 64)), (3, (2, 1, 8, 5)), (70, (2, 2, 4, 8)), (2, (16, 96)), (2, (7, 33))])
@pytest.mark.parametrize("counts", [[1], [0, 6, 1], [40, 64, 33, 2], [200]])
def test_keep_drafts(counts, layers, shape, dtype):
    from railgun_b200 import ops
    rng, g = random.Random(sum(counts)), torch.Generator(device=DEV).manual_seed(layers)
    page, R = shape[-2], len(counts)
    starts = [rng.randrange(3 * page) for _ in counts]
    need = [-(-(s + n) // page) for s, n in zip(starts, counts)]
    pages = torch.randperm(sum(need) + 2, device=DEV, generator=g).to(torch.int32)
    table, used = torch.zeros(R, max(need + [1]), dtype=torch.int32, device=DEV), 0
    for r, n in enumerate(need):
        table[r, :n] = pages[used:used + n]
        used += n
    caches = [torch.randint(0, 200, (sum(need) + 2, *shape), device=DEV, generator=g).to(dtype) for _ in range(layers)]
    want = [c.clone() for c in caches]
    trees = [tree(n, "tree", rng) for n in counts]
    tokens = [rng.randrange(4) for _ in range(sum(counts))]              # few tokens: siblings that hold the same one, too
    chosen = [rng.randrange(4) for _ in range(sum(counts))]
    cu, most = ends(counts), max(counts)
    paths = [kept(t, tokens[a:], chosen[a:]) for t, a in zip(trees, cu)]
    for r, path in enumerate(paths):
        for k, node in enumerate(path):
            a, b = starts[r] + node, starts[r] + k
            for c in want:
                c[table[r, b // page].long(), ..., b % page, :] = c[table[r, a // page].long(), ..., a % page, :].clone()
    counted, path, fresh = ops.keep_drafts(caches, table, i32(cu), i32(starts), i32(sum(trees, [])), i32(tokens), i32(chosen), max_rows=most)
    assert counted.tolist() == [len(p) for p in paths]
    for r, p in enumerate(paths):
        assert path[r].tolist() == p + [-1] * (most - len(p))
        assert fresh[r].tolist() == [chosen[cu[r] + i] for i in p] + [-1] * (most - len(p))
    for c, w in zip(caches, want):
        assert torch.equal(c, w)


def test_a_whole_chain_is_kept():
    """Every guess was right, and a long detour in front of the right ones."""
    from railgun_b200 import ops
    n, page = 300, 16
    for detour in (0, 100):
        parents = [i - 1 for i in range(n)]
        if detour:
            parents[detour] = 0
        tokens = list(range(n))
        chosen = [i + 1 for i in range(n)]
        if detour:
            chosen[0] = detour
        cache = torch.randn(40, 2, 2, page, 8, device=DEV)
        table = torch.randperm(40, device=DEV)[None].to(torch.int32)
        before = cache.clone()
        count, path, fresh = ops.keep_drafts(cache, table, i32([0, n]), i32([50]), i32(parents), i32(tokens), i32(chosen), max_rows=n)
        want = kept(parents, tokens, chosen)
        assert count.item() == len(want) == n - max(0, detour - 1) and path[0, :len(want)].tolist() == want
        rows = lambda c: c[table[0].long()].permute(0, 3, 1, 2, 4).reshape(-1, 2, 2, 8)  # noqa: E731
        expected = rows(before).clone()
        expected[50:50 + len(want)] = rows(before)[[50 + i for i in want]]
        assert torch.equal(rows(cache), expected)


def test_a_cache_twice_is_refused():
    """Its entries would move twice, and the second time from where others had moved to."""
    from railgun_b200 import ops
    cache = torch.randn(8, 2, 2, 16, 8, device=DEV)
    before, args = cache.clone(), (i32([[0, 1]]), i32([0, 3]), i32([3]), i32([-1, 0, 0]), i32([1, 2, 3]), i32([3, 1, 1]))
    for caches in ([cache, cache], [cache, before, cache]):
        with pytest.raises(ops.KernelError, match="twice"):
            ops.keep_drafts(caches, *args, max_rows=3)
        with pytest.raises(ops.KernelError, match="twice"):
            ops.copy_pages(caches, [(0, 1, -1)])
    assert torch.equal(cache, before)


def test_keep_leaves_out_what_it_should():
    from railgun_b200 import ops
    cache = torch.randn(8, 2, 2, 16, 8, device=DEV)
    before = cache.clone()
    table = i32([[0, 1], [2, 3], [4, 5]])
    # a request with a negative start, one with more rows than the call says, and a parent that does not come before its node
    count, path, fresh = ops.keep_drafts(cache, table, i32([0, 2, 6, 9]), i32([-1, 3, 0]), i32([-1, 0, -1, 0, 1, 2, -1, 2, 0]), i32([1] * 9), i32([1] * 9),
                                         max_rows=3)
    assert count.tolist() == [0, 3, 2] and path.tolist() == [[-1] * 3, [0, 1, 2], [0, 2, -1]] and fresh.tolist() == [[-1] * 3, [1] * 3, [1, 1, -1]]
    before[4, :, :, 1] = before[4, :, :, 2]
    assert torch.equal(cache, before)


# ---- copies of pages ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES + [torch.uint8])
@pytest.mark.parametrize("layers,shape", [(1, (2, 2, 16, 64)), (3, (2, 1, 8, 5)), (70, (2, 2, 4, 8)), (2, (16, 96)), (2, (7, 33)), (1, (2, 8, 64, 128))])
@pytest.mark.parametrize("n", [1, 7, 600])
def test_copy_pages(n, layers, shape, dtype):
    from railgun_b200 import ops
    g, rng = torch.Generator(device=DEV).manual_seed(n), random.Random(n)
    page, total = shape[-2], 2 * n + 3
    caches = [torch.randint(0, 200, (total, *shape), device=DEV, generator=g).to(dtype) for _ in range(layers)]
    want = [c.clone() for c in caches]
    order = list(range(total))
    rng.shuffle(order)
    copies = [(order[rng.randrange(n)], order[n + i], rng.choice([-1, 0, 1, page, page // 2])) for i in range(n)] + [(order[-1], order[-1], -1)]
    for a, b, held in copies:
        held = page if held < 0 else held
        for c in want:
            c[b, ..., :held, :] = c[a, ..., :held, :]
    ops.copy_pages(caches, np.array(copies, dtype=np.int32))
    for c, w in zip(caches, want):
        assert torch.equal(c, w)


def test_copy_rows_and_odd_addresses():
    """Buffers of a row a request, and caches on addresses that no wide load can read."""
    from railgun_b200 import ops
    state = torch.randn(6, 3001, device=DEV)
    flat = torch.randn(6, device=DEV)
    want, first = state.clone(), flat.clone()
    want[4], first[4] = want[1], first[1]
    ops.copy_pages(state, [(1, 4, -1)])
    ops.copy_pages(flat, [(1, 4, -1)])
    assert torch.equal(state, want) and torch.equal(flat, first)
    odd = torch.randn(1 + 5 * 2 * 4 * 6, device=DEV).to(torch.bfloat16)[1:].view(5, 2, 4, 6)
    want = odd.clone()
    want[3, :, :2] = want[0, :, :2]
    ops.copy_pages([odd], [(0, 3, 2)])
    assert torch.equal(odd, want)
    ops.copy_pages([odd], [])
    assert torch.equal(odd, want)


def test_copies_beyond_two_to_the_31_bytes():
    from railgun_b200 import ops
    cache = torch.zeros(70000, 2, 8, 16, 128, dtype=torch.bfloat16, device=DEV)
    cache[69999] = torch.randn(2, 8, 16, 128, device=DEV).to(torch.bfloat16)
    ops.copy_pages(cache, [(69999, 69998, 5), (69999, 3, -1)])
    assert torch.equal(cache[69998, :, :, :5], cache[69999, :, :, :5]) and not cache[69998, :, :, 5:].any() and torch.equal(cache[3], cache[69999])
