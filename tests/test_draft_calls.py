"""What the operators of drafted trees and of page copies take and refuse, and what they hand to their launchers, looked at without a GPU."""
import itertools

import numpy as np
import pytest
import torch

from railgun_b200 import native, ops


class Called(Exception):
    pass


@pytest.fixture
def calls(monkeypatch):
    """Runs an operator on CPU tensors up to its launch: the launcher's name and arguments, addresses as numbers, and what was allocated."""
    made, empty = [], torch.empty

    def new(dtype, here, *sizes):
        made.append(empty(sizes, dtype=dtype))
        return made[-1]

    def launch(lib, name, kinds, *args):
        assert len(kinds) == len(args)
        raise Called(name, [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args])
    monkeypatch.setattr(ops, "_tensors", False)
    monkeypatch.setattr(ops, "_current_device", lambda: -1)            # where tensors on the CPU are
    monkeypatch.setattr(ops, "_new", new)
    monkeypatch.setattr(ops, "_launch", launch)
    monkeypatch.setattr(ops, "num_sms", lambda device: 148)
    monkeypatch.setattr(ops, "_tc_error_flag", lambda device: None)

    def check(t, name, dtype=None):
        if not t.is_contiguous() or (dtype is not None and t.dtype != dtype):
            raise ops.KernelError(name)
    monkeypatch.setattr(ops, "_check", check)

    def check_rows(t, name, dtype=None):
        if t.dim() != 2 or t.stride(1) != 1 or t.stride(0) < t.shape[1] or t.dtype != dtype:
            raise ops.KernelError(name)
    monkeypatch.setattr(ops, "_check_rows", check_rows)

    def run(f, *a, **k):
        made.clear()
        with pytest.raises(Called) as e:
            f(*a, **k)
        return (*e.value.args, list(made))
    return run


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def tree_args(T=6, R=2, nh=8, nkv=2, d=64, page=16, dtype=torch.bfloat16, blocks=5, words=1):
    return dict(q=torch.zeros(T, nh * d, dtype=dtype), out=torch.zeros(T, nh * d, dtype=dtype), kv_cache=torch.zeros(9, 2, nkv, page, d, dtype=dtype),
                block_table=ints(R, blocks), cu_rows=ints(R + 1), starts=ints(R), masks=ints(T, words), nh=nh, nkv=nkv, d=d, scale=0.125, max_rows=3,
                max_context=70)


def test_without_a_device_there_is_a_word():
    if torch.cuda.is_available():
        pytest.skip("there is one")
    for f in (lambda: ops.draft_tree(ints(3), ints(2), ints(1), max_rows=3), lambda: ops.tree_attention(**tree_args()),
              lambda: ops.keep_drafts(torch.zeros(1, 2, 3), ints(1, 1), ints(2), ints(1), ints(3), ints(3), ints(3), max_rows=3),
              lambda: ops.copy_pages(torch.zeros(4, 3, 2), [(0, 1, -1)])):
        with pytest.raises(ops.KernelError, match="no CPU path"):
            f()


# ---- attention ----------------------------------------------------------------------------------------------------------
def test_what_tree_attention_refuses(calls):
    calls(ops.tree_attention, **tree_args())                             # as it is, it gets to its launcher
    a = tree_args()
    for bad in (dict(cu_rows=ints(2)), dict(starts=ints(3)), dict(block_table=ints(3, 5)), dict(block_table=ints(10)), dict(masks=ints(5, 1)),
                dict(masks=torch.zeros(6, 1, dtype=torch.int64)), dict(masks=ints(6)), dict(masks=ints(6, 2)[:, :1]), dict(out=a["out"][:5]),
                dict(out=torch.zeros(6, 8 * 64 + 8, dtype=torch.bfloat16)), dict(out=a["out"].float()), dict(q=a["q"][:, :500]), dict(q=a["q"].half()),
                dict(kv_cache=a["kv_cache"].float()), dict(kv_cache=a["kv_cache"][:, :1]), dict(kv_cache=a["kv_cache"][0]),
                dict(kv_cache=torch.zeros(9, 2, 2, 0, 64, dtype=torch.bfloat16)), dict(kv_cache=torch.zeros(0, 2, 2, 16, 64, dtype=torch.bfloat16)), dict(nh=7), dict(nkv=0), dict(d=0), dict(d=257), dict(nkv=3),
                dict(max_rows=-1), dict(max_context=-1), dict(max_rows=1 << 31), dict(max_context=1 << 32)):
        with pytest.raises(ops.KernelError):
            ops.tree_attention(**{**a, **bad})


def test_queries_and_outputs_that_share_memory_are_refused(calls):
    """A row whose output is no number is worked out again from its queries, which would be written over by then."""
    n = 8 * 64
    wide, flat = torch.zeros(7, 3 * n, dtype=torch.bfloat16), torch.zeros(12 * n, dtype=torch.bfloat16)
    first, last = flat[:6 * n].view(6, n), flat[6 * n:].view(6, n)
    for q, out in ((first, first), (wide[:6, :n], wide[:6, :n]), (wide[:6, :n], wide[:6, n - 1:2 * n - 1]), (wide[:6, n:2 * n], wide[:6, 1:n + 1]),
                   (wide[:6, :n], wide[1:, :n]), (wide[1:, :n], wide[:6, :n]), (flat.view(6, 2 * n), last), (first, flat[6 * n - 1:12 * n - 1].view(6, n))):
        with pytest.raises(ops.KernelError, match="share memory"):
            ops.tree_attention(**{**tree_args(), "q": q, "out": out})
    for q, out in ((first, last), (last, first), (wide[:6, :n], wide[:6, n:2 * n]), (wide[:6, 2 * n:], wide[:6, :n]), (wide[:6, n:2 * n], wide[1:, :n]),
                   (wide[:6], wide[:6, n:2 * n])):                       # of the last, only the first columns are read
        calls(ops.tree_attention, **{**tree_args(), "q": q, "out": out})


@pytest.mark.parametrize("step", [(1 << 31) - 8, 1 << 31, (1 << 32) + 512])
def test_rows_that_are_far_apart(calls, monkeypatch, step):
    """Launchers take distances of 32 bits: none is cut to them."""
    def rows(n):
        return torch.empty_strided((n, 512), (step, 1), dtype=torch.bfloat16, device="meta")
    for n in (0, 1):
        got = ops._rows_fit(rows(n), "q", torch.bfloat16, -1, 512)
        assert got[0] == n and 512 <= got[1] < 1 << 31
    if step < 1 << 31:
        assert ops._rows_fit(rows(2), "q", torch.bfloat16, -1, 512) == (2, step)
    else:
        with pytest.raises(ops.KernelError, match="apart"):
            ops._rows_fit(rows(2), "q", torch.bfloat16, -1, 512)


def test_nothing_to_do_is_no_launch(calls):
    for none in (tree_args(T=0), tree_args(R=0), {**tree_args(), "max_rows": 0}):
        ops.tree_attention(**none)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parts_lie_where_their_loads_can_read_them(calls, monkeypatch, dtype):
    """Work that is cut into stretches: places for the parts of all queries and for one more item a worker; (m, l) on their boundaries, where they are behind them."""
    seen = set()
    monkeypatch.setattr(ops, "tree_cluster", lambda *a: 0)
    for (nh, nkv, d, page), T, R, most in itertools.product([(3, 1, 33, 16), (5, 5, 5, 3), (8, 2, 64, 16), (24, 8, 128, 16), (40, 1, 128, 32), (160, 1, 64, 16)],
                                                            (1, 7, 333), (1, 5), (1, 3, 16, 17, 300)):
        name, args, (scratch,) = calls(ops.tree_attention, **{**tree_args(T, R, nh, nkv, d, page, dtype, words=-(-most // 32)), "max_rows": most})
        blocks, workers, queries, least, tile_rows, tensor_cores, cluster, part_o, part_ml, parts, err = args[-11:]
        G, at = nh // nkv, scratch.data_ptr()
        seen.add(tensor_cores)
        assert cluster == 0
        assert part_o == at and part_ml % 8 == 0 and parts % 8 == 0 and least >= 1
        assert at + 4 * d * (T * nh + workers * queries) <= part_ml and parts - part_ml >= 8 * (T * nh + workers * queries)
        assert parts + 8 * T * nh <= at + scratch.numel() * 4
        if tensor_cores:
            assert dtype == torch.bfloat16 and d in (64, 128) and G <= 128
            assert tile_rows * G <= 128 and queries == tile_rows * G * tensor_cores and workers * tensor_cores == 2 * blocks
            assert (tensor_cores == 1) == (min(most, T) * G <= 128 // G * G)
        else:
            assert queries == 16 and workers == blocks
    assert seen == ({0} if dtype == torch.float32 else {0, 1, 2})


def test_cases_that_the_tensor_cores_kernel_cannot_read(calls, monkeypatch):
    """Rows of queries on odd addresses, pages that are no powers of two, scales that are not positive: the general kernel's."""
    monkeypatch.setattr(ops, "tree_cluster", lambda *a: 0)

    def cores(**more):
        return calls(ops.tree_attention, **{**tree_args(), **more})[1][-6]
    assert cores() == 1
    wide = torch.zeros(6, 8 * 64 + 9, dtype=torch.bfloat16)
    for bad in (dict(q=wide[:, 1:513]), dict(q=torch.zeros(6, 517, dtype=torch.bfloat16)), dict(kv_cache=torch.zeros(9, 2, 2, 12, 64, dtype=torch.bfloat16)),
                dict(kv_cache=torch.zeros(9, 2, 2, 4, 64, dtype=torch.bfloat16)), dict(scale=-0.1), dict(scale=0.0), dict(block_table=ints(2, 0))):
        assert cores(**bad) == 0


def test_calls_whose_items_are_whole(calls):
    """Few nodes on short contexts: one launch, no scratch; many, or long contexts, are cut into stretches."""
    name, args, made = calls(ops.tree_attention, **tree_args())
    assert args[-11:-5] == [0, 0, 16, 1, 0, 0] and args[-5] in (1, 2, 4, 8) and args[-4:] == [None] * 4 and not made
    for fast, d, G, nkv in itertools.product((True, False), (64, 128, 192, 256), (1, 4, 7, 200), (1, 8)):
        one = [ops.tree_cluster(1, 1, nkv, G, d, 1, n, fast, 148) for n in (1, 32, 60, 300, 600)]
        assert one[0] == one[1] == 1 and set(one) <= {0, 1, 2, 4, 8}
        assert d > 128 or not fast or ops.tree_cluster(64, 64 * 64, 8, 8, d, 64, 8192, fast, 148) == 0
        assert ops.tree_cluster(64, 64, 8, 8, d, 64, 100, fast, 148) == 0        # room for 64 times the rows that there are
        for rows, context in ((0, 0), (1, 0), (1 << 30, 1 << 30)):
            ops.tree_cluster(1, 1, nkv, G, d, rows, context, fast, 148)


# ---- layout and what is kept ----------------------------------------------------------------------------------------------
def test_what_draft_tree_refuses(calls):
    name, args, made = calls(ops.draft_tree, ints(6), ints(3), ints(2), max_rows=33)
    assert [tuple(t.shape) for t in made] == [(6, 2), (6,)]
    for bad in (dict(parents=ints(6, 1)), dict(parents=torch.zeros(6, dtype=torch.int64)), dict(cu_rows=ints(2)), dict(starts=ints(3)), dict(starts=ints(1, 2)),
                dict(max_rows=-1), dict(max_rows=ops.DRAFT_MOST + 1)):
        with pytest.raises(ops.KernelError):
            ops.draft_tree(**{**dict(parents=ints(6), cu_rows=ints(3), starts=ints(2), max_rows=3), **bad})


def keep_args():
    return dict(caches=[torch.zeros(9, 2, 2, 16, 64) for _ in range(3)], block_table=ints(2, 5), cu_rows=ints(3), starts=ints(2), parents=ints(6), tokens=ints(6),
                chosen=ints(6), max_rows=4)


def test_what_keep_drafts_refuses(calls):
    name, args, made = calls(ops.keep_drafts, **keep_args())
    assert args[1:7] == [3, 9, 4, 16, 16, 16]                            # caches, pages, outer, page, pieces of a row and their bytes
    assert [tuple(t.shape) for t in made] == [(2,), (2, 4), (2, 4)]
    cache = keep_args()["caches"][0]
    for bad in (dict(caches=[]), dict(caches=[cache, cache.clone(), cache]), dict(caches=[cache, cache[:8]]), dict(caches=[cache, cache.double()]), dict(caches=cache.transpose(1, 2)),
                dict(caches=torch.zeros(9, 16)), dict(caches=torch.zeros(0, 2, 16, 64)), dict(block_table=ints(3, 5)), dict(cu_rows=ints(2)),
                dict(tokens=ints(5)), dict(chosen=ints(7)), dict(chosen=torch.zeros(6, dtype=torch.int64)), dict(max_rows=-1), dict(max_rows=ops.DRAFT_MOST + 1)):
        with pytest.raises(ops.KernelError):
            ops.keep_drafts(**{**keep_args(), **bad})


def test_caches_that_share_memory_are_refused(calls):
    """Wherever they begin: entries would move twice.  Caches one behind the other are different ones."""
    both = torch.zeros(10, 2, 2, 16, 64)
    for bad in ([both[:9], both[1:]], [both[1:], both[:9]], [both[:5], both[5:], both[4:9]]):
        with pytest.raises(ops.KernelError, match="share memory"):
            ops.keep_drafts(**{**keep_args(), "caches": bad})
        with pytest.raises(ops.KernelError, match="share memory"):
            ops.copy_pages(bad, [(0, 1, -1)])
    assert calls(ops.keep_drafts, **{**keep_args(), "caches": [both[5:], both[:5]]})[1][1] == 2
    assert calls(ops.copy_pages, [both[5:], both[:5]], [(0, 1, -1)])[1][1] == 2


@pytest.mark.parametrize("shape,dtype,piece", [((4, 2, 8, 64), torch.bfloat16, 16), ((4, 2, 8, 5), torch.bfloat16, 2), ((4, 2, 8, 6), torch.float32, 8),
                                               ((4, 8, 33), torch.uint8, 1), ((4, 8, 12), torch.uint8, 4)])
def test_rows_move_in_the_largest_pieces_that_they_are_made_of(calls, shape, dtype, piece):
    cache = torch.zeros(shape, dtype=dtype)
    args = calls(ops.keep_drafts, **{**keep_args(), "caches": cache})[1]
    assert args[6] == piece and args[5] * piece == shape[-1] * cache.element_size()
    assert calls(ops.copy_pages, cache, [(0, 1, 3)])[1][6] == piece
    if piece > cache.element_size():                                     # a cache on an odd address
        odd = torch.zeros(cache.numel() + 1, dtype=dtype)[1:].view(shape)
        assert calls(ops.copy_pages, odd, [(0, 1, 3)])[1][6] == cache.element_size()


# ---- copies -----------------------------------------------------------------------------------------------------------------
def test_what_copies_are_made_of(calls):
    cache = torch.zeros(9, 2, 2, 16, 64)
    for good in ([(0, 1, 3)], np.array([[0, 1, 3]]), np.array([[0, 1, 3]], dtype=np.int64), torch.tensor([[0, 1, 3]])):
        assert calls(ops.copy_pages, cache, good)[1][8] == 1
    ops.copy_pages(cache, [])                                            # nothing is no launch
    ops.copy_pages(cache, np.zeros((0, 3), np.int32))
    for bad in ([(0, 1)], [0, 1, 3], [(0.0, 1.0, 3.0)], [(0, 1, 1 << 31)], np.zeros((1, 3, 1), np.int32), [("a", "b", "c")]):
        with pytest.raises(ops.KernelError):
            ops.copy_pages(cache, bad)
    with pytest.raises(ops.KernelError):
        ops.copy_pages([], [(0, 1, 3)])
    with pytest.raises(ops.KernelError):
        ops.copy_pages([cache, cache], [(0, 1, 3)])
    with pytest.raises(ops.KernelError):
        ops.copy_pages(torch.zeros(0, 2, 16, 64), [(0, 1, 3)])


@pytest.mark.parametrize("copies,what", [([(0, 9, 1)], "caches"), ([(9, 0, 1)], "caches"), ([(-1, 0, 1)], "caches"), ([(0, -1, 1)], "caches"),
                                         ([(0, 1, 17)], "caches"), ([(0, 1, -2)], "caches"), ([(0, 1, 1), (2, 1, 1)], "once"),
                                         ([(0, 1, 1), (1, 2, 1)], "once"), ([(1, 2, 1), (0, 1, 1)], "once"), ([(3, 3, 1), (0, 1, 1), (0, 1, 1)], "once")])
def test_copies_that_the_launcher_refuses(monkeypatch, copies, what):
    """Pages that are not there, and copies whose order would matter: refused on the host, before anything is launched."""
    def launch(lib, name, kinds, addresses, *args):
        f = getattr(native.load(lib), name)
        f.argtypes = [ops.ctypes.c_char_p, *[ops.ctypes.c_longlong if k == "i" and i == 5 else ops.ctypes.c_int if k == "i" else ops.ctypes.c_void_p
                                            for i, k in enumerate(kinds[1:], 1)], ops.ctypes.c_void_p]
        return f(addresses, *args, None)
    monkeypatch.setattr(ops, "_tensors", False)
    monkeypatch.setattr(ops, "_current_device", lambda: -1)
    monkeypatch.setattr(ops, "_launch", launch)
    monkeypatch.setattr(ops, "num_sms", lambda device: 148)
    monkeypatch.setattr(ops, "_check", lambda *a, **k: None)
    with pytest.raises(ops.KernelError, match=what):
        ops.copy_pages(torch.zeros(9, 2, 2, 16, 8), copies)
