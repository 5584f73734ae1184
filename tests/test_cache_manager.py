"""The cache manager: no page lost, held twice or freed twice, under random
orders of requests; windows give pages back; slots
(pattern of crates/vllm-paged-attention/src/allocator.rs:177-210)."""
import numpy as np
import pytest

from railgun_b200.cache.manager import CacheError, OutOfPages, PageAllocator, PagedKVNeed, StateNeed, group_needs


def test_counts_and_fifo_reuse():
    a = PageAllocator([4], [6], [0], 3)
    assert a.free_pages() == 6 and a.free_slots() == 3
    s = a.add_request(10)
    a.reserve(10, 9)                                   # 3 pages
    assert a.block_table(10).tolist() == [0, 1, 2] and a.free_pages() == 3
    a.reserve(10, 9)                                   # idempotent
    assert a.free_pages() == 3
    a.commit(10, 9)
    assert a.num_computed(10) == 9 and a.slot(10) == s
    a.release(10)
    assert a.free_pages() == 6 and a.free_slots() == 3
    a.add_request(11)
    a.reserve(11, 16)                                  # FIFO: the untouched pages first, then the returned ones
    assert a.block_table(11).tolist() == [3, 4, 5, 0]
    a.check()


def test_errors():
    a = PageAllocator([4], [2], [0], 1)
    a.add_request(1)
    with pytest.raises(CacheError):
        a.add_request(1)                               # duplicate
    with pytest.raises(CacheError):
        a.add_request(2)                               # no slot left
    with pytest.raises(OutOfPages):
        a.reserve(1, 9)
    assert a.free_pages() == 2                         # a failed reserve takes nothing
    with pytest.raises(CacheError):
        a.commit(1, 5)                                 # beyond what is reserved
    with pytest.raises(CacheError):
        a.release(99)
    a.release(1)
    with pytest.raises(CacheError):
        a.release(1)                                   # freed twice
    a.check()


def test_reserve_is_all_groups_or_none():
    a = PageAllocator([4, 4], [8, 2], [0, 0], 2)
    a.add_request(1)
    with pytest.raises(OutOfPages):
        a.reserve(1, 12)                               # group 1 has only 2 pages
    assert a.free_pages(0) == 8 and a.free_pages(1) == 2
    a.check()


def test_window_gives_pages_back():
    a = PageAllocator([4, 4], [32, 32], [0, 6], 2)
    a.add_request(1)
    n = 0
    for step in (3, 5, 1, 1, 7, 2, 1, 1, 1, 9):
        n += step
        a.reserve(1, n)
        a.commit(1, n)
        full, win = a.block_table(1, 0), a.block_table(1, 1)
        assert (full >= 0).all() and len(full) == -(-n // 4)
        first_needed = n - 6 + 1
        for i, p in enumerate(win):
            assert (p < 0) == ((i + 1) * 4 <= first_needed), (n, i, win)
        a.check()
    held = (a.block_table(1, 1) >= 0).sum()
    assert held <= 3 and a.free_pages(1) == 32 - held
    a.release(1)
    assert a.free_pages(1) == 32
    a.check()


@pytest.mark.parametrize("seed", range(6))
def test_random_orders_keep_every_page_accounted_for(seed):
    rng = np.random.default_rng(seed)
    pages, slots = [24, 16], 5
    a = PageAllocator([4, 8], pages, [0, 20], slots)
    live, next_id = {}, 1
    held_at_some_time = set()
    for _ in range(600):
        op = rng.integers(0, 10)
        if op < 2 and len(live) < slots:
            a.add_request(next_id)
            live[next_id] = 0
            next_id += 1
        elif op < 8 and live:
            rid = int(rng.choice(list(live)))
            new_len = live[rid] + int(rng.integers(1, 12))
            try:
                a.reserve(rid, new_len)
            except OutOfPages:
                victim = int(rng.choice(list(live)))
                a.release(victim)
                del live[victim]
                continue
            a.commit(rid, new_len)
            live[rid] = new_len
        elif live:
            rid = int(rng.choice(list(live)))
            a.release(rid)
            del live[rid]
        a.check()
        # no page is held by two requests
        for g in range(2):
            seen = []
            for rid in live:
                seen += [int(p) for p in a.block_table(rid, g) if p >= 0]
            assert len(seen) == len(set(seen))
            assert len(seen) + a.free_pages(g) == pages[g]
            held_at_some_time |= {(g, p) for p in seen}
        assert a.free_slots() == slots - len(live)
    for rid in list(live):
        a.release(rid)
    a.check()
    assert [a.free_pages(g) for g in range(2)] == pages and a.free_slots() == slots
    assert len(held_at_some_time) > sum(pages) * 0.8          # pages were used again and again


def test_needs_are_sorted_into_groups():
    full = PagedKVNeed(2, 16, 0)
    groups, group_of, states = group_needs({
        0: full, 1: PagedKVNeed(2, 16, 8), 2: full, 3: StateNeed((4, 4)), 4: None, 5: PagedKVNeed(1, 16, 0)})
    assert [(n, c) for n, c in groups] == [(full, [0, 2]), (PagedKVNeed(2, 16, 8), [1]), (PagedKVNeed(1, 16, 0), [5])]
    assert group_of == {0: 0, 2: 0, 1: 1, 5: 2} and list(states) == [3]


def test_groups_get_the_page_geometry_they_ask_for():
    """Needs that say nothing get the engine's page size, pool and precision; a need may ask for its own page
    size, a smaller pool (a windowed group), another precision and another shape of page."""
    import torch
    from railgun_b200.cache.manager import CacheManager, PagedKVNeed, StateNeed
    needs = {0: PagedKVNeed(2, 16), 1: PagedKVNeed(2, 16),                       # one group, two cache ids
             2: PagedKVNeed(1, 32, window=24, page_size=8, pool_tokens=96),      # windowed: small pages, small pool
             3: PagedKVNeed(0, 0, dtype="float32", page_shape=("page", 40)),     # one compressed vector per token
             4: StateNeed((5, 3), "float32"), 5: None}
    cm = CacheManager(needs, page_size=16, max_tokens=256, max_requests=4, dtype=torch.bfloat16, device="cpu")
    assert [(g.page_size, g.num_pages, g.cache_ids) for g in cm.groups] == [(16, 16, [0, 1]), (8, 12, [2]), (16, 16, [3])]
    assert cm.kv[0].shape == (16, 2, 2, 16, 16) and cm.kv[0].dtype == torch.bfloat16
    assert cm.kv[2].shape == (12, 2, 1, 8, 32) and cm.page_size_of(2) == 8
    assert cm.kv[3].shape == (16, 16, 40) and cm.kv[3].dtype == torch.float32
    assert cm.state[4].shape == (4, 5, 3) and 5 not in cm.kv and 5 not in cm.state
    assert cm.bytes_per_token() == 2 * (2 * 2 * 16 * 2) + 2 * 1 * 32 * 2 + 40 * 4
    # the allocator has the groups' own page sizes and pools: 20 tokens take 2, 3 and 2 pages
    cm.alloc.add_request(1)
    cm.alloc.reserve(1, 20)
    assert [len(cm.alloc.block_table(1, g)) for g in range(3)] == [2, 3, 2]
    assert [cm.alloc.free_pages(g) for g in range(3)] == [14, 9, 14]
    cm.alloc.check()


def test_shrink_gives_the_pages_behind_back():
    a = PageAllocator([4, 8], [10, 6], [0, 0], 2)
    a.add_request(1)
    a.reserve(1, 30)
    a.commit(1, 30)
    assert a.free_pages(0) == 2 and a.free_pages(1) == 2
    before = a.block_table(1, 0).tolist()
    a.shrink(1, 9)
    assert a.block_table(1, 0).tolist() == before[:3] and a.num_computed(1) == 9
    assert a.free_pages(0) == 7 and a.free_pages(1) == 4
    a.check()
    a.shrink(1, 12)                                    # within what it has: no page more, no page less
    assert a.free_pages(0) == 7 and a.num_computed(1) == 12
    for bad in (-1, 13, 100):
        with pytest.raises(CacheError):
            a.shrink(1, bad)
    with pytest.raises(CacheError):
        a.shrink(2, 1)
    a.reserve(1, 20)                                   # and it grows again
    a.shrink(1, 0)
    assert a.free_pages(0) == 10 and a.free_pages(1) == 6
    a.check()
    b = PageAllocator([4], [10], [6], 1)
    b.add_request(1)
    b.reserve(1, 8)
    with pytest.raises(CacheError):
        b.shrink(1, 4)                                 # a window goes by position


def test_a_fork_shares_full_pages_and_copies_the_one_that_is_being_filled():
    a = PageAllocator([4, 8], [10, 6], [0, 0], 4)
    a.add_request(1)
    a.reserve(1, 18)                                    # pages behind the position stay the parent's
    a.commit(1, 10)
    a.set_request(1, prompt_len=7, temperature=0.5, seed=9)
    copies = a.fork(1, 2)
    parent, child = a.block_table(1, 0).tolist(), a.block_table(2, 0).tolist()
    assert child[:2] == parent[:2] and len(child) == 3 and child[2] not in parent
    assert [c.tolist() for c in copies] == [[[parent[2], child[2], 2]], [[a.block_table(1, 1)[1], a.block_table(2, 1)[1], 2]]]
    assert all(c.dtype == np.int32 for c in copies)
    assert a.num_computed(2) == 10 and a.record(2)["request_id"] == 2 and a.record(2)["prompt_len"] == 7 and a.record(2)["seed"] == 9
    assert a.free_pages(0) == 10 - 5 - 1 and a.free_pages(1) == 6 - 3 - 1
    a.check()
    # a fork of the fork where the pages are full: nothing to copy
    a.reserve(2, 16)
    a.commit(2, 16)
    assert [c.tolist() for c in a.fork(2, 3)] == [[], []]
    assert a.block_table(3, 0).tolist() == a.block_table(2, 0).tolist()
    a.check()
    # nobody writes into what is shared
    with pytest.raises(CacheError):
        a.commit(1, 7)
    with pytest.raises(CacheError):
        a.shrink(3, 13)
    with pytest.raises(CacheError):
        a.commit(3, 12)                                 # the page from 12 on is shared
    with pytest.raises(CacheError):
        a.shrink(3, 12)                                 # and in the other group it would be in the middle of one
    a.shrink(3, 8)
    a.reserve(3, 9)
    assert a.block_table(3, 0)[2] not in a.block_table(2, 0).tolist()
    a.check()
    a.commit(1, 11)                                     # its own page
    a.commit(1, 10)
    before = a.free_pages(0)
    a.release(1)
    assert a.free_pages(0) == before + 3                # two of five pages are others' as well
    a.check()
    a.release(2)
    a.release(3)
    assert a.free_pages(0) == 10 and a.free_pages(1) == 6 and a.free_slots() == 4
    a.check()


def test_a_fork_takes_all_or_nothing():
    a = PageAllocator([4, 8], [3, 3], [0, 0], 2)
    a.add_request(1)
    a.reserve(1, 10)
    a.commit(1, 10)                                     # all pages of the first group
    with pytest.raises(OutOfPages):
        a.fork(1, 2)
    assert not a.has(2) and a.free_pages(1) == 1 and a.free_slots() == 1
    a.check()
    a.shrink(1, 8)
    a.fork(1, 2)
    with pytest.raises(CacheError):
        a.fork(1, 3)                                    # no slot
    with pytest.raises(CacheError):
        a.fork(1, 2)                                    # there is one
    with pytest.raises(CacheError):
        a.fork(7, 8)
    a.check()
    empty = PageAllocator([4], [2], [0], 2)
    empty.add_request(1)
    assert [c.tolist() for c in empty.fork(1, 2)] == [[]] and empty.block_table(2).tolist() == []
    empty.check()


def test_forks_with_windows_and_chunks():
    """Pages that a window has passed are nobody's; shared ones go back when the last request has passed them."""
    a = PageAllocator([4, 4], [12, 12], [6, 0], 3, chunks=[0, 8])
    a.add_request(1)
    a.reserve(1, 14)
    a.commit(1, 14)
    free = [a.free_pages(g) for g in range(2)]
    copies = a.fork(1, 2)
    for g in range(2):
        parent, child = a.block_table(1, g).tolist(), a.block_table(2, g).tolist()
        assert parent[:3] == child[:3] and copies[g].tolist() == [[parent[3], child[3], 2]] and a.free_pages(g) == free[g] - 1
    a.check()
    a.reserve(1, 30)
    a.commit(1, 30)
    a.check()
    held = [p for g in range(2) for p in a.block_table(2, g).tolist() if p >= 0]
    assert held and a.num_computed(2) == 14
    a.release(1)
    a.check()
    a.reserve(2, 30)
    a.commit(2, 30)
    a.check()
    a.release(2)
    assert [a.free_pages(g) for g in range(2)] == [12, 12]
    a.check()


def test_nobody_goes_back_behind_what_is_shared():
    """A page of one's own, and one that is shared after it: going back to the first would lead into the second."""
    a = PageAllocator([4], [12], [6], 3)
    a.add_request(1)
    a.reserve(1, 12)
    a.commit(1, 12)
    a.fork(1, 2)
    a.reserve(2, 14)
    a.commit(2, 14)                                     # has passed the page of entries 4 to 7; 8 to 11 are shared
    assert a.block_table(2).tolist()[:2] == [-1, -1] and a.block_table(2)[2] == a.block_table(1)[2]
    for n in (5, 7, 8, 11):
        with pytest.raises(CacheError):
            a.commit(1, n)
    a.commit(1, 12)
    a.reserve(1, 20)
    a.commit(1, 17)
    a.commit(1, 16)                                     # nothing behind is another's
    a.check()


def test_random_forks_keep_the_books():
    rng = np.random.default_rng(4)
    pages = [40, 25]
    a = PageAllocator([3, 5], pages, [0, 7], 9)
    live = {}
    for step in range(3000):
        kind = rng.integers(5)
        if kind == 0 and len(live) < 9:
            a.add_request(step)
            live[step] = 0
        elif kind == 1 and live:
            parent = int(rng.choice(list(live)))
            try:
                a.fork(parent, step)
                live[step] = live[parent]
            except CacheError:
                assert not a.has(step)
        elif kind in (2, 3) and live:
            rid = int(rng.choice(list(live)))
            n = live[rid] + int(rng.integers(1, 9))
            try:
                a.reserve(rid, n)
                a.commit(rid, n)
                live[rid] = n
            except OutOfPages:
                pass
        elif live:
            rid = int(rng.choice(list(live)))
            a.release(rid)
            del live[rid]
        a.check()
    for rid in live:
        a.release(rid)
    a.check()
    assert [a.free_pages(g) for g in range(2)] == pages


@pytest.mark.parametrize("need,page_size,held", [
    (PagedKVNeed(2, 8), 4, 2),                                           # keys and values
    (PagedKVNeed(1, 8, page_shape=("page", 8)), 4, 2),
    (PagedKVNeed(1, 8, page_shape=(3, "page", 8)), 4, 2),
    (PagedKVNeed(4, 8, page_shape=("page", 4, 8)), 4, -1),               # as many heads as a page has tokens: not the tokens' axis
    (PagedKVNeed(4, 8, page_shape=(4, 8, "page")), 4, -1),
    (PagedKVNeed(1, 8, page_shape=("page",)), 4, -1),
    (PagedKVNeed(1, 8, page_shape=()), 4, -1),
    (PagedKVNeed(2, 8, page_size=2, tokens_per_entry=2), 4, -1),         # entries of two tokens
])
def test_a_fork_copies_tokens_only_along_their_own_axis(monkeypatch, need, page_size, held):
    """The page that is being filled is copied as far as it is full where its last axis but one is the tokens', whole elsewhere."""
    import torch
    from railgun_b200 import ops
    from railgun_b200.cache.manager import CacheManager
    copied = []
    monkeypatch.setattr(ops, "copy_pages", lambda caches, copies: copied.append((caches, np.asarray(copies).tolist())))
    cache = CacheManager({"a": need, "b": need}, page_size, 40, 3, torch.float32, "cpu")
    cache.alloc.add_request(1)
    cache.alloc.reserve(1, 6)
    cache.alloc.commit(1, 6)
    cache.fork(1, 2)
    (caches, copies), = copied
    assert [c.data_ptr() for c in caches] == [cache.kv["a"].data_ptr(), cache.kv["b"].data_ptr()]
    assert copies == [[int(cache.alloc.block_table(1)[1]), int(cache.alloc.block_table(2)[1]), held]]
    cache.alloc.check()


def test_who_would_move_entries_asks_whether_their_pages_are_shared():
    a = PageAllocator([4, 8], [12, 8], [0, 0], 3)
    a.add_request(1)
    a.reserve(1, 22)
    a.commit(1, 22)
    assert not a.shares(1) and not a.shares(1, 0) and not a.shares(1, 22)
    a.fork(1, 2)
    for r in (1, 2):                                    # entries 0 to 19 and 0 to 15; the pages behind are each one's own
        assert a.shares(r) and a.shares(r, 1) and a.shares(r, 1 << 30) and not a.shares(r, 0)
    with pytest.raises(CacheError):
        a.shares(7)
    for end in (-1, 1 << 31):
        with pytest.raises(CacheError):
            a.shares(1, end)
    a.release(1)
    assert not a.shares(2)
    windows = PageAllocator([4], [12], [6], 3)          # what a window has passed is nobody's
    windows.add_request(1)
    windows.reserve(1, 12)
    windows.commit(1, 12)
    windows.fork(1, 2)
    assert not windows.shares(2, 4) and windows.shares(2, 8)
    windows.reserve(1, 30)
    windows.commit(1, 30)
    assert not windows.shares(1) and not windows.shares(2)


def test_prompts_whose_pages_are_shared_are_not_evicted(monkeypatch):
    """Before any entry moves, and before a prompt goes on that would have to."""
    import torch
    from railgun_b200.examples import long_prompts
    moved = []
    monkeypatch.setattr(long_prompts.ops, "evict_entries", lambda *a, **k: moved.append(a))
    lp = object.__new__(long_prompts.LongPrompts)
    lp.alloc, lp.page_size, lp.budget, lp.max_entries = PageAllocator([4], [40], [0], 4), 4, 8, 100
    lp.protect_first = lp.protect_last = lp.nkv = lp.d = 1
    lp.kv = lp.weights = lp.places = [None]
    lp.device, lp.check_end = torch.device("cpu"), lambda n: None
    lp.alloc.add_request(1)
    lp.alloc.reserve(1, 14)
    lp.alloc.commit(1, 14)
    prompt = long_prompts.Prompt(1, lp.alloc.slot(1), 14, 14, 0)
    lp.alloc.fork(1, 2)
    with pytest.raises(ValueError, match="other requests"):
        lp.evict([prompt])
    with pytest.raises(ValueError, match="other requests"):
        lp.go_on(prompt, 3)
    assert not moved and lp.alloc.num_computed(1) == prompt.entries == 14
    lp.alloc.release(2)
    lp.evict([prompt])
    assert len(moved) == 1 and lp.alloc.num_computed(1) == prompt.entries == 8


def test_a_step_of_drafts_has_a_tree_for_each_text():
    """More trees than texts, or fewer: nothing is reserved, nothing is run."""
    from railgun_b200.engine.request import SamplingParams
    from railgun_b200.examples import drafts
    d = object.__new__(drafts.Drafts)
    d.alloc = PageAllocator([4], [40], [0], 4)
    texts = []
    for r in (1, 2):
        d.alloc.add_request(r)
        d.alloc.reserve(r, 5)
        d.alloc.commit(r, 5)
        texts.append(drafts.Text(r, [1, 2, 3, 4, 5, 6], 5, SamplingParams()))
    free, tree = d.alloc.free_pages(), ([-1], [6])
    for bad in ([], [tree], [tree] * 3):
        with pytest.raises(ValueError, match="a tree for each text"):
            d.step(texts, bad)
    assert d.step([], []) == []
    assert d.alloc.free_pages() == free and [t.checked for t in texts] == [0, 0]
