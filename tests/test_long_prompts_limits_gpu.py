"""The example of the operators over the cache (railgun_b200/examples/long_prompts.py): its bookkeeping, and what it refuses."""
import pytest

from helpers import TINY, model_dir, prompts

pytestmark = pytest.mark.gpu


def long_prompts(name="C", dtype="float32", **more):
    from railgun_b200.examples.long_prompts import LongPrompts
    return LongPrompts(model_dir(name), dtype, page_size=TINY[name][2], **{**dict(num_pages=64, max_entries=300), **more})


def text(name, *lengths, seed=7):
    return prompts(TINY[name][0]["vocab_size"], lengths, seed=seed)


def test_the_allocator_knows_what_is_in_the_cache():
    lp = long_prompts()
    prompt = lp.read(text("C", 40)[0])
    lp.go_on(prompt, 12)
    assert prompt.entries == 52 and lp.alloc.num_computed(prompt.request) == 52
    lp = long_prompts(budget=30, protect_last=4)
    prompt = lp.read(text("C", 40)[0])
    assert lp.alloc.num_computed(prompt.request) == 30
    for n in (5, 11, 1):                                                # one more than a page above the budget, and on
        lp.go_on(prompt, n)
        assert lp.alloc.num_computed(prompt.request) == prompt.entries < 30 + 16
    lp.alloc.check()


def test_positions_end_where_the_model_ends():
    """Behind its last position a model has no rotation: nothing is computed there, and nothing has changed."""
    most = TINY["A"][0]["max_position_embeddings"]
    first, question = text("A", most - 6, 3)
    lp = long_prompts("A")
    prompt = lp.read(first)
    before = (prompt.tokens, prompt.entries, prompt.next_token, lp.alloc.free_pages())
    with pytest.raises(ValueError):
        lp.go_on(prompt, 7)
    with pytest.raises(ValueError):
        lp.answer(prompt, [question[:1], question], 5)
    assert (prompt.tokens, prompt.entries, prompt.next_token, lp.alloc.free_pages()) == before
    assert [len(a) for a in lp.answer(prompt, [question[:1], question], 4)] == [4, 4]
    tokens = lp.go_on(prompt, 6)
    assert len(tokens) == 6 and prompt.tokens == most
    with pytest.raises(ValueError):
        lp.go_on(prompt, 1)


def test_there_is_room_for_so_many_entries():
    lp = long_prompts(max_entries=50)
    prompt = lp.read(text("C", 40)[0])
    with pytest.raises(ValueError):
        lp.go_on(prompt, 11)
    assert prompt.entries == prompt.tokens == 40                        # refused before anything was done
    assert len(lp.go_on(prompt, 10)) == 10
    lp = long_prompts(max_entries=46, budget=30, protect_last=4)         # a page above the budget is all that it takes
    prompt = lp.read(text("C", 46)[0])
    assert len(lp.go_on(prompt, 60)) == 60
    lp = long_prompts(max_entries=45, budget=30, protect_last=4)
    prompt = lp.read(text("C", 45)[0])
    with pytest.raises(ValueError):
        lp.go_on(prompt, 60)


@pytest.mark.parametrize("bad", [[], [-1], [3, TINY["C"][0]["vocab_size"]], [1 << 40]])
def test_questions_are_tokens_of_the_model(bad):
    """A token that the model does not have would be a row of zeros, and answered."""
    lp = long_prompts()
    prompt = lp.read(text("C", 20)[0])
    free = lp.alloc.free_pages()
    with pytest.raises(ValueError):
        lp.answer(prompt, [[1, 2], bad], 3)
    assert lp.alloc.free_pages() == free
    assert lp.answer(prompt, [], 3) == []


@pytest.mark.parametrize("bad", [dict(budget=0), dict(budget=-3), dict(watch=0), dict(protect_first=-1), dict(protect_last=-1), dict(max_entries=0)])
def test_what_is_asked_of_the_budget(bad):
    with pytest.raises(ValueError):
        long_prompts(**bad)


def test_what_fails_gives_everything_back():
    from railgun_b200.cache.manager import CacheError
    lp = long_prompts(num_pages=4, max_requests=4)
    prompt = lp.read(text("C", 30)[0])                                  # two pages of 16
    for questions, n in (([[1, 2]] * 3, 3), ([[1]], 40), ([[1]] * 4, 2)):  # pages for two, for 32 tokens; slots for three
        with pytest.raises(CacheError):
            lp.answer(prompt, questions, n)
        assert lp.alloc.free_pages() == 2
    before = (prompt.tokens, prompt.entries, prompt.next_token)
    with pytest.raises(CacheError):
        lp.go_on(prompt, 40)
    assert (prompt.tokens, prompt.entries, prompt.next_token) == before and lp.alloc.free_pages() == 2
    assert len(lp.answer(prompt, [[1, 2]] * 2, 3)) == 2
    with pytest.raises(CacheError):
        lp.read(text("C", 100)[0])
    lp.prefill_fails = lambda batch: 1 / 0
    forward, lp.forward = lp.forward, lp.prefill_fails
    with pytest.raises(ZeroDivisionError):
        lp.read(text("C", 20)[0])
    with pytest.raises(ZeroDivisionError):
        lp.answer(prompt, [[1]], 2)
    lp.forward = forward
    assert lp.alloc.free_pages() == 2
    lp.forget(prompt)
    lp.alloc.check()
    prompt = lp.read(text("C", 64)[0])                                  # every page and slot can be had again
    lp.forget(prompt)


@pytest.mark.parametrize("budget,first,last", [(32, 4, 32), (20, 4, 32), (3, 4, 32), (40, 50, 3)])
def test_the_newest_entries_stay_in_a_small_budget(budget, first, last):
    """Fewer entries than there are protected ones: the first of the text, and of the others the newest."""
    lp = long_prompts(budget=budget, protect_first=first, protect_last=last)
    prompt = lp.read(text("C", 100)[0])
    head = min(first, budget)
    for n in (0, 40):
        lp.go_on(prompt, n)
        tail = min(last, budget - head)
        for places in lp.places:
            for kept in places[prompt.slot, :, :prompt.entries].tolist():
                assert len(kept) == len(set(kept)) and set(range(head)) <= set(kept)
                assert set(range(prompt.tokens - tail, prompt.tokens)) <= set(kept)
