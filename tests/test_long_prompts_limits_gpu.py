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
