"""The operators over the cache together, behind a model's layers (railgun_b200/examples/long_prompts.py)."""
import pytest

from helpers import TINY, model_dir, prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", sorted(TINY))
def test_without_a_budget_the_tokens_are_the_engines(name):
    """Nothing is evicted: the same sums in another order.  32-bit, and the plain model's logits are far apart."""
    from railgun_b200.engine.engine import Engine
    from railgun_b200.engine.request import SamplingParams
    from railgun_b200.examples.long_prompts import LongPrompts
    vocab, page = TINY[name][0]["vocab_size"], TINY[name][2]
    text, *questions = prompts(vocab, [75, 3, 1, 6, 2], seed=5)
    lp = LongPrompts(model_dir(name), "float32", page_size=page, num_pages=128, max_entries=200)
    prompt = lp.read(text)
    eng = Engine(model_dir(name), dtype="float32", block_size=page, num_gpu_blocks=256, max_model_len=200)
    want = [o.token_ids for o in eng.generate([text + q for q in questions], SamplingParams(max_new_tokens=9))]
    assert lp.answer(prompt, questions, 9) == want
    assert lp.go_on(prompt, 12) == eng.generate([text], SamplingParams(max_new_tokens=12))[0].token_ids
    lp.forget(prompt)
    assert lp.alloc.free_pages() == 128
    lp.alloc.check()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_within_a_budget(dtype):
    """Entries, pages, places and weights stay within it, the first and the newest entries among them."""
    import torch
    from railgun_b200.examples.long_prompts import LongPrompts
    vocab, page = TINY["C"][0]["vocab_size"], TINY["C"][2]
    text, question = prompts(vocab, [150, 3], seed=6)
    lp = LongPrompts(model_dir("C"), dtype, page_size=page, num_pages=64, max_entries=300, budget=48, protect_last=8)
    prompt = lp.read(text)
    assert prompt.entries == 48 and lp.alloc.free_pages() == 64 - 48 // page
    kept = lp.places[0][prompt.slot, :, :48].sort(-1).values
    for head in kept:
        places = head.tolist()
        assert len(set(places)) == 48 and places[:4] == [0, 1, 2, 3] and places[-8:] == list(range(142, 150))
    assert bool((lp.weights[0][prompt.slot, :, :48] > 0).all())
    assert all(len(a) == 5 for a in lp.answer(prompt, [question, question[:1]], 5))
    tokens = lp.go_on(prompt, 60)
    assert len(tokens) == 60 and 48 <= prompt.entries < 48 + page and prompt.tokens == 210
    newest = lp.places[1][prompt.slot, :, :prompt.entries]
    assert bool((newest.amax(-1) == 209).all()) and all(len(set(h.tolist())) == prompt.entries for h in newest)
    # the rows' weights of every step were shared out among the entries: no more than heads a step, no entry negative
    w = lp.weights[0][prompt.slot, :, :prompt.entries]
    assert bool(torch.isfinite(w).all()) and bool((w >= 0).all())
    lp.alloc.check()


def test_the_command(capsys):
    from railgun_b200.examples.long_prompts import main
    assert main(["--model", str(model_dir("A")), "--budget", "32", "--prompt-tokens", "90", "--questions", "3", "--max-tokens", "5"]) == 0
    said = capsys.readouterr().out
    assert "kept 32 entries" in said and said.count("answer") == 3
