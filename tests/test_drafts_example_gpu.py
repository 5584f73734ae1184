"""Trees of guesses behind a model's layers (railgun_b200/examples/drafts.py): a text gets the tokens that it would get one by one."""
import random

import numpy as np
import pytest

from helpers import TINY, model_dir, prompts

pytestmark = pytest.mark.gpu


def drafts(name="A", dtype="float32", **more):
    from railgun_b200.examples.drafts import Drafts
    return Drafts(model_dir(name), dtype, page_size=TINY[name][2], **{**dict(max_tokens=800, max_requests=8), **more})


def engine(name, dtype="float32"):
    from railgun_b200.engine.engine import Engine
    return Engine(model_dir(name), dtype=dtype, block_size=TINY[name][2], num_gpu_blocks=256, max_model_len=200)


def repeating(vocab, n, seed):
    rng = random.Random(seed)
    few = [rng.randrange(vocab) for _ in range(5)]
    return [rng.choice(few) for _ in range(n)]


@pytest.mark.parametrize("temperature", [0.0, 0.9])
@pytest.mark.parametrize("name", sorted(TINY))
def test_the_tokens_are_the_engines(name, temperature):
    """Whatever is guessed, greedily and drawn: 32-bit, and the plain model's logits are far apart."""
    from railgun_b200.engine.request import SamplingParams
    vocab = TINY[name][0]["vocab_size"]
    texts = [repeating(vocab, 41, 1), *prompts(vocab, [17, 1], seed=3)]
    params = [SamplingParams(max_new_tokens=20, temperature=temperature, top_k=40 if temperature else 0, seed=s) for s in (5, 6, 7)]
    eng = engine(name)
    want = [eng.generate([t], p)[0].token_ids for t, p in zip(texts, params)]
    d = drafts(name)
    free = d.alloc.free_pages()
    read = [d.read(t, p) for t, p in zip(texts, params)]
    assert d.go_on(read, 20) == want
    assert all(t.brought >= 19 for t in read)
    for t in read:
        assert d.alloc.num_computed(t.request) == len(t.tokens) - 1
    for t in read:
        d.forget(t)
    assert d.alloc.free_pages() == free
    d.alloc.check()


@pytest.mark.parametrize("name", ["A", "C"])
def test_right_guesses_bring_several_tokens_a_step(name):
    """Trees that hold the engine's own tokens, beside wrong ones in front of them: all of a path is kept, in one step."""
    from railgun_b200.engine.request import SamplingParams
    vocab = TINY[name][0]["vocab_size"]
    prompt, = prompts(vocab, [23], seed=9)
    want = engine(name).generate([prompt], SamplingParams(max_new_tokens=14))[0].token_ids
    d = drafts(name)
    text = d.read(prompt)
    assert text.generated == want[:1]
    wrong = lambda t: (t + 1) % vocab  # noqa: E731
    # a wrong guess in front of every right one, and children of wrong ones
    parents, tokens, at = [-1], [want[0]], 0
    for t in want[1:6]:
        parents += [at, len(parents), at]
        tokens += [wrong(t), t, t]
        at = len(parents) - 1
    assert d.step([text], [(parents, tokens)]) == [want[1:7]] and text.checked == 16
    # half of a path
    assert d.step([text], [([-1, 0, 1, 2], [want[6], want[7], wrong(want[8]), want[9]])]) == [want[7:9]]
    assert d.step([text], [([-1], [want[8]])]) == [want[9:10]]
    assert d.go_on([text], 14) == [want]


def test_forks_share_pages_and_differ_in_their_draws():
    from railgun_b200.engine.request import SamplingParams
    name = "C"
    vocab, page = TINY[name][0]["vocab_size"], TINY[name][2]
    prompt = repeating(vocab, 3 * page + 5, 2)
    d, eng = drafts(name), engine(name)
    free = d.alloc.free_pages()
    first = d.read(prompt, SamplingParams(temperature=0.8, seed=1))
    texts = [first, d.fork(first, 2), d.fork(first, 3)]
    assert free - d.alloc.free_pages() == 4 + 2                          # three full pages are everybody's
    d.alloc.check()
    got = d.go_on(texts, 12)
    assert got[0] == eng.generate([prompt], SamplingParams(max_new_tokens=12, temperature=0.8, seed=1))[0].token_ids
    assert len({t[0] for t in got}) == 1 and len({tuple(t) for t in got}) == 3      # the first token was there when they forked
    # a greedy fork in the middle goes on like its parent
    greedy = d.read(prompt, SamplingParams())
    d.go_on([greedy], 7)
    twin = d.fork(greedy, 0)
    d.forget(greedy)
    want = eng.generate([prompt], SamplingParams(max_new_tokens=16))[0].token_ids
    assert d.go_on([twin], 16) == [want]
    for t in [*texts, twin]:
        d.forget(t)
    assert d.alloc.free_pages() == free
    d.alloc.check()


def test_in_bfloat16_tokens_are_near_the_best():
    """Every token is one that the plain model in 64 bits holds for as good as the best, within what bfloat16 loses."""
    from plain_llama import PlainLlama
    vocab = TINY["C"][0]["vocab_size"]
    d = drafts("C", "bfloat16", nodes=24)
    prompt = repeating(vocab, 60, 4)
    text = d.read(prompt)
    tokens, = d.go_on([text], 24)
    logits = PlainLlama(model_dir("C")).forward(prompt + tokens)
    tol = 6e-2 * np.abs(logits).max()
    for i, t in enumerate(tokens):
        row = logits[len(prompt) - 1 + i]
        assert row[t] >= row.max() - tol


def test_guesses():
    from railgun_b200.examples.drafts import guess
    assert guess([5], 8, 4) == ([-1], [5])
    assert guess([1, 2, 3, 1, 2], 8, 3) == ([-1, 0, 1, 2], [2, 3, 1, 2])
    parents, tokens = guess([7, 1, 8, 7, 1, 9, 7, 1], 16, 2)
    assert tokens[0] == 1 and {(parents[i], t) for i, t in enumerate(tokens) if i} == {(0, 9), (1, 7), (0, 8), (3, 7)}
    assert len(guess([1, 2] * 50, 5, 40)[0]) == 5 and guess([1, 2] * 50, 5, 0) == ([-1], [2])
    for n in range(1, 9):
        parents, _ = guess([1, 2, 1, 3, 1, 2, 1], n, 5)
        assert len(parents) <= n and all(p < i for i, p in enumerate(parents))


def test_what_it_refuses_leaves_everything_as_it_was():
    from railgun_b200.cache.manager import CacheError
    from railgun_b200.engine.request import SamplingParams
    vocab = TINY["A"][0]["vocab_size"]
    most = TINY["A"][0]["max_position_embeddings"]
    d = drafts("A", max_tokens=most + 40, max_requests=2)
    text = d.read(prompts(vocab, [most - 3], seed=1)[0])
    last, before = text.tokens[-1], (list(text.tokens), d.alloc.free_pages(), d.alloc.num_computed(text.request))
    for parents, tokens in (([-1, 0, 1, 2], [last, 1, 1, 1]), ([-1], [(last + 1) % vocab]), ([-1, 1], [last, 1]), ([0], [last]), ([-1, 0], [last, vocab]),
                            ([-1, 0], [last]), ([], [])):
        with pytest.raises(ValueError):
            d.step([text], [(parents, tokens)])
    with pytest.raises(ValueError):
        d.step([text, text], [([-1], [last])] * 2)
    with pytest.raises(ValueError):
        d.go_on([text], 6)
    with pytest.raises(CacheError):
        d.step([text], [([-1] + [0] * 99, [last] + [1] * 99)])           # no pages for so many
    with pytest.raises(ValueError):
        d.read([])
    with pytest.raises(ValueError):
        d.read([1], SamplingParams(temperature=-1.0))
    with pytest.raises(ValueError):
        drafts(nodes=0)
    forward, d.forward = d.forward, lambda batch: 1 / 0
    with pytest.raises(ZeroDivisionError):
        d.step([text], [([-1, 0], [last, 1])])
    free = d.alloc.free_pages()
    with pytest.raises(ZeroDivisionError):
        d.read([1, 2])
    assert d.alloc.free_pages() == free
    d.forward = forward
    assert (list(text.tokens), d.alloc.free_pages(), d.alloc.num_computed(text.request)) == before
    other = d.fork(text, 1)
    with pytest.raises(CacheError):
        d.fork(text, 2)                                                  # no slot
    assert len(d.go_on([text, other], 4)) == 2
    d.alloc.check()


def test_the_command(capsys):
    from railgun_b200.examples.drafts import main
    assert main(["--model", str(model_dir("A")), "--prompt-tokens", "60", "--samples", "3", "--max-tokens", "9", "--temperature", "0.7"]) == 0
    said = capsys.readouterr().out
    assert said.count("text ") == 3 and "nodes were checked" in said


@pytest.mark.parametrize("architecture", ["windows and states"])
def test_a_cache_of_several_kinds_forks(architecture):
    """Groups with pages of their own kinds and states of fixed size: the child's numbers are the parent's."""
    import torch
    from railgun_b200.cache.manager import CacheManager, PagedKVNeed, StateNeed
    needs = {0: PagedKVNeed(2, 16), 1: PagedKVNeed(2, 16), 2: PagedKVNeed(1, 32, window=24, page_size=8, pool_tokens=96),
             3: PagedKVNeed(0, 0, dtype="float32", page_shape=("page", 40)), 4: StateNeed((5, 3), "float32"), 5: None,
             6: PagedKVNeed(1, 8, tokens_per_entry=4), 7: StateNeed((), "float32")}
    cm = CacheManager(needs, page_size=16, max_tokens=256, max_requests=3, dtype=torch.bfloat16, device="cuda:0")
    g = torch.Generator(device="cuda:0").manual_seed(1)
    for t in [*cm.kv.values(), *cm.state.values()]:
        t.copy_(torch.randn(t.shape, generator=g, device="cuda:0"))
    cm.alloc.add_request(1)
    cm.alloc.reserve(1, 45)
    cm.alloc.commit(1, 45)
    before = {cid: t.clone() for cid, t in cm.kv.items()}
    cm.fork(1, 2)
    for group, info in enumerate(cm.groups):
        parent, child = cm.alloc.block_table(1, group), cm.alloc.block_table(2, group)
        last = 45 // info.page_size
        assert parent[:last].tolist() == child[:last].tolist() and parent[last] != child[last]
        held = 45 % info.page_size
        for cid in info.cache_ids:
            t = cm.kv[cid]
            if info.need.tokens_per_entry > 1:
                assert torch.equal(t[child[last]], t[parent[last]])
            else:
                assert torch.equal(t[child[last]][..., :held, :], t[parent[last]][..., :held, :])
                assert torch.equal(t[child[last]][..., held:, :], before[cid][child[last]][..., held:, :])
            others = [p for p in range(t.shape[0]) if p != child[last]]
            assert torch.equal(t[others], before[cid][others])
    for t in cm.state.values():
        assert torch.equal(t[cm.alloc.slot(2)], t[cm.alloc.slot(1)])
    cm.alloc.check()
