"""The example of the operators over the cache (railgun_b200/examples/long_prompts.py) against a model in 64 bits that sees the same
entries: tokens, the weights that entries receive, and which of them stay.

The plain model keeps every layer's keys and values by the tokens' places in the text and masks the places that were dropped; it knows
nothing of pages, and keys and values that eviction moved are where they always were."""
import numpy as np
import pytest

from helpers import TINY, model_dir, prompts
from plain_llama import PlainLlama, embedding, linear, rms_norm, rope, swiglu

pytestmark = pytest.mark.gpu
# Logits of the tiny models, of the largest among them: what smoke() of the whole engine allows a token's logit.
LOGITS = {"float32": 1e-4, "bfloat16": 6e-2}
# A softmax weight's relative error is twice its score's error: scores of up to some 30, of activations that have come through two or
# three layers of sums of a few hundred products in 32 bits (some 5e-5), with as much room again.
WEIGHTS = 5e-3


class Plain(PlainLlama):
    """One text's keys and values, layer by layer, in 64 bits."""

    def start(self):
        self.keys = [np.zeros((0, self.nkv, self.d)) for _ in range(self.L)]
        self.values = [np.zeros((0, self.nkv, self.d)) for _ in range(self.L)]
        return self

    def fork(self):
        other = object.__new__(Plain)
        other.__dict__.update(self.__dict__)
        other.keys, other.values = list(self.keys), list(self.values)
        return other

    def feed(self, tokens, seen):
        """Tokens at the places behind the text so far; seen(layer, kv head, place of the row): the earlier places that it sees, or None for
        all.  Returns logits [T, V] and the softmax weights p[layer][head][row] over all places."""
        first, T, G = len(self.keys[0]), len(tokens), self.nh // self.nkv
        places = np.arange(first, first + T)
        x, weights = embedding(self.w["model.embed_tokens.weight"], tokens), []
        for li in range(self.L):
            lw = self.layer_weights(li)
            h = rms_norm(x, lw["ln1"], self.eps)
            q = rope(linear(h, lw["q"]).reshape(T, self.nh, self.d), places, self.inv_freq)
            self.keys[li] = np.concatenate([self.keys[li], rope(linear(h, lw["k"]).reshape(T, self.nkv, self.d), places, self.inv_freq)])
            self.values[li] = np.concatenate([self.values[li], linear(h, lw["v"]).reshape(T, self.nkv, self.d)])
            out, p = np.zeros((T, self.nh, self.d)), np.zeros((self.nh, T, first + T))
            for head in range(self.nh):
                k = head // G
                s = q[:, head] @ self.keys[li][:, k].T * self.d ** -0.5
                for t in range(T):
                    there = np.arange(first + T) <= first + t
                    some = seen(li, k, first + t)
                    if some is not None:
                        there[:first + t] = False
                        there[list(some)] = True
                    row = np.where(there, s[t], -np.inf)
                    row = np.exp(row - row.max())
                    p[head, t] = row / row.sum()
                out[:, head] = p[head] @ self.values[li][:, k]
            weights.append(p)
            x = x + linear(out.reshape(T, -1), lw["o"])
            h = rms_norm(x, lw["ln2"], self.eps)
            x = x + swiglu(h, lw["gate"], lw["up"], lw["down"])
        x = rms_norm(x, self.w["model.norm.weight"], self.eps)
        return linear(x, self.w["model.embed_tokens.weight"] if self.tied else self.w["lm_head.weight"]), weights


def kept(lp, prompt):
    """places[layer][kv head], and their weights"""
    n = prompt.entries
    return ([x[prompt.slot, :, :n].tolist() for x in lp.places], [x[prompt.slot, :, :n].double().cpu().numpy() for x in lp.weights])


def good(logits, token, dtype):
    assert logits[token] >= logits.max() - LOGITS[dtype] * np.abs(logits).max(), (token, int(logits.argmax()))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,n,budget,watch", [("A", 90, 32, 20), ("B", 131, 40, 32), ("C", 150, 48, 1), ("C", 70, 69, 70)])
def test_tokens_after_eviction_are_the_plain_models(name, n, budget, watch, dtype):
    from railgun_b200.examples.long_prompts import LongPrompts
    vocab, page = TINY[name][0]["vocab_size"], TINY[name][2]
    first, last, decay, exact = 3, 7, 0.75, dtype == "float32"
    text, *questions = prompts(vocab, [n, 3, 1, 2], seed=n)
    lp = LongPrompts(model_dir(name), dtype, page_size=page, num_pages=64, max_entries=256, budget=budget, watch=watch, protect_first=first,
                     protect_last=last)
    plain = Plain(model_dir(name)).start()
    G = plain.nh // plain.nkv
    prompt = lp.read(text)
    logits, p = plain.feed(text, lambda *a: None)
    good(logits[-1], prompt.next_token, dtype)
    # every entry's weight from the watched rows; the heaviest stay, the protected among them
    sums = [x.reshape(plain.nkv, G, n, n)[:, :, n - watch:].sum((1, 2)) for x in p]

    def check_kept(sums, newest):
        places, weights = kept(lp, prompt)
        for li in range(plain.L):
            for k in range(plain.nkv):
                mine = places[li][k]
                assert len(set(mine)) == len(mine) == prompt.entries
                if exact:
                    assert np.allclose(weights[li][k], sums[li][k][mine], rtol=WEIGHTS, atol=1e-12)
                assert set(range(first)) <= set(mine) and set(range(newest + 1 - last, newest + 1)) <= set(mine)
        return places

    def check_choice(before, places, sums, newest):
        """Of the places before, none that went is heavier than one that stayed and is not protected."""
        for li in range(plain.L):
            for k in range(plain.nkv):
                gone = set(before[li][k]) - set(places[li][k])
                free = [e for e in places[li][k] if first <= e <= newest - last]
                assert len(gone) == len(before[li][k]) - budget
                if exact and free:
                    assert max(sums[li][k][e] for e in gone) <= min(sums[li][k][e] for e in free) * (1 + 2 * WEIGHTS)

    places = check_kept(sums, n - 1)
    check_choice([[range(n)] * plain.nkv] * plain.L, places, sums, n - 1)
    # answers behind what stayed
    for q, answer in zip(questions, lp.answer(prompt, questions, 6)):
        one, all_ = plain.fork(), plain.fork()
        assert len(answer) == 6
        logits, _ = one.feed(q + answer[:-1], lambda li, k, at: [*places[li][k], *range(n, at)])
        for row, token in zip(logits[len(q) - 1:], answer):
            good(row, token, dtype)
        # what went would have had a say
        more, _ = all_.feed(q + answer[:-1], lambda *a: None)
        if budget < n - 1:
            assert np.abs(more - logits).max() > 10 * LOGITS["float32"] * np.abs(logits).max()
    # and on, within the budget: every step's token, weights and evictions
    evictions = 0
    for _ in range(3 * page):
        before, tokens = [[list(x) for x in layer] for layer in places], prompt.tokens
        token = prompt.next_token
        assert lp.go_on(prompt, 1, decay=decay) == [token]
        logits, p = plain.feed([token], lambda li, k, at: before[li][k])
        good(logits[-1], prompt.next_token, dtype)
        for li in range(plain.L):
            added = p[li].reshape(plain.nkv, G, tokens + 1).sum(1)
            grown = np.zeros((plain.nkv, tokens + 1))
            for k in range(plain.nkv):
                grown[k, before[li][k]] = decay * sums[li][k][before[li][k]]
            sums[li] = grown + added
        places = check_kept(sums, tokens)
        full = [[[*x, tokens] for x in layer] for layer in before]
        if len(places[0][0]) == len(before[0][0]) + 1:
            assert [[sorted(x) for x in layer] for layer in places] == [[sorted(x) for x in layer] for layer in full]
        else:
            evictions += 1
            check_choice(full, places, sums, tokens)
    assert evictions >= 2 and prompt.tokens == n + 3 * page
