"""Guessed tokens checked together: the operators of drafted trees and of page copies, behind a Llama model's layers.

``Drafts.read`` runs a prompt through the model.  ``go_on`` continues texts, each on pages of its own: what the text says next is guessed from
where its last tokens stood before, several guesses make a tree, and one step checks the trees of all texts (``ops.draft_tree``,
``ops.tree_attention``); what the model itself chose is kept of them (``ops.keep_drafts``), and the pages behind go back.  A text gets the
tokens that it would get one by one, whatever was guessed: every node's token is chosen by the model's own logits, greedily or by
the draw that has the token's number.  ``fork`` lets another text go on from where one is (``CacheManager.fork``): full pages are shared,
the one that is being filled is copied (``ops.copy_pages``).

    python -m railgun_b200.examples.drafts --model DIR --prompt-tokens 200 --samples 4 --nodes 16
"""
from __future__ import annotations

import argparse
import copy
import dataclasses

import numpy as np
import torch

from .. import ops
from ..cache.manager import CacheManager
from ..engine.batch import StepBatch, StepEntry, build_step_batch
from ..engine.request import SamplingParams
from ..engine.runner import _CacheViews, build_model, parse_dtype
from ..parts.attention import PagedAttention
from .long_prompts import LongPromptAttention  # noqa: F401  (the mixer that attends as the step at hand wants it)


@dataclasses.dataclass
class Text:
    """A text that goes on: the tokens of the prompt and those generated so far, of which the last is not in the cache yet."""
    request: int
    tokens: list
    prompt: int
    params: SamplingParams
    checked: int = 0          # nodes that steps have checked, and tokens that they brought
    brought: int = 0

    @property
    def generated(self) -> list:
        return self.tokens[self.prompt:]


def guess(tokens, nodes: int, depth: int) -> tuple:
    """A tree of up to ``nodes`` guesses of what follows ``tokens``: what followed the last places where its last two tokens, or its
    last one, stood.  Returns (parents, tokens) with the last token as node 0; a path is ``depth`` guesses long at most."""
    parents, said, child = [-1], [tokens[-1]], {}
    for n in (2, 1):
        end = tokens[-n:]
        for at in range(len(tokens) - n - 1, -1, -1):
            if len(said) >= nodes or len(tokens) <= n:
                break
            if tokens[at:at + n] != end:
                continue
            node = 0
            for t in tokens[at + n:at + n + depth]:
                if (node, t) not in child:
                    if len(said) >= nodes:
                        break
                    child[node, t] = len(said)
                    parents.append(node)
                    said.append(t)
                node = child[node, t]
    return parents, said


class Drafts:
    def __init__(self, model_dir, dtype="bfloat16", device="cuda:0", page_size: int = 16, max_tokens: int = 16384, max_requests: int = 64,
                 nodes: int = 16, depth: int = 6):
        if nodes < 1 or nodes > ops.DRAFT_MOST or depth < 0:
            raise ValueError(f"a tree of 1 to {ops.DRAFT_MOST} nodes, and paths of no fewer than no guesses")
        from ..config.registry import load_config
        spec_of = load_config(model_dir)[0].model_spec

        def override(config):
            spec = spec_of(config)
            layers = tuple(dataclasses.replace(s, mixer=dataclasses.replace(s.mixer, kind="long_prompt_attention")) for s in spec.layers)
            return dataclasses.replace(spec, layers=layers)
        self.device, self.dtype = torch.device(device), parse_dtype(dtype)
        _, _, self.model = build_model(model_dir, self.dtype, device, spec_override=override)
        self.cache = CacheManager(self.model.cache_needs(), page_size, max_tokens, max_requests, self.dtype, self.device)
        if len(self.cache.groups) != 1 or self.cache.state or self.cache.groups[0].need.window:
            raise ValueError("drafts are for models whose layers all keep the keys and values of all tokens")
        self.alloc, self.views, self.page_size, self.nodes, self.depth = self.cache.alloc, _CacheViews(self.cache), page_size, nodes, depth
        self.kv = list(self.cache.kv.values())
        self.next_request = 0

    def ints(self, values, dtype=torch.int32) -> torch.Tensor:
        return torch.tensor(values, dtype=dtype).to(self.device)

    def choose(self, logits, texts_of_rows, numbers) -> torch.Tensor:
        """The model's token for every row: greedy, or the draw that has the token's number among the text's generated ones."""
        params = [t.params for t in texts_of_rows]
        if all(p.temperature == 0 for p in params):
            return ops.argmax(logits)
        return ops.sample(logits, self.ints([p.temperature for p in params], torch.float32), self.ints([p.top_k for p in params]),
                          self.ints([p.top_p for p in params], torch.float32), self.ints([p.seed for p in params], torch.int64),
                          self.ints(numbers, torch.int64))

    def forward(self, batch) -> torch.Tensor:
        logits = self.model.forward(batch, self.views)
        ops.tc_gemm_check()
        return logits

    # ---- a prompt, and texts that go on from where another is ----------------------------------------------------------
    def read(self, tokens, params: SamplingParams | None = None) -> Text:
        params = params or SamplingParams()
        params.validate()
        request, n = self.next_request, len(tokens)
        if n == 0:
            raise ValueError("a prompt is one token or more")
        self.next_request += 1
        batch = build_step_batch([StepEntry(request, list(tokens), [n - 1])], self.alloc, [self.page_size], self.model.vocab_size,
                                 self.model.spec.max_position, self.device)
        batch.attend = lambda part, qkv, cache: PagedAttention.attend(part, qkv, batch, cache)
        text = Text(request, list(tokens), n, params)
        try:
            text.tokens.append(int(self.choose(self.forward(batch), [text], [0])[0]))
            self.alloc.commit(request, n)
        except BaseException:
            self.alloc.release(request)
            raise
        return text

    def fork(self, text: Text, seed: int) -> Text:
        """Another text that goes on from here; its draws are those of ``seed``."""
        request = self.next_request
        self.cache.fork(text.request, request)
        self.next_request += 1
        return Text(request, list(text.tokens), text.prompt, dataclasses.replace(copy.copy(text.params), seed=seed))

    def forget(self, text: Text) -> None:
        self.alloc.release(text.request)

    # ---- trees -------------------------------------------------------------------------------------------------------
    def step(self, texts, trees) -> list:
        """Check a tree for each text: [(parents, tokens)], node 0 the text's last token.  Returns the tokens that each text gets, one
        or more, and adds them to it."""
        if len({t.request for t in texts}) != len(texts):
            raise ValueError("a text stands once in a step")
        if len(trees) != len(texts):
            raise ValueError(f"{len(trees)} trees; a step has a tree for each text, {len(texts)} of them")
        if not texts:
            return []
        counts, starts = [len(tokens) for _, tokens in trees], [len(t.tokens) - 1 for t in texts]
        for (parents, tokens), text, start in zip(trees, texts, starts):
            depths = []
            for i, (p, t) in enumerate(zip(parents, tokens)):
                if not 0 <= t < self.model.vocab_size or not (p == -1 if i == 0 else 0 <= p < i):
                    raise ValueError(f"node {i} of a tree: token {t}, parent {p}")
                depths.append(0 if i == 0 else depths[p] + 1)
            if not tokens or len(parents) != len(tokens) or len(tokens) > ops.DRAFT_MOST or tokens[0] != text.tokens[-1]:
                raise ValueError("a tree begins with the text's last token, and its nodes have a parent each")
            if start + max(depths) >= self.model.spec.max_position:
                raise ValueError(f"a text of {start + max(depths) + 1} tokens; the model ends at {self.model.spec.max_position}")
        done = False
        try:
            for text, start, n in zip(texts, starts, counts):
                self.alloc.reserve(text.request, start + n)
            tables = [self.alloc.block_table(t.request) for t in texts]
            width, T, most = max(len(t) for t in tables), sum(counts), max(counts)
            table = self.ints([[*t.tolist(), *[0] * (width - len(t))] for t in tables])
            slots = np.concatenate([t[(a + np.arange(n)) // self.page_size] * self.page_size + (a + np.arange(n)) % self.page_size
                                    for t, a, n in zip(tables, starts, counts)])
            cu, first = self.ints(np.cumsum([0, *counts])), self.ints(starts)
            parents, tokens = (self.ints(sum((list(x[k]) for x in trees), [])) for k in (0, 1))
            masks, positions = ops.draft_tree(parents, cu, first, max_rows=most)
            rows, longest = torch.arange(T + 1, dtype=torch.int32, device=self.device), max(a + n for a, n in zip(starts, counts))
            batch = StepBatch(
                num_tokens=T, num_requests=T, num_wanted=T, max_query_len=1, max_context_len=longest, token_ids=tokens, positions=positions,
                req_of_token=rows[:T], want_rows=rows[:T], cu_seqlens=rows, context_lens=positions + 1, start_pos=positions, state_slots=rows[:T],
                slot_mapping=[self.ints(slots)], block_table=[table], err_flag=torch.zeros(1, dtype=torch.int32, device=self.device),
                decode_only=True)

            def attend(part, qkv, cache):
                out = torch.empty(T, part.nh * part.d, dtype=qkv.dtype, device=qkv.device)
                ops.tree_attention(qkv[:, :part.nh * part.d], out, cache.kv, table, cu, first, masks, part.nh, part.nkv, part.d, part.scale,
                                   max_rows=most, max_context=longest)
                return out

            batch.attend = attend
            logits = self.forward(batch)
            numbers = [n for t, tree in zip(texts, trees) for n in self.numbers(t, tree[0])]
            chosen = self.choose(logits, [t for t, n in zip(texts, counts) for _ in range(n)], numbers)
            kept, _, fresh = ops.keep_drafts(self.kv, table, cu, first, parents, tokens, chosen, max_rows=most)
            kept, fresh = kept.tolist(), fresh.tolist()
            ops.tc_gemm_check()
            done = True
        finally:
            for i, (text, start) in enumerate(zip(texts, starts)):
                self.alloc.shrink(text.request, start + (kept[i] if done else 0))
        got = [f[:n] for f, n in zip(fresh, kept)]
        for text, new, n in zip(texts, got, counts):
            text.tokens += new
            text.checked += n
            text.brought += len(new)
        return got

    @staticmethod
    def numbers(text: Text, parents) -> list:
        """The number, among the text's generated tokens, of the token behind each node."""
        depths = []
        for i, p in enumerate(parents):
            depths.append(0 if i == 0 else depths[p] + 1)
        return [len(text.tokens) - text.prompt + x for x in depths]

    def go_on(self, texts, max_new_tokens: int) -> list:
        """Texts go on until they have ``max_new_tokens`` generated tokens each; the generated tokens of each."""
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be >= 1")
        for t in texts:
            if t.prompt + max_new_tokens - 1 > self.model.spec.max_position:
                raise ValueError(f"a text of {t.prompt + max_new_tokens - 1} tokens; the model ends at {self.model.spec.max_position}")
        while True:
            some = [t for t in texts if len(t.generated) < max_new_tokens]
            if not some:
                return [t.generated[:max_new_tokens] for t in texts]
            # a path no longer than what is still wanted: the last token is chosen behind it
            trees = [guess(t.tokens, self.nodes, min(self.depth, max_new_tokens - len(t.generated) - 1)) for t in some]
            self.step(some, trees)


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--model", required=True, help="a Llama model folder (railgun random-weights makes one)")
    ap.add_argument("--dtype", default="bfloat16")
    ap.add_argument("--prompt-tokens", type=int, default=200)
    ap.add_argument("--samples", type=int, default=4, help="texts that go on from the prompt")
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--nodes", type=int, default=16, help="of a tree, the last certain token among them")
    ap.add_argument("--max-tokens", type=int, default=32)
    a = ap.parse_args(argv)
    room = a.prompt_tokens + (a.samples + 1) * (a.max_tokens + a.nodes + 32)
    d = Drafts(a.model, a.dtype, max_tokens=room, max_requests=a.samples + 1, nodes=a.nodes)
    g = torch.Generator().manual_seed(0)
    few = torch.randint(0, d.model.vocab_size, (12,), generator=g).tolist()         # a prompt that repeats itself
    prompt = [few[i] for i in torch.randint(0, 12, (a.prompt_tokens,), generator=g).tolist()]
    first = d.read(prompt, SamplingParams(temperature=a.temperature))
    texts = [first, *(d.fork(first, seed) for seed in range(1, a.samples))]
    print(f"read {first.prompt} tokens; {len(texts)} texts go on; {d.alloc.free_pages()} pages are free")
    for i, tokens in enumerate(d.go_on(texts, a.max_tokens)):
        print(f"text {i}: {tokens}")
    print(f"{sum(t.checked for t in texts)} nodes were checked for {sum(t.brought for t in texts)} tokens")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
