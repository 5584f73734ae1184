"""Long prompts on a budget: the operators over the cache together, behind a Llama model's layers.

``LongPrompts.read`` runs a prompt through the model, adds up the weights that its last rows give every cached entry
(``ops.prompt_key_weights``), and keeps the ``budget`` heaviest entries of every layer and kv head (``ops.evict_entries``), whose pages
alone stay.  ``answer`` lets any number of questions be answered behind such a prompt, read once for all of them in every
step (``ops.prefix_attention``).  ``go_on`` continues one prompt for as long as it likes within its budget: every token adds to the
weights of the entries that it looks at (``ops.weighed_attention``), and a page above the budget the lightest entries go.

    python -m railgun_b200.examples.long_prompts --model DIR --budget 256 --prompt-tokens 2000

The attention part is the model's own with another ``attend``; an entry is where a token's key and value lie, its place the
token's position in the text: once entries are evicted, the two differ.
"""
from __future__ import annotations

import argparse
import dataclasses

import torch

from .. import ops
from ..cache.manager import PageAllocator
from ..engine.batch import StepBatch, StepEntry, build_step_batch
from ..engine.runner import build_model, parse_dtype
from ..parts.attention import PagedAttention
from ..parts.base import CacheView
from ..parts.registry import register_mixer


class LongPromptAttention(PagedAttention):
    """Attention as the step at hand wants it: ``batch.attend(part, qkv, cache)``."""

    def attend(self, qkv, batch, cache):
        return batch.attend(self, qkv, cache)


register_mixer("long_prompt_attention", LongPromptAttention)


@dataclasses.dataclass
class Prompt:
    """A prompt that has been read: what is kept of it."""
    request: int
    slot: int
    tokens: int               # of the text so far
    entries: int              # that are kept of each layer and kv head
    next_token: int


class LongPrompts:
    def __init__(self, model_dir, dtype="bfloat16", device="cuda:0", page_size: int = 16, num_pages: int = 1024, max_requests: int = 64,
                 max_entries: int = 8192, budget: int | None = None, watch: int = 32, protect_first: int = 4, protect_last: int = 32):
        def spec_of(config):
            spec = arch_spec(config)
            layers = tuple(dataclasses.replace(s, mixer=dataclasses.replace(s.mixer, kind="long_prompt_attention")) for s in spec.layers)
            return dataclasses.replace(spec, layers=layers)
        if (budget is not None and budget < 1) or min(watch, max_entries) < 1 or min(protect_first, protect_last) < 0:
            raise ValueError("at least one entry of budget and of room, one row that is watched, and no fewer protected entries than none")
        from ..config.registry import load_config
        arch_spec = load_config(model_dir)[0].model_spec
        self.device, self.dtype = torch.device(device), parse_dtype(dtype)
        _, _, self.model = build_model(model_dir, self.dtype, device, spec_override=spec_of)
        self.page_size, self.budget, self.watch = page_size, budget, watch
        self.protect_first, self.protect_last, self.max_entries = protect_first, protect_last, max_entries
        self.alloc = PageAllocator([page_size], [num_pages], [0], max_requests)
        self.next_request = 0
        part = self.model.layers[0].mixer
        self.nkv, self.d = part.nkv, part.d
        n = len(self.model.order)
        # per layer: pages; and per state slot the entries' weights and places
        self.kv = [torch.zeros(num_pages, 2, part.nkv, page_size, part.d, dtype=self.dtype, device=device) for _ in range(n)]
        shape = (max_requests, part.nkv, max_entries)
        self.weights = [torch.zeros(shape, device=device) for _ in range(n)]
        self.places = [torch.zeros(shape, dtype=torch.int32, device=device) for _ in range(n)]

    def view(self, cache_id) -> CacheView:
        return CacheView(cache_id, group=0, kv=self.kv[cache_id], page_size=self.page_size)

    def ints(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).to(self.device)

    def table_of(self, requests) -> torch.Tensor:
        tables = [self.alloc.block_table(r) for r in requests]
        width = max([1, *(len(t) for t in tables)])
        return self.ints([[*t.tolist(), *[0] * (width - len(t))] for t in tables])

    def check_end(self, tokens: int) -> None:
        if tokens > self.model.spec.max_position:
            raise ValueError(f"a text of {tokens} tokens; the model ends at {self.model.spec.max_position}")

    def forward(self, batch) -> torch.Tensor:
        logits = self.model.forward(batch, self)
        ops.tc_gemm_check()
        return logits

    # ---- a prompt ---------------------------------------------------------------------------------------------------
    def read(self, tokens) -> Prompt:
        n, request = len(tokens), self.next_request
        if not 0 < n <= self.max_entries:
            raise ValueError(f"a prompt of {n} tokens; there is room for {self.max_entries} entries")
        self.next_request += 1
        batch = build_step_batch([StepEntry(request, list(tokens), [n - 1])], self.alloc, [self.page_size], self.model.vocab_size,
                                 self.model.spec.max_position, self.device)
        rows = min(self.watch, n)
        cu, first, fresh = self.ints([0, rows]), self.ints([n - rows]), self.ints([0])

        def attend(part, qkv, cache):
            out = PagedAttention.attend(part, qkv, batch, cache)
            ops.prompt_key_weights(qkv[n - rows:], cache.kv, self.weights[cache.cache_id], batch.state_slots, batch.block_table[0],
                                   cu, first, fresh, part.nh, part.nkv, part.d, part.scale, max_rows=rows, max_context=n)
            return out

        batch.attend = attend
        try:
            prompt = Prompt(request, self.alloc.slot(request), n, n, int(ops.argmax(self.forward(batch))[0]))
            self.alloc.commit(request, n)
            for places in self.places:
                places[prompt.slot, :, :n] = torch.arange(n, dtype=torch.int32, device=self.device)
            if self.budget is not None and n > self.budget:
                self.evict([prompt])
        except BaseException:
            self.alloc.release(request)
            raise
        return prompt

    def check_own(self, prompt: Prompt) -> None:
        """Eviction moves entries into those that stay: their pages have to be the prompt's alone."""
        if self.alloc.shares(prompt.request, min(prompt.entries, self.budget)):
            raise ValueError(f"request {prompt.request}: entries cannot be evicted from pages that other requests hold, too")

    def evict(self, prompts) -> None:
        """Every layer's and kv head's lightest entries above the budget go, and with them the pages behind."""
        for p in prompts:
            self.check_own(p)
        table, slots = self.table_of([p.request for p in prompts]), self.ints([p.slot for p in prompts])
        lens, keep = self.ints([p.entries for p in prompts]), self.ints([self.budget] * len(prompts))
        newest = self.ints([p.tokens - 1 for p in prompts])
        # more protected entries than the budget holds: of equals the first would stay, but the newest are what is wanted
        first = min(self.protect_first, self.budget)
        last = min(self.protect_last, self.budget - first)
        for kv, weights, places in zip(self.kv, self.weights, self.places):
            ops.evict_entries(kv, weights, places, weights, places, slots, table, lens, keep, newest, self.nkv, self.d, first, last,
                              max_context=max(p.entries for p in prompts))
        for p in prompts:
            p.entries = min(p.entries, self.budget)
            self.alloc.shrink(p.request, p.entries)

    def step(self, requests, tokens, positions, entries, attend) -> list:
        """One token a request, at ``positions`` in the text, to be its entry ``entries``; the tokens that follow."""
        T = len(requests)
        for r, e in zip(requests, entries):
            self.alloc.reserve(r, e + 1)
        table = self.table_of(requests)
        at = self.ints(entries)
        page = table.gather(1, (at // self.page_size).long()[:, None])[:, 0]
        rows = torch.arange(T + 1, dtype=torch.int32, device=self.device)
        batch = StepBatch(
            num_tokens=T, num_requests=T, num_wanted=T, max_query_len=1, max_context_len=max(entries) + 1, token_ids=self.ints(tokens),
            positions=self.ints(positions), req_of_token=rows[:T], want_rows=rows[:T], cu_seqlens=rows, context_lens=at + 1, start_pos=at,
            state_slots=self.ints([self.alloc.slot(r) for r in requests]), slot_mapping=[page * self.page_size + at % self.page_size],
            block_table=[table], err_flag=torch.zeros(1, dtype=torch.int32, device=self.device), decode_only=True)

        def run(part, qkv, cache):
            out = torch.empty(T, part.nh * part.d, dtype=qkv.dtype, device=qkv.device)
            attend(part, qkv[:, :part.nh * part.d], out, batch, cache)
            return out

        batch.attend = run
        after = ops.argmax(self.forward(batch)).tolist()
        for r, e in zip(requests, entries):
            self.alloc.commit(r, e + 1)
        return after

    # ---- many questions behind one prompt ---------------------------------------------------------------------------
    def answer(self, prompt: Prompt, questions, max_new_tokens: int) -> list:
        """Greedy answers to the questions (lists of tokens), all behind ``prompt``."""
        if not questions:
            return []
        if any(len(q) < 1 or min(q) < 0 or max(q) >= self.model.vocab_size for q in questions):
            raise ValueError(f"a question is one token or more, each in [0, {self.model.vocab_size})")
        T, longest = len(questions), max(len(q) for q in questions) + max_new_tokens
        self.check_end(prompt.tokens + longest - 1)
        requests = [self.next_request + i for i in range(T)]
        self.next_request += T
        try:
            for r in requests:
                self.alloc.add_request(r)
                self.alloc.reserve(r, longest - 1)
            groups, prefix = self.ints([[0, T, prompt.entries]]), self.table_of([prompt.request])
            answers = [[] for _ in questions]
            feed = [q[0] for q in questions]
            for i in range(longest - 1):
                def attend(part, q, out, batch, cache):
                    ops.prefix_attention(q, out, cache.kv, prefix, groups, batch.block_table[0], batch.start_pos, part.nh, part.nkv, part.d,
                                         part.scale, max_rows=T, max_prefix=prompt.entries, max_own=i + 1)
                after = self.step(requests, feed, [prompt.tokens + i] * T, [i] * T, attend)
                for t, q in enumerate(questions):
                    if i + 1 >= len(q) and len(answers[t]) < max_new_tokens:
                        answers[t].append(after[t])
                    feed[t] = q[i + 1] if i + 1 < len(q) else after[t]
        finally:
            for r in requests:
                if self.alloc.has(r):
                    self.alloc.release(r)
        return answers

    # ---- one prompt goes on within its budget --------------------------------------------------------------------------
    def go_on(self, prompt: Prompt, max_new_tokens: int, decay: float = 1.0) -> list:
        """Greedy tokens behind ``prompt``; a page above the budget the lightest entries go."""
        self.check_end(prompt.tokens + max_new_tokens)
        most, out = prompt.entries + max_new_tokens, []
        if self.budget is not None:
            if most >= self.budget + self.page_size:    # entries will go
                self.check_own(prompt)
            most = min(most, self.budget + self.page_size)
        if most > self.max_entries:
            raise ValueError(f"{most} entries; there is room for {self.max_entries}")
        self.alloc.reserve(prompt.request, most)        # all there is need for, or nothing is done
        for _ in range(max_new_tokens):
            token, entry = prompt.next_token, prompt.entries
            out.append(token)
            for places in self.places:
                places[prompt.slot, :, entry] = prompt.tokens

            def attend(part, q, o, batch, cache):
                ops.weighed_attention(q, o, cache.kv, self.weights[cache.cache_id], batch.state_slots, batch.block_table[0],
                                      batch.start_pos, part.nh, part.nkv, part.d, part.scale, max_context=entry + 1, decay=decay)
            prompt.next_token = self.step([prompt.request], [token], [prompt.tokens], [entry], attend)[0]
            prompt.tokens += 1
            prompt.entries += 1
            if self.budget is not None and prompt.entries >= self.budget + self.page_size:
                self.evict([prompt])
        return out

    def forget(self, prompt: Prompt) -> None:
        self.alloc.release(prompt.request)


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--model", required=True, help="a Llama model folder (railgun random-weights makes one)")
    ap.add_argument("--dtype", default="bfloat16")
    ap.add_argument("--budget", type=int, default=256, help="entries kept of each layer and kv head")
    ap.add_argument("--prompt-tokens", type=int, default=1000)
    ap.add_argument("--questions", type=int, default=8)
    ap.add_argument("--max-tokens", type=int, default=16)
    a = ap.parse_args(argv)
    pages = lambda n: -(-n // 16)  # noqa: E731
    lp = LongPrompts(a.model, a.dtype, num_pages=pages(a.prompt_tokens + a.max_tokens) + a.questions * pages(5 + a.max_tokens),
                     max_requests=a.questions + 2, max_entries=a.prompt_tokens + a.max_tokens + 64, budget=a.budget)
    g = torch.Generator().manual_seed(0)
    draw = lambda n: torch.randint(0, lp.model.vocab_size, (n,), generator=g).tolist()  # noqa: E731
    prompt = lp.read(draw(a.prompt_tokens))
    print(f"read {prompt.tokens} tokens, kept {prompt.entries} entries of each layer and kv head; {lp.alloc.free_pages()} pages are free")
    for i, tokens in enumerate(lp.answer(prompt, [draw(3 + i % 3) for i in range(a.questions)], a.max_tokens)):
        print(f"answer {i}: {tokens}")
    print(f"and on: {lp.go_on(prompt, a.max_tokens)}")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
