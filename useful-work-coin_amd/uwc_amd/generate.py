"""Greedy generation and beam search for several prompts at once over the paged 8-bit cache (uwc_amd.kv): a Hugging
Face Qwen3 or Llama CausalLM in bfloat16 or float16, its linears plain or replaced by
uwc_amd.model.convert_qwen3 (integer or mined) or convert_4bit, without the cache and attention of transformers. The
reference's counterpart is DetQwen3.generate_greedy (runtime/detrt/qwen3.py:296-334): one sequence, whole
fp32 rows.

    gen = PagedGenerator(model, pages=4096)
    tokens = gen.generate([prompt_a, prompt_b], steps=64)
    system = gen.keep(instructions)                                  # a prefix that many prompts have
    best = gen.beam([question_a, question_b], steps=64, beams=4, prefix=system)

Prompts run packed, in chunks of at most `chunk` tokens each; then every step is one token of every
sequence. The tokens of a step stay on the GPU and feed the next one, so nothing is copied to the host
before the end. Beams share the pages of what they have in common (uwc_amd.pages): a step
copies the last page of a beam that goes on more than once, and frees those of one that ends.
"""
from __future__ import annotations

import torch

from . import kv, pages as pool


def _qkv(att):
    """The projection of a layer's input to its packed q, k and v heads: one call where convert_qwen3
    has fused them."""
    shared = getattr(att.q_proj, "shared", None)
    if shared is not None:
        return shared.ml
    return lambda x: torch.cat([att.q_proj(x), att.k_proj(x), att.v_proj(x)], -1)


def _rotation(rotary, n: int, dev):
    """cos and sin (n, head_dim) of positions 0 .. n - 1, for sequences of any length up to n: the rotation must not
    depend on the length, as that of dynamic and long-context scalings does past the length a model was trained at."""
    def table(n):
        cos, sin = rotary(torch.zeros(1, dtype=torch.float32, device=dev), torch.arange(n, device=dev)[None])
        return cos[0].float().contiguous(), sin[0].float().contiguous()

    whole = table(n)
    few = table(min(n, 2))  # also leaves the module as short sequences want it
    if not all(torch.allclose(a[:2], b, rtol=1e-4, atol=0.0) for a, b in zip(whole, few)):
        raise AssertionError(f"PagedGenerator: the model's rotation at {n} positions is another than that of short sequences; "
                             "give `positions` up to which it stays the same")
    return whole


class Prefix:
    """Tokens kept in a generator's cache: the pages that hold them, in their order, and how many tokens they are."""

    def __init__(self, pages: list[int], length: int):
        self.pages, self.length = pages, length


class PagedGenerator:
    """The layers of `model` over caches of `pages` pages of `page` tokens each, shared by all sequences.
    positions: rows of the rotation tables (the model's own limit by default), the longest that a sequence may get; a
    model whose rotation depends on the length up to there is refused."""

    def __init__(self, model, pages: int, page: int = 64, positions: int | None = None):
        cfg = model.config
        self.model, self.page = model, page
        self.H, self.Hkv = cfg.num_attention_heads, cfg.num_key_value_heads
        self.hd = getattr(cfg, "head_dim", None) or cfg.hidden_size // self.H
        self.dtype = model.model.embed_tokens.weight.dtype
        dev = self.dev = model.model.embed_tokens.weight.device
        self.caches = [kv.new_cache(pages, self.Hkv, self.hd, page, dev) for _ in model.model.layers]
        self.free = list(range(pages))
        self.kept: list[Prefix] = []
        self.positions = positions or cfg.max_position_embeddings
        self.cos, self.sin = _rotation(model.model.rotary_emb, self.positions, dev)
        self.layers = []
        for layer in model.model.layers:
            att = layer.self_attn
            norms = [getattr(att, n, None) for n in ("q_norm", "k_norm")]
            self.layers.append((layer, _qkv(att), *[n.weight.detach().float() if n is not None else None for n in norms],
                                norms[0].variance_epsilon if norms[0] is not None else 0.0,
                                int(getattr(att, "sliding_window", None) or 0), att.scaling))

    @torch.no_grad()
    def forward(self, ids, table, ctx, lens, cu, max_new: int, max_len: int) -> torch.Tensor:
        """Hidden rows (T, hidden) of new tokens `ids` (T,), packed as uwc_amd.kv packs them: sequence b has
        ctx[b] tokens in the cache before and lens[b] after."""
        x = self.model.model.embed_tokens(ids)
        for cache, (layer, qkv, qn, kn, eps, window, scale) in zip(self.caches, self.layers):
            y = qkv(layer.input_layernorm(x)).to(self.dtype)
            q = kv.append(cache, y, table, ctx, self.cos, self.sin, cu=cu, q_norm=qn, k_norm=kn, eps=eps)
            o = kv.attend(cache, q, table, lens, cu=cu, max_new=max_new, max_len=max_len, window=window, scale=scale)
            x = x + layer.self_attn.o_proj(o.view(len(ids), -1)).to(self.dtype)
            x = x + layer.mlp(layer.post_attention_layernorm(x)).to(self.dtype)
        return self.model.model.norm(x)

    def _ints(self, x) -> torch.Tensor:
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def _sizes(self, fn, prompts, steps: int, chunk: int, start: int = 0) -> list[int]:
        sizes = [len(p) for p in prompts]
        if not sizes or min(sizes) < 1 or steps < 1 or chunk < 1:
            raise AssertionError(f"{fn}: prompts of at least one token, steps and chunk of at least one")
        if start + max(sizes) + steps - 1 > self.positions:
            raise AssertionError(f"{fn}: {start + max(sizes)} + {steps} tokens exceed {self.positions} positions")
        return sizes

    def _room(self, fn, need: int):
        if need > len(self.free):
            raise AssertionError(f"{fn}: {need} pages are needed, {len(self.free)} are free")

    def _prefill(self, prompts, table, start: int, chunk: int) -> torch.Tensor:
        """Hidden rows of the prompts' last tokens; `start` tokens of every sequence are in the cache already."""
        B, sizes = len(prompts), [len(p) for p in prompts]
        last = torch.empty((B, self.model.config.hidden_size), dtype=self.dtype, device=self.dev)
        for at in range(0, max(sizes), chunk):
            done = [min(n, at) for n in sizes]
            new = [min(n - d, chunk) for n, d in zip(sizes, done)]
            cu = [0]
            for n in new:
                cu.append(cu[-1] + n)
            ids = torch.tensor([t for p, d, n in zip(prompts, done, new) for t in p[d:d + n]], device=self.dev)
            h = self.forward(ids, table, self._ints([start + d for d in done]), self._ints([start + d + n for d, n in zip(done, new)]),
                             self._ints(cu), max(new), start + max(d + n for d, n in zip(done, new)))
            ends = [b for b in range(B) if new[b] and done[b] + new[b] == sizes[b]]
            last[ends] = h[[cu[b + 1] - 1 for b in ends]]
        return last

    @torch.no_grad()
    def generate(self, prompts, steps: int, chunk: int = 2048) -> list[list[int]]:
        """`steps` >= 1 greedy tokens after each of the prompts (lists of at least one token id)."""
        sizes = self._sizes("generate", prompts, steps, chunk)
        held = [-(-(n + steps - 1) // self.page) for n in sizes]
        self._room("generate", sum(held))
        mine = [[self.free.pop() for _ in range(n)] for n in held]
        try:
            table = self._ints([p + [-1] * (max(held) - len(p)) for p in mine])
            out = [self.model.lm_head(self._prefill(prompts, table, 0, chunk)).argmax(-1)]
            ctx = self._ints(sizes)
            for i in range(steps - 1):
                h = self.forward(out[-1], table, ctx, ctx + 1, None, 1, max(sizes) + i + 1)
                out.append(self.model.lm_head(h).argmax(-1))
                ctx = ctx + 1
            return torch.stack(out, 1).tolist()
        finally:
            for p in mine:
                self.free.extend(reversed(p))

    @torch.no_grad()
    def beam(self, prompts, steps: int, beams: int, prefix: Prefix | None = None, chunk: int = 2048):
        """For each of the prompts, which follow `prefix` where it is given, the `beams` continuations of `steps` tokens that a beam search
        ends with, the likeliest first: (tokens, the sum of their log probabilities)."""
        start = prefix.length if prefix is not None else 0
        sizes = self._sizes("beam", prompts, steps, chunk, start)
        B, longest, page = len(prompts), max(sizes), self.page
        if not 1 <= beams <= self.model.config.vocab_size or B * beams > pool.ROWS:
            raise AssertionError(f"beam: {beams} beams of {B} prompts (at least one, no more than the vocabulary, {pool.ROWS} in all)")
        if prefix is not None and not any(p is prefix for p in self.kept):
            raise AssertionError("beam: the prefix is not kept here")
        pages = lambda n: -(-n // page)  # noqa: E731
        self._room("beam", B * (pages(start + longest) - start // page) + sum(
            beams * (pages(start + n + steps - 1) - (start + n) // page) for n in sizes))
        first = prefix.pages if prefix is not None else []
        table = self._ints([first + [-1] * (pages(start + longest + steps - 1) - len(first))])
        refs = torch.ones(self.caches[0][0].shape[0], dtype=torch.int32)  # those not free are held by prefixes
        refs[self.free] = 0
        refs[first] += 1  # and by the row that the prompts branch from
        refs = refs.to(self.dev)
        table, _, refs, _ = pool.fork(self.caches, table, self._ints([start]), refs, self._ints([0] * B), room=longest)
        logp = torch.log_softmax(self.model.lm_head(self._prefill(prompts, table, start, chunk)).float(), -1)
        V = logp.shape[1]
        score, tokens = logp.topk(beams)
        row = torch.arange(B, device=self.dev)[:, None] * beams
        told = tokens.reshape(-1, 1)
        lens = self._ints([start + n for n in sizes])
        parents = torch.arange(B, dtype=torch.int32, device=self.dev).repeat_interleave(beams)
        for i in range(steps - 1):
            table, lens, refs, _ = pool.fork(self.caches, table, lens, refs, parents, room=1)
            h = self.forward(told[:, -1], table, lens, lens + 1, None, 1, start + longest + i + 1)
            lens = lens + 1
            logp = torch.log_softmax(self.model.lm_head(h).float(), -1)
            score, best = (score.view(B, beams, 1) + logp.view(B, beams, V)).view(B, beams * V).topk(beams)
            chosen = (row + best // V).flatten()
            told = torch.cat([told[chosen], (best % V).view(-1, 1)], 1)
            parents = chosen.int()
        told, score = told.view(B, beams, steps).tolist(), score.tolist()
        return [list(zip(t, s)) for t, s in zip(told, score)]

    @torch.no_grad()
    def keep(self, tokens, chunk: int = 2048) -> Prefix:
        """Puts a prefix into the cache, for beam(), until forget()."""
        self._sizes("keep", [tokens], 1, chunk)
        n = -(-len(tokens) // self.page)
        self._room("keep", n)
        mine = [self.free.pop() for _ in range(n)]
        try:
            self._prefill([list(tokens)], self._ints([mine]), 0, chunk)
        except BaseException:
            self.free.extend(reversed(mine))
            raise
        self.kept.append(Prefix(mine, len(tokens)))
        return self.kept[-1]

    def forget(self, prefix: Prefix):
        """Gives a kept prefix's pages back."""
        if not any(p is prefix for p in self.kept):
            raise AssertionError("forget: the prefix is not kept here")
        self.kept = [p for p in self.kept if p is not prefix]
        self.free.extend(reversed(prefix.pages))

    def resize(self, pages: int):
        """Makes the caches hold `pages` pages, at least those that kept prefixes have; their pages move to the front first.
        Where memory runs out on the way, a larger pool stays as it was, and a smaller one has its `pages` pages but still the memory
        of the layers that were not reached, which another call gives back."""
        held, now = [i for p in self.kept for i in p.pages], self.caches[0][0].shape[0]
        if pages < max(1, len(held)):
            raise AssertionError(f"resize: {pages} pages, of which {len(held)} are in use")
        if pages < now and held:
            refs = torch.zeros(now, dtype=torch.int32)
            refs[held] = 1
            # one row holds them all: a page is named once
            table, _ = pool.compact(self.caches, self._ints([held]), refs.to(self.dev))
            held = table[0].tolist()
            moved = iter(held)
            for p in self.kept:
                p.pages = [next(moved) for _ in p.pages]
        # A layer at a time: the old and the new cache of one layer alone exist together. What is free and how many pages the layers
        # have are in step before memory is asked for, and after it is refused
        if pages <= now:
            self.caches = [tuple(x[:pages] for x in c) for c in self.caches]
            self._free_all_but(held, pages)
        try:
            for i in range(len(self.caches)):
                self.caches[i] = tuple(torch.cat([x, x.new_zeros((pages - now, *x.shape[1:]))]) if pages > now else x.clone()
                                       for x in self.caches[i])
        except BaseException:
            self.caches = [tuple(x[:now] for x in c) for c in self.caches]
            raise
        self._free_all_but(held, pages)

    def _free_all_but(self, held, pages: int):
        held = set(held)
        self.free = [i for i in range(pages) if i not in held]
