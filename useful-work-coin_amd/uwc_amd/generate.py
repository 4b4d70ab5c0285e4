"""Greedy generation for several prompts at once over the paged 8-bit cache (uwc_amd.kv): a Hugging
Face Qwen3 or Llama CausalLM in bfloat16 or float16, its linears plain or replaced by
uwc_amd.model.convert_qwen3 (integer or mined), without the cache and attention of transformers. The
reference's counterpart is DetQwen3.generate_greedy (runtime/detrt/qwen3.py:296-334): one sequence, whole
fp32 rows.

    gen = PagedGenerator(model, pages=4096)
    tokens = gen.generate([prompt_a, prompt_b], steps=64)

Prompts run packed, in chunks of at most `chunk` tokens each; then every step is one token of every
sequence. The tokens of a step stay on the GPU and feed the next one, so nothing is copied to the host
before the end.
"""
from __future__ import annotations

import torch

from . import kv


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

    @torch.no_grad()
    def generate(self, prompts, steps: int, chunk: int = 2048) -> list[list[int]]:
        """`steps` >= 1 greedy tokens after each of the prompts (lists of at least one token id)."""
        B, sizes = len(prompts), [len(p) for p in prompts]
        if not B or min(sizes) < 1 or steps < 1 or chunk < 1:
            raise AssertionError("generate: prompts of at least one token, steps and chunk of at least one")
        if max(sizes) + steps - 1 > self.positions:
            raise AssertionError(f"generate: {max(sizes)} + {steps} tokens exceed {self.positions} positions")
        held = [-(-(n + steps - 1) // self.page) for n in sizes]
        if sum(held) > len(self.free):
            raise AssertionError(f"generate: {sum(held)} pages are needed, {len(self.free)} are free")
        mine = [[self.free.pop() for _ in range(n)] for n in held]
        try:
            table = self._ints([p + [-1] * (max(held) - len(p)) for p in mine])
            last = torch.empty((B, self.model.config.hidden_size), dtype=self.dtype, device=self.dev)
            for at in range(0, max(sizes), chunk):
                done = [min(n, at) for n in sizes]
                new = [min(n - d, chunk) for n, d in zip(sizes, done)]
                cu = [0]
                for n in new:
                    cu.append(cu[-1] + n)
                ids = torch.tensor([t for p, d, n in zip(prompts, done, new) for t in p[d:d + n]], device=self.dev)
                h = self.forward(ids, table, self._ints(done), self._ints([d + n for d, n in zip(done, new)]), self._ints(cu),
                                 max(new), max(d + n for d, n in zip(done, new)))
                ends = [b for b in range(B) if new[b] and done[b] + new[b] == sizes[b]]
                last[ends] = h[[cu[b + 1] - 1 for b in ends]]
            out = [self.model.lm_head(last).argmax(-1)]
            ctx = self._ints(sizes)
            for i in range(steps - 1):
                h = self.forward(out[-1], table, ctx, ctx + 1, None, 1, max(sizes) + i + 1)
                out.append(self.model.lm_head(h).argmax(-1))
                ctx = ctx + 1
            return torch.stack(out, 1).tolist()
        finally:
            for p in mine:
                self.free.extend(reversed(p))
