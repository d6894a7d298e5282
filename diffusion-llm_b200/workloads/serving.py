"""Serving with the stand-in backbone: prompts of different lengths generated together over a
paged KV cache.

``PagedGeneration`` prefills the prompts in chunks (block-causal, as the reference encodes
clean tokens, model/bd3lm.py:142-172) and then generates block after block, ``steps`` ancestral
steps each (sample/sampler.py:100-122), all sequences packed into one call per layer:
``PagedKVCache.rope_qkv`` (QKV split, RoPE, page write) and ``PagedKVCache.attend``. Between
the backbone and the fused sampler step, ``process_logits`` penalises tokens the sequence holds
already and applies a bias and a grammar's mask of allowed tokens. A sequence that has its
tokens leaves the batch and its pages serve the others.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from bd3attn.logits import process_logits
from bd3attn.paged_cache import PagedKVCache
from bd3attn.sampler import subs_sample_step
from workloads.backbone import Backbone, rope_tables


class PagedGeneration:
    """Args:
        model: a Backbone (its block size is the generation's).
        max_seqs, max_len, num_pages, page_size: the cache's.
        chunk: prompt tokens of a sequence per prefill call, a multiple of the block size.
        repetition, presence, frequency: penalties of tokens that a sequence holds.
        bias: (vocab,) fp32 or None.
    """

    def __init__(self, model: Backbone, max_seqs: int, max_len: int, num_pages: int,
                 page_size: int = 64, steps: int = 16, chunk: int = 512, repetition: float = 1.0,
                 presence: float = 0.0, frequency: float = 0.0, bias: torch.Tensor | None = None,
                 seed: int = 0):
        if chunk % model.block_size:
            raise ValueError("chunk must be a multiple of the block size")
        self.m, self.bs, self.H, self.steps, self.chunk = (model, model.block_size, model.n_heads,
                                                           steps, chunk)
        dev, dt = model.head.weight.device, model.head.weight.dtype
        d = model.embed.embedding_dim
        self.cache = PagedKVCache(len(model.layers), self.H, num_pages, max_seqs, max_len, page_size,
                                  d // self.H, dt, dev)
        cos, sin = rope_tables(d // self.H, max_len, dev)
        self.cos, self.sin = cos.contiguous(), sin.contiguous()
        self.penalties = [float(x) for x in (repetition, presence, frequency)]
        self.bias, self.max_len = bias, max_len
        self.gen = torch.Generator().manual_seed(seed)

    def forward(self, tokens: torch.Tensor, with_logits: bool = True):
        """The packed new tokens (tokens,) of the cache's current begin() through every layer."""
        x = self.m.embed(tokens)
        for i, layer in enumerate(self.m.layers):
            q = self.cache.rope_qkv(i, layer.qkv(layer.norm1(x)), self.H, self.cos, self.sin)
            x = x + layer.out(self.cache.attend(i, q, self.bs).flatten(1))
            x = x + layer.down(F.gelu(layer.up(layer.norm2(x)), approximate="tanh"))
        return self.m.head(self.m.norm(x)) if with_logits else None

    def prefill(self, prompts: dict[int, torch.Tensor]) -> None:
        """Encode and commit the prompts (sequence -> tokens), a chunk of each per call."""
        at = 0
        while any(len(p) > at for p in prompts.values()):
            part = {s: p[at:at + self.chunk] for s, p in prompts.items() if len(p) > at}
            self.cache.begin({s: len(p) for s, p in part.items()})
            self.forward(torch.cat(list(part.values())), with_logits=False)
            self.cache.commit()
            at += self.chunk

    @torch.no_grad()
    def run(self, prompts: list[torch.Tensor], n_blocks: list[int],
            allowed: torch.Tensor | None = None) -> list[torch.Tensor]:
        """Generate n_blocks[i] blocks after prompts[i] (int64 device tokens, whole blocks).
        allowed: packed words (pack_mask) of the tokens that may be generated, (words,) or one
        row per sequence. Returns each sequence's generated tokens. Whatever ends the run, an error
        among it, the cache has its sequences' pages back."""
        if any(len(p) % self.bs for p in prompts):
            raise ValueError("prompts must be whole blocks")
        seqs: dict[int, int] = {}  # prompt -> its sequence while it has one
        try:
            for i in range(len(prompts)):
                if n_blocks[i] > 0:
                    seqs[i] = self.cache.add()
            return self._generate(prompts, n_blocks, allowed, seqs)
        finally:
            for s in seqs.values():
                self.cache.release(s)

    def _generate(self, prompts, n_blocks, allowed, seqs) -> list[torch.Tensor]:
        dev, bs, mask = self.cos.device, self.bs, self.m.mask_index
        self.prefill({s: prompts[i] for i, s in seqs.items() if len(prompts[i])})
        buf = torch.zeros((len(prompts), self.max_len), dtype=torch.int64, device=dev)
        for i, p in enumerate(prompts):
            buf[i, :len(p)] = p
        done = [0] * len(prompts)
        while live := [i for i in range(len(prompts)) if done[i] < n_blocks[i]]:
            self.cache.begin({seqs[i]: bs for i in live})
            rows = torch.tensor(live, device=dev)
            first = torch.tensor([len(prompts[i]) + done[i] * bs for i in live], device=dev)
            cols = first[:, None] + torch.arange(bs, device=dev)
            block = torch.full((len(live), bs), mask, dtype=torch.int64, device=dev)
            rep, pres, freq = (torch.full((len(live),), x, device=dev) for x in self.penalties)
            words = allowed if allowed is None or allowed.dim() == 2 else \
                allowed.expand(len(prompts), -1)
            words = None if words is None else words[rows].contiguous()
            for k in range(self.steps):
                logits = self.forward(block.flatten()).view(len(live), bs, -1)
                buf[rows[:, None], cols] = block
                process_logits(logits, buf[rows], (first + bs).to(torch.int32), rep, pres, freq,
                               self.bias, words, out=logits)
                subs_sample_step(logits, block, mask, 1 - k / self.steps, 1 - (k + 1) / self.steps,
                                 generator=self.gen, out=block)
            self.forward(block.flatten(), with_logits=False)  # the finished block's K/V
            self.cache.commit()
            buf[rows[:, None], cols] = block
            for i in live:
                done[i] += 1
                if done[i] == n_blocks[i]:
                    self.cache.release(seqs.pop(i))
        return [buf[i, len(p):len(p) + done[i] * bs].clone() for i, p in enumerate(prompts)]
