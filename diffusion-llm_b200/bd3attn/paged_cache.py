"""A paged KV cache for a batch of sequences of different lengths, with the fused QKV + RoPE +
page write and the attention over it.

``KVCache`` (``kv_cache.py``) holds one batch whose sequences grow together; here every layer's
keys and values live in pages of ``page_size`` positions that sequences take from one pool as
they grow and give back when they end, so prompts of any lengths, blocks under denoising and
single tokens share a call:

    cache = PagedKVCache(n_layers, n_kv_heads, num_pages, max_seqs=64, max_len=4096)
    a, b = cache.add(), cache.add()              # two sequences
    cache.begin({a: 500, b: 16})                 # 500 and 16 new tokens, packed a's first
    for layer in range(n_layers):
        q = cache.rope_qkv(layer, qkv, n_heads, cos, sin)    # writes k and v, returns q
        o = cache.attend(layer, q, block_size)
    cache.commit()                               # the new tokens stay

Until ``commit`` the new positions are provisional: the next ``rope_qkv`` of the same ``begin``
writes them again (a denoising step that repeats the block with other tokens), and another
``begin`` starts from the committed lengths. ``begin`` is the only place where the host tells
the device anything (page table, lengths, offsets); the layers' calls read them there, so one
step can be captured in a CUDA graph and replayed for as long as the numbers of new tokens stay
the same. Between ``commit`` and the next ``begin`` there is no step, and the layers' calls raise.
"""

from __future__ import annotations

import torch

from bd3attn import ops


class PagedKVCache:
    """Pages of post-RoPE keys/values of all layers, and which sequence holds which.

    Args:
        n_layers, n_kv_heads, head_dim: the model's (head_dim 64 for ``attend``).
        num_pages: pages of the pool (each holds page_size positions of every layer).
        max_seqs: sequences at a time; max_len: positions of one sequence at most.
        page_size: positions per page, a multiple of 8.
        dtype: bf16 or f16 (rope_qkv also takes fp32, attend does not).
    """

    def __init__(self, n_layers: int, n_kv_heads: int, num_pages: int, max_seqs: int, max_len: int,
                 page_size: int = 64, head_dim: int = 64, dtype=torch.bfloat16, device="cuda"):
        if min(n_layers, n_kv_heads, num_pages, max_seqs, max_len) < 1:
            raise ValueError("sizes must be >= 1")
        if page_size < 8 or page_size % 8:
            raise ValueError("page_size must be a multiple of 8")
        self.page_size, self.max_len, self.max_seqs = page_size, max_len, max_seqs
        shape = (num_pages, n_kv_heads, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.n_kv_heads = n_kv_heads
        width = -(-max_len // page_size)
        # the device's view of the sequences of the current begin(), in its order
        self.page_table = torch.zeros((max_seqs, width), dtype=torch.int32, device=device)
        self.kv_lens = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.cu_q = torch.zeros(max_seqs + 1, dtype=torch.int32, device=device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}   # sequence -> its pages
        self._len: dict[int, int] = {}           # sequence -> committed positions
        self._next = 0
        self._new: dict[int, int] = {}           # the current begin()
        self._open = False                       # between begin() and commit()
        self.max_new = self.tokens = 0
        # of attend; made here, since a zeroing that a graph capture records runs only at its replays
        self._workspace = ops.paged_workspace(self.page_table.device) if self.page_table.is_cuda else None

    def add(self) -> int:
        """A new, empty sequence; returns its handle."""
        if len(self._len) == self.max_seqs:
            raise RuntimeError(f"the cache holds {self.max_seqs} sequences already")
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._len[seq] = [], 0
        return seq

    def release(self, seq: int) -> None:
        """End a sequence: its pages go back to the pool. In the middle of a step the packed rows
        stay as they are (the pages serve others from the next begin() on) and the other
        sequences commit theirs."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._len[seq]
        self._new.pop(seq, None)

    def length(self, seq: int) -> int:
        """Committed positions of a sequence."""
        return self._len[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def begin(self, new: dict[int, int]) -> None:
        """Give the sequences of ``new`` that many new positions after their committed ones (pages
        taken as needed) and pack their tokens in the dict's order. RuntimeError, with nothing
        changed, if the pool or a sequence's max_len does not suffice."""
        need = 0
        for seq, n in new.items():
            if n < 0:
                raise ValueError("a sequence's new tokens must be >= 0")
            total = self._len[seq] + n
            if total > self.max_len:
                raise RuntimeError(f"sequence {seq}: {total} positions, max_len is {self.max_len}")
            need += max(0, -(-total // self.page_size) - len(self._pages[seq]))
        if need > len(self._free):
            raise RuntimeError(f"{need} pages needed, {len(self._free)} free")
        rows, cu, lens = [], [0], []
        width = self.page_table.shape[1]
        for seq, n in new.items():
            pages, total = self._pages[seq], self._len[seq] + n
            while len(pages) * self.page_size < total:
                pages.append(self._free.pop())
            rows.append(pages + [0] * (width - len(pages)))
            cu.append(cu[-1] + n)
            lens.append(total)
        self._new, self._open = dict(new), True
        self.max_new, self.tokens = max(new.values(), default=0), cu[-1]
        # sequences past the last one have no tokens and no positions
        spare = self.max_seqs - len(new)
        cu += [cu[-1]] * spare
        lens += [0] * spare
        if rows:
            self.page_table[:len(rows)].copy_(torch.tensor(rows, dtype=torch.int32))
        self.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        self.cu_q.copy_(torch.tensor(cu, dtype=torch.int32))

    def commit(self) -> None:
        """The new positions of the last begin() stay."""
        for seq, n in self._new.items():
            self._len[seq] += n
        self._new, self.max_new, self.tokens, self._open = {}, 0, 0, False

    def _check_step(self, rows: int) -> None:
        """The device holds the last begin()'s lengths and table: of use until its commit() only."""
        if not self._open:
            raise RuntimeError("rope_qkv and attend belong between begin() and commit()")
        if rows < self.tokens:
            raise AssertionError(f"{rows} rows for the step's {self.tokens} new tokens")

    def rope_qkv(self, layer_idx: int, qkv: torch.Tensor, n_heads: int, cos_table: torch.Tensor,
                 sin_table: torch.Tensor, q_out: torch.Tensor | None = None) -> torch.Tensor:
        """Rotated queries (tokens, n_heads, head_dim) of the layer's packed QKV projection
        (tokens, (n_heads + 2 * n_kv_heads) * head_dim); its rotated keys and its values go
        into the layer's pages. RuntimeError outside a step (begin() to commit())."""
        self._check_step(qkv.shape[0])
        return ops.qkv_rope_paged_raw(qkv, n_heads, self.n_kv_heads, cos_table, sin_table,
                                      self.k[layer_idx], self.v[layer_idx], self.page_table,
                                      self.kv_lens, self.cu_q, q_out=q_out)

    def attend(self, layer_idx: int, q: torch.Tensor, block_size: int,
               return_lse: bool = False):
        """Block-causal attention (tokens, n_heads, head_dim) of the new tokens over their
        sequences' committed and new positions. The cache's calls share its workspace: they
        must be ordered, as on one stream. RuntimeError outside a step (begin() to commit())."""
        self._check_step(q.shape[0])
        return ops.paged_attn_raw(q, self.k[layer_idx], self.v[layer_idx], self.page_table,
                                  self.kv_lens, self.cu_q, max(self.max_new, 1), block_size,
                                  return_lse=return_lse, workspace=self._workspace)
