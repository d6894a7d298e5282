"""The serving operators over a paged KV cache in float64, one sequence at a time, from their
definitions: attention of packed new tokens, the QKV split with rotary positions and the page
write, and the processing of logits."""

from __future__ import annotations

import math

import torch


def rows_of(pages: torch.Tensor, table_row: torch.Tensor, n: int) -> torch.Tensor:
    """Positions 0 .. n-1 of one sequence's cache (heads, n, D): page table_row[p // size], row
    p % size. Table entries past the last position are not looked at."""
    size = pages.shape[2]
    ids = table_row[:-(-n // size)].long()
    return pages[ids].transpose(0, 1).flatten(1, 2)[:, :n]


def paged_attention(q, k_pages, v_pages, page_table, kv_lens, cu_q, block_size, scale=None):
    """(O, LSE, sum_c p_c |V_c|) in float64 of the packed rows q (tokens, q heads, D): token t of a
    sequence with n new tokens and m positions sits at position m - n + t and sees
    [0, min((position // block_size + 1) * block_size, m)); O = 0 and LSE = -inf where that is
    empty. The third result bounds the effect of rounding the probabilities."""
    T, Hq, D = q.shape
    G = Hq // k_pages.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    o = torch.zeros(T, Hq, D, dtype=torch.float64)
    mag = torch.zeros_like(o)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    for b in range(len(kv_lens)):
        a, e, m = int(cu_q[b]), int(cu_q[b + 1]), int(kv_lens[b])
        if e == a or m == 0:
            continue
        k = rows_of(k_pages, page_table[b], m).double()
        v = rows_of(v_pages, page_table[b], m).double()
        pos = torch.arange(m - (e - a), m)
        hi = ((pos.div(block_size, rounding_mode="floor") + 1) * block_size).clamp(max=m)
        hi[pos < 0] = 0
        hidden = torch.arange(m) >= hi[:, None]
        seen = hi > 0
        for h in range(Hq):
            x = (q[a:e, h].double() @ k[h // G].T * scale).masked_fill(hidden, -math.inf)
            p = torch.softmax(x[seen], -1)
            o[a:e, h][seen] = p @ v[h // G]
            mag[a:e, h][seen] = p @ v[h // G].abs()
            lse[a:e, h][seen] = torch.logsumexp(x[seen], -1)
    return o, lse, mag


def rope_write(qkv, n_heads, n_kv_heads, cos, sin, k_pages, v_pages, page_table, kv_lens, cu_q):
    """(q, k_pages, v_pages) in float64 after the write: q and k rotated by each token's position
    (pairs (x_i, x_{i + D/2}) by the angle whose cosine and sine the tables hold)."""
    size = k_pages.shape[2]
    x = qkv.double().unflatten(1, (n_heads + 2 * n_kv_heads, -1))
    D = x.shape[-1]
    q = torch.zeros(len(qkv), n_heads, D, dtype=torch.float64)
    kp, vp = k_pages.double(), v_pages.double()
    for b in range(len(kv_lens)):
        a, e, m = int(cu_q[b]), int(cu_q[b + 1]), int(kv_lens[b])
        for t in range(a, e):
            pos = m - (e - t)
            c, s = cos[pos].double(), sin[pos].double()
            x1, x2 = x[t, :, :D // 2], x[t, :, D // 2:]
            r = torch.cat([x1 * c - x2 * s, x1 * s + x2 * c], -1)
            q[t] = r[:n_heads]
            page, row = int(page_table[b, pos // size]), pos % size
            kp[page, :, row] = r[n_heads:n_heads + n_kv_heads]
            vp[page, :, row] = x[t, n_heads + n_kv_heads:]
    return q, kp, vp


def process_logits(logits, history=None, history_len=None, repetition=None, presence=None,
                   frequency=None, bias=None, allowed=None):
    """Processed logits in float64; ``allowed`` is a boolean mask (batch, vocab) or
    (batch, seq, vocab) here."""
    B, S, V = logits.shape
    x = logits.double().clone()
    for b in range(B):
        n = torch.zeros(V, dtype=torch.float64)
        if history is not None:
            for v in history[b, :int(history_len[b])].tolist():
                if 0 <= v < V:
                    n[v] += 1
        r = 1.0 if repetition is None else float(repetition[b])
        f = 0.0 if frequency is None else float(frequency[b])
        p = 0.0 if presence is None else float(presence[b])
        y = torch.where(x[b] > 0, x[b] / r, x[b] * r) - (f * n + p)
        x[b] = torch.where(n > 0, y, x[b])
    if bias is not None:
        x = x + (bias.double() if bias.dim() == 1 else bias.double()[:, None])
    if allowed is not None:
        x = x.masked_fill(~(allowed if allowed.dim() == 3 else allowed[:, None]), -math.inf)
    return x
