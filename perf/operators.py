"""Serving operators over a paged KV cache, as cases that can be measured: attention of a chunk
of new tokens over the cache, the fused QKV split + RoPE + write into the cache's pages, and
the processing of a step's logits (penalties for repeated tokens, a bias, a grammar mask).

``run`` computes a case in plain torch operations, or, where ``own`` is true, through this
repository's entry points (``bd3attn.ops.paged_attn_raw``, ``bd3attn.ops.qkv_rope_paged_raw``,
``bd3attn.logits.process_logits``) on the same inputs. ``exact`` is the same in 64 bits.

The cache: ``k_pages`` and ``v_pages`` are (pages, kv heads, page size, 64); row p of sequence b
sits in page ``page_table[b, p // page_size]`` at row ``p % page_size``. The new tokens of all
sequences are packed one after the other: sequence b's are rows cu_q[b] .. cu_q[b + 1], and they
are the last of its kv_lens[b] positions. A token in block i (position // block_size) sees every
position in blocks up to i; block_size 1 is causal attention.
"""

import math
import os
import random
import sys

import torch

own = False

HEAD_DIM = 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- the cases --------------------------------------------------------------------------------

def listed():
    return [
        # one sequence, one block of a denoising step over a short cache: the smallest call, all latency
        attend("attend, one block", 1, 12, 12, (16, 16), (1040, 1040), 16, 16, "bf16"),
        # a batch in the middle of generation: a 16-token block each, caches from 1K to 16K
        attend("attend, blocks of a batch", 32, 12, 12, (16, 16), (1024, 16384), 64, 16, "bf16"),
        # one token each and grouped heads, lengths from 1 up; the LSE goes on to a merge
        attend("attend, single tokens", 64, 32, 8, (1, 1), (1, 8192), 16, 1, "f16", lse=True),
        # a chunk of a long prompt after 8K committed tokens (chunked prefill)
        attend("attend, prompt chunk", 1, 12, 12, (2048, 2048), (8192, 8192), 64, 16, "bf16", lse=True),
        # whole prompts of uneven lengths, nothing cached before them
        attend("attend, whole prompts", 4, 12, 12, (1500, 4096), (0, 0), 128, 16, "bf16"),
        # chunks, blocks and single tokens in one call, pages that do not divide a tile, a sequence with no tokens
        attend("attend, mixed batch", 13, 16, 4, (0, 1000), (0, 6000), 48, 4, "bf16", lens=24),
        # four blocks over 64K-token caches: few rows, a long axis
        attend("attend, long cache", 2, 12, 12, (64, 64), (65536, 65536), 256, 16, "bf16"),
        # one layer's new K and V of a denoising step
        write("write, blocks of a batch", 64, 12, 12, (16, 16), (0, 4096), 64, "bf16"),
        # one layer's K and V of a prompt chunk, grouped heads, uneven lengths
        write("write, prompt chunks", 5, 32, 8, (700, 3000), (0, 3000), 16, "f16"),
        # one sequence's next token: latency
        logits("logits, one row", 1, 1, 50258, "bf16", (300, 300), bias="", allowed=""),
        # a denoising step of a batch: 16 rows share a sequence's history, bias and grammar mask
        logits("logits, blocks of a batch", 64, 16, 50258, "bf16", (64, 1024), bias="vocab", allowed="sequence"),
        # single tokens, fp32 logits of an odd vocabulary, long histories, a mask for each row
        logits("logits, single tokens", 96, 1, 128001, "f32", (1, 16384), bias="sequence", allowed="row"),
    ]


def attend(name, batch, heads, kv_heads, new, past, page, block, dtype, lse=False, lens=7):
    return dict(name=name, op="attend", batch=batch, heads=heads, kv_heads=kv_heads, new_lo=new[0],
                new_hi=new[1], past_lo=past[0], past_hi=past[1], page=page, block=block,
                dtype=dtype, lse=lse, lens=lens)


def write(name, batch, heads, kv_heads, new, past, page, dtype, lens=7):
    return dict(name=name, op="write", batch=batch, heads=heads, kv_heads=kv_heads, new_lo=new[0],
                new_hi=new[1], past_lo=past[0], past_hi=past[1], page=page, dtype=dtype, lens=lens)


def logits(name, batch, rows, vocab, dtype, history, bias, allowed, lens=7):
    return dict(name=name, op="logits", batch=batch, rows=rows, vocab=vocab, dtype=dtype,
                hist_lo=history[0], hist_hi=history[1], bias=bias, allowed=allowed, lens=lens)


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm (from 0: over that of one more)."""
    if lo >= hi:
        return lo
    more = int(lo == 0)
    return min(hi, int(math.exp(rng.uniform(math.log(lo + more), math.log(hi + 1 + more)))) - more)


def draw(rng):
    op = rng.choice(("attend", "attend", "write", "logits"))
    lens = rng.randrange(1 << 20)
    if op == "logits":
        while True:
            c = logits("", _log_int(rng, 1, 128), rng.choice((1, 1, 4, 16, 32)), _log_int(rng, 1000, 160000),
                       rng.choice(("bf16", "f16", "f32")), (rng.choice((0, 1)), _log_int(rng, 16, 16384)),
                       rng.choice(("", "vocab", "sequence")), rng.choice(("", "sequence", "row")), lens)
            if work(c)["bytes"] <= 240e6:
                break
    else:
        kv_heads = rng.choice((1, 2, 4, 8, 12))
        heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 8))
        while True:
            batch, page = _log_int(rng, 1, 64), rng.choice((8, 16, 32, 48, 64, 128, 256))
            dtype = rng.choice(("bf16", "f16"))
            hi = _log_int(rng, 1, 4096)
            new = (rng.choice((hi, hi, 0, 1)), hi)
            if op == "write":
                c = write("", batch, heads, kv_heads, new, (0, _log_int(rng, 1, 4096)), page, dtype, lens)
                if 0 < work(c)["flops"] and work(c)["bytes"] <= 4.2e8:
                    break
            else:
                past = _log_int(rng, 1, 65536)
                c = attend("", batch, heads, kv_heads, new, (rng.choice((0, past)), past), page,
                           rng.choice((1, 4, 16, 64)), dtype, rng.choice((True, False)), lens)
                w = work(c)
                pairs = batch * heads * hi * (hi + past)  # of the plain form's padded scores
                if w["bytes"] <= 4.2e8 and 0 < w["flops"] <= 5.8e10 and pairs <= 8e8 and batch * kv_heads * (hi + past) <= 1.4e7:
                    break
    del c["name"]
    return c


def _lengths(case):
    """[(new tokens, all tokens)] of the sequences: the case's own, in every run of it."""
    rng = random.Random(case["lens"])
    got = []
    for _ in range(case["batch"]):
        n = _log_int(rng, case["new_lo"], case["new_hi"])
        got.append((n, n + _log_int(rng, case["past_lo"], case["past_hi"])))
    return got


def _histories(case):
    rng = random.Random(case["lens"])
    return [_log_int(rng, case["hist_lo"], case["hist_hi"]) for _ in range(case["batch"])]


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "logits":
        rows, words = case["batch"] * case["rows"], -(-case["vocab"] // 32)
        b = 2 * rows * case["vocab"] * size + 8 * sum(_histories(case)) + 16 * case["batch"]
        b += {"": 0, "vocab": 4, "sequence": 4 * case["batch"]}[case["bias"]] * case["vocab"]
        b += {"": 0, "sequence": 4 * case["batch"], "row": 4 * rows}[case["allowed"]] * words
        return {"bytes": b, "flops": 4 * rows * case["vocab"]}
    lens, hq, hkv, row = _lengths(case), case["heads"], case["kv_heads"], HEAD_DIM * size
    tokens = sum(n for n, _ in lens)
    if case["op"] == "write":
        # the projection in, q and the new rows of the cache out, a row of both tables a position
        return {"bytes": 2 * tokens * (hq + 2 * hkv) * row + tokens * HEAD_DIM * 4, "flops": 3 * tokens * (hq + hkv) * HEAD_DIM}
    pairs, rows = 0, 0
    for n, kv in lens:
        seen = [min(kv, ((kv - n + i) // case["block"] + 1) * case["block"]) for i in range(n)]
        pairs += sum(seen)
        rows += max(seen, default=0)
    b = 2 * tokens * hq * row + 2 * rows * hkv * row + 4 * sum(-(-kv // case["page"]) for _, kv in lens)
    return {"bytes": b + 4 * tokens * hq * case["lse"], "flops": 4 * HEAD_DIM * hq * pairs}


# ---- what a program has in hand before the call ----------------------------------------------

def _pages(case, seed, g):
    """The cache of the case's sequences (in an order of the seed's) and where their rows sit:
    pages handed out in no order, table entries past a sequence's pages -1."""
    lens = _lengths(case)
    random.Random(seed).shuffle(lens)
    ps, hkv, dt = case["page"], case["kv_heads"], DTYPES[case["dtype"]]
    need = [-(-kv // ps) for _, kv in lens]
    width = max(max(need), 1)
    ids = random.Random(seed + 1).sample(range(sum(need) + 3), sum(need))
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    shape = (sum(need) + 3, hkv, ps, HEAD_DIM)
    cu = [0]
    for n, _ in lens:
        cu.append(cu[-1] + n)
    return {
        "k_pages": torch.randn(shape, generator=g, device="cuda", dtype=dt),
        "v_pages": torch.randn(shape, generator=g, device="cuda", dtype=dt),
        "page_table": torch.tensor(table, dtype=torch.int32, device="cuda"),
        "kv_lens": torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda"),
        "cu_q": torch.tensor(cu, dtype=torch.int32, device="cuda"),
        "max_new": max(n for n, _ in lens), "max_kv": max(kv for _, kv in lens), "tokens": cu[-1],
    }


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "logits":
        B, S, V = case["batch"], case["rows"], case["vocab"]
        lens = _histories(case)
        random.Random(seed).shuffle(lens)
        s["logits"] = (3 * torch.randn(B, S, V, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
        # tokens repeat, as text does: ids crowd at the front of the vocabulary
        u = torch.rand(B, max(max(lens), 1), generator=g, device="cuda")
        s["history"] = (u.pow(3) * V).long().clamp_(max=V - 1)
        s["history_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["repetition"] = 1 + 0.5 * torch.rand(B, generator=g, device="cuda")
        s["presence"] = torch.rand(B, generator=g, device="cuda")
        s["frequency"] = 0.2 * torch.rand(B, generator=g, device="cuda")
        shape = {"": None, "vocab": (V,), "sequence": (B, V)}[case["bias"]]
        s["bias"] = shape and torch.randn(shape, generator=g, device="cuda")
        shape = {"": None, "sequence": (B, -(-V // 32)), "row": (B, S, -(-V // 32))}[case["allowed"]]
        # a grammar's tokens come in runs: words that are all allowed, all forbidden or mixed
        s["allowed"] = None
        if shape:
            bits = torch.randint(-2 ** 31, 2 ** 31, shape, generator=g, device="cuda")
            kind = torch.randint(0, 4, shape, generator=g, device="cuda")
            s["allowed"] = torch.where(kind == 0, bits, torch.where(kind == 1, -1, 0)).int()
            s["allowed"][..., 0] |= 2  # a token is always left
        return s
    s.update(_pages(case, seed, g))
    dt, hq, hkv = DTYPES[case["dtype"]], case["heads"], case["kv_heads"]
    if case["op"] == "attend":
        s["q"] = torch.randn(s["tokens"], hq, HEAD_DIM, generator=g, device="cuda", dtype=dt)
        return s
    s["qkv"] = torch.randn(s["tokens"], (hq + 2 * hkv) * HEAD_DIM, generator=g, device="cuda", dtype=dt)
    inv = 10000.0 ** (-torch.arange(0, HEAD_DIM, 2, dtype=torch.float64, device="cuda") / HEAD_DIM)
    angle = torch.arange(case["new_hi"] + case["past_hi"], dtype=torch.float64, device="cuda")[:, None] * inv
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# ---- one pass ---------------------------------------------------------------------------------

_entry = {}


def _library():
    if not _entry:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "diffusion-llm_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        from bd3attn import ops
        from bd3attn.logits import process_logits
        _entry.update(ops=ops, process_logits=process_logits)
    return _entry


def run(s):
    op = s["case"]["op"]
    if own:
        return {"attend": _own_attend, "write": _own_write, "logits": _own_logits}[op](s)
    return {"attend": _plain_attend, "write": _plain_write, "logits": _plain_logits}[op](s)


def _own_attend(s):
    ops, c = _library()["ops"], s["case"]
    if "workspace" not in s:  # a program keeps one beside its cache
        s["workspace"] = ops.paged_workspace(s["q"].device)
    return ops.paged_attn_raw(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_lens"], s["cu_q"],
                              s["max_new"], c["block"], return_lse=c["lse"], workspace=s["workspace"])


def _own_write(s):
    c = s["case"]
    q = _library()["ops"].qkv_rope_paged_raw(s["qkv"], c["heads"], c["kv_heads"], s["cos"], s["sin"], s["k_pages"],
                                             s["v_pages"], s["page_table"], s["kv_lens"], s["cu_q"])
    return q, s["k_pages"], s["v_pages"]


def _own_logits(s):
    return _library()["process_logits"](
        s["logits"], history=s["history"], history_len=s["history_len"], repetition=s["repetition"],
        presence=s["presence"], frequency=s["frequency"], bias=s["bias"], allowed=s["allowed"])


def _plain_attend(s):
    """Every sequence padded to the longest: its pages gathered, scores in 32 bits, softmax by hand."""
    c, q = s["case"], s["q"]
    hq, hkv, ps, n, m = c["heads"], c["kv_heads"], c["page"], max(s["max_new"], 1), max(s["max_kv"], 1)
    B, g, dev = c["batch"], hq // hkv, q.device
    pos = torch.arange(m, device=dev)
    page = s["page_table"].long().clamp(min=0)[:, pos // ps]                       # (B, m)
    k = s["k_pages"][page, :, pos % ps].float()                                    # (B, m, hkv, 64)
    v = s["v_pages"][page, :, pos % ps].float()
    start, kv = s["cu_q"][:-1].long(), s["kv_lens"].long()
    new = s["cu_q"].long().diff()
    row = torch.arange(n, device=dev)
    if not s["tokens"]:
        o, lse = q.clone(), q.new_zeros(q.shape[:2], dtype=torch.float32)
        return (o, lse) if c["lse"] else o
    at = (start[:, None] + row).clamp(max=s["tokens"] - 1)                         # (B, n)
    qp = q[at].float().view(B, n, hkv, g, HEAD_DIM).permute(0, 2, 3, 1, 4).reshape(B, hkv, g * n, HEAD_DIM)
    x = torch.matmul(qp, k.permute(0, 2, 3, 1)).mul_(HEAD_DIM ** -0.5)             # (B, hkv, g n, m)
    x = x.view(B, hkv, g, n, m)
    qpos = kv[:, None] - new[:, None] + row                                        # (B, n)
    sees = (pos // c["block"] <= (qpos // c["block"])[..., None]) & (pos < kv[:, None, None]) & (qpos >= 0)[..., None]
    x.masked_fill_(~sees[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hkv, g * n, m), v.permute(0, 2, 1, 3)).view(B, hkv, g, n, HEAD_DIM)
    o = torch.where(total > 0, o / total, 0.0)
    lse = torch.where(total > 0, top + total.log(), -math.inf)[..., 0]
    live = row < new[:, None]                                                      # (B, n): b-major, as the packed rows are
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, hq, HEAD_DIM)[live].to(q.dtype)
    lse = lse.permute(0, 3, 1, 2).reshape(B, n, hq)[live]
    return (o, lse) if c["lse"] else o


def _places(s):
    """Of each packed token: its position, and the page and row that it is kept in."""
    t = torch.arange(s["tokens"], device=s["cu_q"].device)
    cu, ps = s["cu_q"].long(), s["case"]["page"]
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    pos = s["kv_lens"].long()[b] - cu[b + 1] + t
    return pos, s["page_table"].long()[b, pos // ps], pos % ps


def _plain_write(s):
    c, x = s["case"], s["qkv"]
    hq, hkv = c["heads"], c["kv_heads"]
    pos, page, row = _places(s)
    y = x.float().view(-1, hq + 2 * hkv, HEAD_DIM)
    co, si = s["cos"][pos][:, None], s["sin"][pos][:, None]
    a, b = y[:, :hq + hkv, :HEAD_DIM // 2], y[:, :hq + hkv, HEAD_DIM // 2:]
    r = torch.cat([a * co - b * si, a * si + b * co], -1).to(x.dtype)
    s["k_pages"][page, :, row] = r[:, hq:]
    s["v_pages"][page, :, row] = y[:, hq + hkv:].to(x.dtype)
    return r[:, :hq].contiguous(), s["k_pages"], s["v_pages"]


def _plain_logits(s):
    """x > 0 ? x / r : x * r for tokens of the history, then - (frequency count + presence),
    then + bias; tokens that the mask forbids become -inf."""
    x, V = s["logits"].float(), s["logits"].shape[-1]
    live = torch.arange(s["history"].shape[1], device=x.device) < s["history_len"][:, None]
    count = torch.zeros(x.shape[0], V, device=x.device).scatter_add_(1, s["history"], live.float())[:, None]
    r, f, p = (s[k][:, None, None] for k in ("repetition", "frequency", "presence"))
    x = torch.where(count > 0, torch.where(x > 0, x / r, x * r) - (f * count + p), x)
    if s["bias"] is not None:
        x = x + (s["bias"] if s["bias"].dim() == 1 else s["bias"][:, None])
    if s["allowed"] is not None:
        bits = (s["allowed"][..., None] >> torch.arange(32, device=x.device)) & 1
        ok = bits.flatten(-2)[..., :V].bool()
        x = x.masked_fill(~(ok if ok.dim() == 3 else ok[:, None]), -math.inf)
    return x.to(s["logits"].dtype)


# ---- the definitions in 64 bits, one sequence at a time ---------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        rows = []
        for b in range(case["batch"]):
            x = s["logits"][b].double()
            n = torch.bincount(s["history"][b, :int(s["history_len"][b])], minlength=case["vocab"]).double()
            r, f, p = (float(s[k][b]) for k in ("repetition", "frequency", "presence"))
            hit = torch.minimum(x * r, x / r) - f * n - p  # r >= 1: the smaller of the two
            x = torch.where(n > 0, hit, x)
            if case["bias"]:
                x = x + (s["bias"] if case["bias"] == "vocab" else s["bias"][b]).double()
            if case["allowed"]:
                at = torch.arange(case["vocab"], device=x.device)
                word = s["allowed"][b][..., at // 32].long()
                x[(word >> (at % 32) & 1).expand_as(x) == 0] = -math.inf
            rows.append(x)
        return torch.stack(rows)
    cu, kv, ps = s["cu_q"].tolist(), s["kv_lens"].tolist(), case["page"]
    hq, hkv = case["heads"], case["kv_heads"]
    if case["op"] == "write":
        q = torch.zeros(s["tokens"], hq, HEAD_DIM, dtype=torch.float64, device="cuda")
        k, v = s["k_pages"].double(), s["v_pages"].double()
        for b in range(case["batch"]):
            x = s["qkv"][cu[b]:cu[b + 1]].double().unflatten(1, (hq + 2 * hkv, HEAD_DIM))
            pos = torch.arange(kv[b] - len(x), kv[b], device="cuda")
            z = torch.view_as_complex(x[:, :hq + hkv].unflatten(2, (2, HEAD_DIM // 2)).transpose(2, 3).contiguous())
            z = z * torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
            z = torch.cat([z.real, z.imag], -1)
            q[cu[b]:cu[b + 1]] = z[:, :hq]
            page = s["page_table"][b].long()[pos // ps]
            k[page, :, pos % ps], v[page, :, pos % ps] = z[:, hq:], x[:, hq + hkv:]
        return q, k, v
    o = torch.zeros(s["tokens"], hq, HEAD_DIM, dtype=torch.float64, device="cuda")
    lse = torch.full((s["tokens"], hq), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        n, m = cu[b + 1] - cu[b], kv[b]
        pages = s["page_table"][b, :-(-m // ps)].long()
        seen = (torch.arange(m - n, m, device="cuda") // case["block"] + 1) * case["block"]
        mask = torch.arange(m, device="cuda") >= seen[:, None]
        for h in range(hq if n else 0):
            k, v = (s[t][pages, h * hkv // hq].reshape(-1, HEAD_DIM)[:m].double() for t in ("k_pages", "v_pages"))
            x = (s["q"][cu[b]:cu[b + 1], h].double() @ k.T / math.sqrt(HEAD_DIM)).masked_fill_(mask, -math.inf)
            lse[cu[b]:cu[b + 1], h] = torch.logsumexp(x, -1)
            o[cu[b]:cu[b + 1], h] = torch.softmax(x, -1) @ v
    return (o, lse) if case["lse"] else o
