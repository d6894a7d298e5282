"""Tensor-level wrappers over the C ABI (one call per entry point of include/bd3_attn.h).

Every function takes CUDA tensors, allocates its outputs (and workspace) with the caching
allocator, and enqueues the kernels on the current CUDA stream of the inputs' device.
They are also registered as ``torch.ops.bd3.*`` custom ops with fake (meta) implementations
so that ``torch.compile`` can trace callers without graph breaks.
"""

from __future__ import annotations

import ctypes

import torch

from bd3attn._lib import (BD3_BF16, BD3_F16, BD3_F32, LIB, check, i64_array)

_DTYPE_CODE = {torch.bfloat16: BD3_BF16, torch.float16: BD3_F16, torch.float32: BD3_F32}


def _code(dtype: torch.dtype) -> int:
    if dtype not in _DTYPE_CODE:
        raise TypeError(f"unsupported dtype {dtype}")
    return _DTYPE_CODE[dtype]


def _rows_contig(x: torch.Tensor) -> torch.Tensor:
    """The kernels read rows with TMA: the last dim must be contiguous and the other
    strides 16-byte multiples; other layouts are copied (as the reference's
    _last_stride_1 / .contiguous() do)."""
    if x.stride(-1) != 1 or any((s * x.element_size()) % 16 for s in x.stride()[:-1]) \
            or x.data_ptr() % 16:
        return x.contiguous()
    return x


def _s3(x: torch.Tensor):
    return (x.stride(0), x.stride(1), x.stride(2))


def _stream(x: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(x.device).cuda_stream)


def _ptr(x):
    return ctypes.c_void_p(x.data_ptr()) if x is not None else ctypes.c_void_p(0)


def _check_cuda(*xs):
    for x in xs:
        if not x.is_cuda:
            raise AssertionError("inputs must be on CUDA")


# ---------------------------------------------------------------------------------------
def attn_fwd_raw(q, k, v, block_size: int):
    """(O, LSE) of BD3-LM training attention; q, k, v: (B, H, 2n, 64) bf16/f16."""
    _check_cuda(q, k, v)
    q, k, v = _rows_contig(q), _rows_contig(k), _rows_contig(v)
    B, H, S, D = q.shape
    o = torch.empty((B, H, S, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, S), dtype=torch.float32, device=q.device)
    strides = i64_array(_s3(q) + _s3(k) + _s3(v) + _s3(o))
    with torch.cuda.device(q.device):
        check("bd3_attn_fwd", LIB.bd3_attn_fwd(
            _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), B, H, S // 2, D, strides,
            int(block_size), _code(q.dtype), _stream(q)))
    return o, lse


def attn_bwd_raw(q, k, v, o, lse, do, block_size: int, deterministic: bool = False):
    """(dQ, dK, dV) of BD3-LM training attention. deterministic: dQ's partials are added as
    64-bit fixed-point integers (bd3_attn_bwd_det), so dQ is the same on every run; otherwise
    they are added in fp32 in the order the key tiles finish."""
    _check_cuda(q, k, v, o, lse, do)
    q, k, v, o, do = (_rows_contig(t) for t in (q, k, v, o, do))
    B, H, S, D = q.shape
    dq = torch.empty((B, H, S, D), dtype=q.dtype, device=q.device)
    dk = torch.empty_like(dq)
    dv = torch.empty_like(dq)
    size_fn, fn, name = ((LIB.bd3_attn_bwd_det_workspace_size, LIB.bd3_attn_bwd_det,
                          "bd3_attn_bwd_det") if deterministic else
                         (LIB.bd3_attn_bwd_workspace_size, LIB.bd3_attn_bwd, "bd3_attn_bwd"))
    ws_bytes = size_fn(B, H, S // 2, D)
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=q.device)
    lse = lse.contiguous()
    strides = i64_array(_s3(q) + _s3(k) + _s3(v) + _s3(o) + _s3(do) + _s3(dq) + _s3(dk)
                        + _s3(dv))
    with torch.cuda.device(q.device):
        check(name, fn(
            _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), _ptr(do), _ptr(dq), _ptr(dk),
            _ptr(dv), B, H, S // 2, D, strides, int(block_size), _code(q.dtype), _ptr(ws),
            ws.numel(), _stream(q)))
    return dq, dk, dv


def f32_to_f16_scaled_raw(q, k, v):
    """fp32 q, k, v (B, H, rows, 64) as fp16 at tf32's significand (bd3_f32_to_f16_scaled):
    returns (q * 2^-a, k * 2^a, v * 2^-c in fp16, exps) with exps = (a, c, 2^c) fp32 on the
    device. q may have another row count than k and v."""
    _check_cuda(q, k, v)
    q, k, v = (x if x.stride(-1) == 1 and x.data_ptr() % 16 == 0
               and all(st % 4 == 0 for st in x.stride()[:-1]) else x.contiguous()
               for x in (q, k, v))
    B, H, Sq, D = q.shape
    Skv = k.shape[2]
    if k.shape != v.shape or k.shape[:2] != q.shape[:2] or k.shape[3] != D:
        raise AssertionError("q, k, v must be (B, H, rows, head_dim) with k, v alike")
    q16 = torch.empty((B, H, Sq, D), dtype=torch.float16, device=q.device)
    k16 = torch.empty((B, H, Skv, D), dtype=torch.float16, device=q.device)
    v16 = torch.empty_like(k16)
    exps = torch.empty(3, dtype=torch.float32, device=q.device)
    ws = torch.empty(4, dtype=torch.int32, device=q.device)
    strides = i64_array(_s3(q) + _s3(k) + _s3(v))
    with torch.cuda.device(q.device):
        check("bd3_f32_to_f16_scaled", LIB.bd3_f32_to_f16_scaled(
            _ptr(q), _ptr(k), _ptr(v), strides, B, H, Sq, Skv, D, _ptr(q16), _ptr(k16),
            _ptr(v16), _ptr(exps), _ptr(ws), _stream(q)))
    return q16, k16, v16, exps


@torch.library.custom_op("bd3::f32_to_f16_scaled", mutates_args=())
def f32_to_f16_scaled_op(q: torch.Tensor, k: torch.Tensor,
                         v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor,
                                                   torch.Tensor]:
    return f32_to_f16_scaled_raw(q, k, v)


@f32_to_f16_scaled_op.register_fake
def _(q, k, v):
    return (q.new_empty(tuple(q.shape), dtype=torch.float16),
            k.new_empty(tuple(k.shape), dtype=torch.float16),
            v.new_empty(tuple(v.shape), dtype=torch.float16),
            q.new_empty((3,), dtype=torch.float32))


def decode_plan(B, H, q_len, kv_len, block_size, q_pos0=-1, kv_pos0=0):
    ns = ctypes.c_int64(0)
    wb = ctypes.c_size_t(0)
    check("bd3_decode_plan", LIB.bd3_decode_plan(B, H, q_len, kv_len, block_size, q_pos0,
                                                 kv_pos0, ctypes.byref(ns), ctypes.byref(wb)))
    return ns.value, wb.value


def decode_raw(q, k, v, block_size: int, q_pos0: int = -1, kv_pos0: int = 0,
               out_dtype=None, return_lse: bool = False, n_splits: int | None = None,
               kv_len_dev=None):
    """Block-causal decode attention of the q_len queries over kv_len keys.

    kv_len_dev: an int32 device tensor of one element holding the key count; k and v are then
    the whole cache storage (B, H, capacity, 64), the queries sit at the count's end and
    q_pos0 / kv_pos0 / n_splits are ignored. The launch does not depend on the count, so a
    CUDA graph captured around it replays every step of a growing cache.
    """
    _check_cuda(q, k, v)
    q, k, v = _rows_contig(q), _rows_contig(k), _rows_contig(v)
    B, H, q_len, D = q.shape
    kv_len = k.shape[2]
    out_dtype = q.dtype if out_dtype is None else out_dtype
    if kv_len_dev is not None:
        return _decode_devlen(q, k, v, int(block_size), kv_len_dev, out_dtype, return_lse)
    ns, wb = decode_plan(B, H, q_len, kv_len, int(block_size), q_pos0, kv_pos0)
    if n_splits is not None and q_len <= 64:
        ns = int(n_splits)
        wb = B * H * ns * q_len * 65 * 4 if ns > 1 else 0
    o = torch.empty((B, H, q_len, D), dtype=out_dtype, device=q.device)
    lse = torch.empty((B, H, q_len), dtype=torch.float32, device=q.device) if return_lse else None
    ws = torch.empty(max(wb, 16), dtype=torch.uint8, device=q.device)
    strides = i64_array(_s3(q) + _s3(k) + _s3(v) + _s3(o))
    with torch.cuda.device(q.device):
        check("bd3_decode_attn", LIB.bd3_decode_attn(
            _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), B, H, q_len, kv_len, D, strides,
            int(block_size), int(q_pos0), int(kv_pos0), ns, _code(q.dtype), _code(out_dtype),
            _ptr(ws), wb, _stream(q)))
    return (o, lse) if return_lse else o


def _decode_devlen(q, k, v, block_size, kv_len_dev, out_dtype, return_lse):
    _check_cuda(kv_len_dev)
    if kv_len_dev.dtype != torch.int32 or kv_len_dev.numel() != 1:
        raise AssertionError("kv_len_dev must be a one-element int32 device tensor")
    B, H, q_len, D = q.shape
    capacity = k.shape[2]
    ns, wb = decode_plan(B, H, q_len, capacity, block_size, -1, 0)
    o = torch.empty((B, H, q_len, D), dtype=out_dtype, device=q.device)
    lse = torch.empty((B, H, q_len), dtype=torch.float32, device=q.device) if return_lse else None
    ws = torch.empty(max(wb, 16), dtype=torch.uint8, device=q.device)
    strides = i64_array(_s3(q) + _s3(k) + _s3(v) + _s3(o))
    with torch.cuda.device(q.device):
        check("bd3_decode_attn_devlen", LIB.bd3_decode_attn_devlen(
            _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), B, H, q_len, capacity, D, strides,
            block_size, _ptr(kv_len_dev), ns, _code(q.dtype), _code(out_dtype), _ptr(ws), wb,
            _stream(q)))
    return (o, lse) if return_lse else o


def live_decode_raw(q, k, v, live_idx, live_cnt, kv_block: int, block_size: int,
                    out_dtype=None, return_lse: bool = False, n_splits: int | None = None):
    """Decode over a per-(batch, head) list of live KV blocks.

    live_idx: (B, H, max_live) int32 ascending block indices (entries past live_cnt ignored);
    live_cnt: (B, H) int32.
    n_splits: None takes the planned split count; k >= 1 splits every (batch, head)'s list
    over k CTAs (k > 1 merges their partials with the combine kernel).
    """
    _check_cuda(q, k, v, live_idx, live_cnt)
    q, k, v = _rows_contig(q), _rows_contig(k), _rows_contig(v)
    B, H, q_len, D = q.shape
    kv_len = k.shape[2]
    out_dtype = q.dtype if out_dtype is None else out_dtype
    live_idx = live_idx.to(torch.int32).contiguous()
    live_cnt = live_cnt.to(torch.int32).contiguous()
    max_live = live_idx.shape[-1]
    ns = ctypes.c_int64(0)
    wb = ctypes.c_size_t(0)
    check("bd3_decode_live_plan", LIB.bd3_decode_live_plan(
        B, H, q_len, max_live, int(kv_block), ctypes.byref(ns), ctypes.byref(wb)))
    if n_splits is not None:
        if n_splits < 1:
            raise ValueError("n_splits must be >= 1")
        ns.value = int(n_splits)
        wb.value = B * H * n_splits * q_len * 65 * 4 if n_splits > 1 else 0
    o = torch.empty((B, H, q_len, D), dtype=out_dtype, device=q.device)
    lse = torch.empty((B, H, q_len), dtype=torch.float32, device=q.device) if return_lse else None
    ws = torch.empty(max(wb.value, 16), dtype=torch.uint8, device=q.device)
    strides = i64_array(_s3(q) + _s3(k) + _s3(v) + _s3(o))
    with torch.cuda.device(q.device):
        check("bd3_decode_live_blocks", LIB.bd3_decode_live_blocks(
            _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), _ptr(live_idx), _ptr(live_cnt),
            max_live, max_live, int(kv_block), B, H, q_len, kv_len, D, strides, int(block_size),
            ns.value, _code(q.dtype), _code(out_dtype), _ptr(ws), wb.value, _stream(q)))
    return (o, lse) if return_lse else o


def lse_merge_raw(parts, lses, out_dtype=torch.bfloat16):
    """Merge G partials: parts (G, B, H, rows, 64) fp32, lses (G, B, H, rows) fp32 ->
    (O (B, H, rows, 64) in out_dtype, LSE (B, H, rows) fp32)."""
    _check_cuda(parts, lses)
    parts = parts.contiguous()
    lses = lses.contiguous()
    G, B, H, rows, D = parts.shape
    o = torch.empty((B, H, rows, D), dtype=out_dtype, device=parts.device)
    lse = torch.empty((B, H, rows), dtype=torch.float32, device=parts.device)
    with torch.cuda.device(parts.device):
        check("bd3_lse_merge", LIB.bd3_lse_merge(
            _ptr(parts), _ptr(lses), _ptr(o), _ptr(lse), B, H, G, rows, D, B * H * rows * D,
            rows * D, B * H * rows, rows, i64_array(_s3(o)), _code(out_dtype), _stream(parts)))
    return o, lse


def debug_wait_timeout(limit_ns: int, arrive: bool = False, device=None) -> tuple[int, int]:
    """Run the bounded-wait self-check (bd3_debug_wait_timeout) on the current stream and
    return (1 if the wait gave up else 0, the wait's duration in ns). Synchronises."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    out = torch.zeros(2, dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        check("bd3_debug_wait_timeout", LIB.bd3_debug_wait_timeout(
            int(limit_ns), 1 if arrive else 0, _ptr(out),
            ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)))
    res = out.cpu()
    return int(res[0]), int(res[1])


def debug_wait_site() -> dict | None:
    """Where the first bounded wait that ran out gave up since the last read (block, thread,
    barrier shared-memory address, awaited parity), or None; reading clears it."""
    out = (ctypes.c_uint32 * 4)()
    check("bd3_debug_wait_site", LIB.bd3_debug_wait_site(out))
    if not out[0]:
        return None
    return {"block": out[1], "thread": out[2], "smem_addr": out[3] & 0x7FFFFFFF,
            "parity": out[3] >> 31}


def device_status(clear: bool = True) -> int:
    """Sticky device-side error bits (1: a bounded wait ran out; 2: a kernel rejected its
    launch; 4: a RoPE position was outside the table). Synchronises."""
    return int(LIB.bd3_device_status(1 if clear else 0))


# ---------------------------------------------------------------------------------------
# torch.library registrations (used under torch.compile; eager callers use the raw calls)
@torch.library.custom_op("bd3::attn_fwd", mutates_args=())
def attn_fwd_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                block_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    return attn_fwd_raw(q, k, v, block_size)


@attn_fwd_op.register_fake
def _(q, k, v, block_size):
    B, H, S, D = q.shape
    return q.new_empty((B, H, S, D)), q.new_empty((B, H, S), dtype=torch.float32)


@torch.library.custom_op("bd3::attn_bwd", mutates_args=())
def attn_bwd_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                lse: torch.Tensor, do: torch.Tensor, block_size: int,
                deterministic: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return attn_bwd_raw(q, k, v, o, lse, do, block_size, deterministic)


@attn_bwd_op.register_fake
def _(q, k, v, o, lse, do, block_size, deterministic):
    shape = tuple(q.shape)
    return q.new_empty(shape), q.new_empty(shape), q.new_empty(shape)


@torch.library.custom_op("bd3::decode", mutates_args=())
def decode_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              block_size: int) -> torch.Tensor:
    return decode_raw(q, k, v, block_size)


@decode_op.register_fake
def _(q, k, v, block_size):
    return q.new_empty(tuple(q.shape))


def qkv_rope_cache_raw(qkv, n_heads: int, cos_table, sin_table, k_cache, v_cache, row0: int,
                       positions=None, pos0: int = 0, q_out=None):
    """Split a fused QKV projection, rotate q and k (the reference's RoPE), write k and v to
    rows [row0, row0 + seq) of the caches in place and q to q_out; returns q_out.

    qkv: (B, S, 3 * n_heads * D) with its last dim ordered (three, heads, head_dim);
    cos_table, sin_table: (max_pos, D / 2) fp32 (RoPE's buffers); k_cache, v_cache:
    (B, n_heads, rows, D) in qkv's dtype; positions: (S,) int64 absolute positions on the
    device, or None for pos0, pos0 + 1, ...; q_out: (B, n_heads, S, D) or None to allocate.
    row0 < 0 takes the first cache row from the device value positions[0] (positions
    required), so a captured CUDA graph writes each new block at its own rows.
    """
    _check_cuda(qkv, cos_table, sin_table, k_cache, v_cache)
    if qkv.dim() != 3:
        raise AssertionError("qkv must be (batch, seq, 3 * n_heads * head_dim)")
    B, S, F = qkv.shape
    if F % (3 * n_heads):
        raise AssertionError("qkv's last dim must be 3 * n_heads * head_dim")
    D = F // (3 * n_heads)
    if qkv.stride(-1) != 1:
        qkv = qkv.contiguous()
    if q_out is None:
        q_out = torch.empty((B, n_heads, S, D), dtype=qkv.dtype, device=qkv.device)
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("q_out", q_out)):
        if t.dtype != qkv.dtype or t.stride(-1) != 1 or t.shape[0] != B or t.shape[1] != n_heads \
                or t.shape[-1] != D:
            raise AssertionError(f"{name} must be (B, n_heads, rows, head_dim) in qkv's dtype")
    if k_cache.shape[2] != v_cache.shape[2]:
        raise AssertionError("k_cache and v_cache must have the same rows")
    cos_table = cos_table.float().contiguous()
    sin_table = sin_table.float().contiguous()
    if positions is not None:
        positions = positions.to(device=qkv.device, dtype=torch.int64).contiguous()
        if positions.numel() != S:
            raise AssertionError("positions must have one entry per token")
    strides = i64_array(_s3(q_out) + _s3(k_cache) + _s3(v_cache))
    with torch.cuda.device(qkv.device):
        check("bd3_qkv_rope_cache", LIB.bd3_qkv_rope_cache(
            _ptr(qkv), i64_array((qkv.stride(0), qkv.stride(1))), B, S, n_heads, D,
            _ptr(positions), int(pos0), _ptr(cos_table), _ptr(sin_table), cos_table.shape[0],
            _ptr(q_out), _ptr(k_cache), _ptr(v_cache), strides, int(row0), k_cache.shape[2],
            _code(qkv.dtype), _stream(qkv)))
    return q_out


@torch.library.custom_op("bd3::qkv_rope_cache", mutates_args=("k_cache", "v_cache"))
def qkv_rope_cache_op(qkv: torch.Tensor, n_heads: int, cos_table: torch.Tensor,
                      sin_table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      row0: int, positions: torch.Tensor | None = None) -> torch.Tensor:
    """qkv_rope_cache_raw as a custom op: writes the caches in place, returns q."""
    return qkv_rope_cache_raw(qkv, n_heads, cos_table, sin_table, k_cache, v_cache, row0,
                              positions=positions)


@qkv_rope_cache_op.register_fake
def _(qkv, n_heads, cos_table, sin_table, k_cache, v_cache, row0, positions=None):
    B, S, F = qkv.shape
    return qkv.new_empty((B, n_heads, S, F // (3 * n_heads)))


# ---------------------------------------------------------------------------------------
# Paged KV cache
# These calls are short enough for the host's part to matter: array types are made once, the
# stream is read as a plain handle, and the device context is entered only where it changes
# something.
_I64x9, _I64x11 = ctypes.c_int64 * 9, ctypes.c_int64 * 11


def _check_on(index: int, *xs) -> None:
    """All on the CUDA device of that index (get_device() is -1 on the CPU)."""
    for x in xs:
        if x.get_device() != index:
            raise AssertionError("all tensors must be on the same CUDA device")


def _raw_stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _check_pages(k_pages, v_pages, page_table, kv_lens, cu_q, dtype, n_kv_heads, D):
    ks = k_pages.shape
    if len(ks) != 4 or ks != v_pages.shape or ks[1] != n_kv_heads or ks[3] != D:
        raise AssertionError("k_pages and v_pages must be (pages, kv heads, page size, head_dim)")
    if k_pages.dtype is not dtype or v_pages.dtype is not dtype:
        raise AssertionError("k_pages and v_pages must be in the new tokens' dtype")
    i32 = torch.int32
    if page_table.dtype is not i32 or kv_lens.dtype is not i32 or cu_q.dtype is not i32:
        raise AssertionError("page_table, kv_lens and cu_q must be int32")
    ts, bs, cs = page_table.shape, kv_lens.shape, cu_q.shape
    if len(ts) != 2 or len(bs) != 1 or len(cs) != 1 or ts[0] != bs[0] or cs[0] != bs[0] + 1 \
            or not kv_lens.is_contiguous() or not cu_q.is_contiguous() \
            or (page_table.stride(1) != 1 and ts[1] > 1):
        raise AssertionError("page_table must be (B, pages), kv_lens (B,) and cu_q (B + 1,)")
    kst, vst = k_pages.stride(), v_pages.stride()
    if kst[3] != 1 or vst[3] != 1:
        raise AssertionError("the pages' head_dim must be contiguous")
    return bs[0], ts[1], kst, vst


def paged_workspace(device=None) -> torch.Tensor:
    """A workspace for paged_attn_raw on `device` (bd3_paged_workspace_size bytes, zeroed). Keep
    it and pass it to every call; calls that share one must be ordered (one stream). Not to be
    made under a graph capture: the zeroing would run at the graph's replays."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None \
        else torch.device(device)
    with torch.cuda.device(device):
        n = LIB.bd3_paged_workspace_size()
        if n == 0:
            check("bd3_paged_workspace_size", 3)
        return torch.zeros(n, dtype=torch.uint8, device=device)


def paged_attn_raw(q, k_pages, v_pages, page_table, kv_lens, cu_q, max_q_len: int,
                   block_size: int, scale: float | None = None, out_dtype=None,
                   return_lse: bool = False, workspace=None):
    """Block-causal attention of packed new tokens over a paged KV cache.

    q: (tokens, q heads, 64) bf16/f16, sequence b's rows [cu_q[b], cu_q[b+1]); k_pages, v_pages:
    (pages, kv heads, page size, 64) in q's dtype, any strides, page size a multiple of 8;
    page_table: (B, pages per sequence) int32; kv_lens: (B,) int32 positions of each sequence,
    the new tokens (its last ones) included; cu_q: (B + 1,) int32, rows before its first and past
    its last entry are in no sequence and their output is undefined; max_q_len: the most new
    tokens of a sequence (one with more is cut and sets device status bit 2). Tensors of lengths
    stay on the device: a captured CUDA graph serves other lengths and tables. workspace:
    paged_workspace(), kept by the caller (None: a new zeroed one). Returns O (tokens, q heads,
    64), with the LSE (tokens, q heads) if asked.
    Forward only, as the other decode functions.
    """
    _check_cuda(q)
    dev = q.device
    if torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return paged_attn_raw(q, k_pages, v_pages, page_table, kv_lens, cu_q, max_q_len,
                                  block_size, scale, out_dtype, return_lse, workspace)
    if q.dim() != 3:
        raise AssertionError("q must be (tokens, q heads, head_dim)")
    T, Hq, D = q.shape
    max_q_len = int(max_q_len)
    if max_q_len < 1 and T > 0:
        raise AssertionError("max_q_len must be >= 1 where there are tokens")
    n_pages, Hkv, page_size = k_pages.shape[:3] if k_pages.dim() == 4 else (0, 0, 0)
    B, width, ks, vs = _check_pages(k_pages, v_pages, page_table, kv_lens, cu_q, q.dtype, Hkv, D)
    qs = q.stride()
    if qs[2] != 1 or qs[0] % 8 or qs[1] % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        qs = q.stride()
    code = _code(q.dtype)
    _check_on(dev.index, k_pages, v_pages, page_table, kv_lens, cu_q)
    if out_dtype is None or out_dtype == q.dtype:
        o, out_code = torch.empty_like(q, memory_format=torch.contiguous_format), code
    else:
        o, out_code = torch.empty((T, Hq, D), dtype=out_dtype, device=dev), _code(out_dtype)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
    if workspace is None:
        workspace = paged_workspace(dev)
    elif workspace.device != dev:
        raise AssertionError("the workspace must be on q's device")
    rc = LIB.bd3_paged_attn(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), o.data_ptr(),
        lse.data_ptr() if return_lse else None, page_table.data_ptr(), kv_lens.data_ptr(),
        cu_q.data_ptr(), B, T, max_q_len, Hq, Hkv, D, n_pages, page_size, width,
        _I64x11(qs[0], qs[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], Hq * D, D,
                page_table.stride(0)),
        int(block_size), D ** -0.5 if scale is None else float(scale), code, out_code,
        workspace.data_ptr(), workspace.nbytes, _raw_stream(dev))
    if rc:
        check("bd3_paged_attn", rc)
    return (o, lse) if return_lse else o


def qkv_rope_paged_raw(qkv, n_heads: int, n_kv_heads: int, cos_table, sin_table, k_pages, v_pages,
                       page_table, kv_lens, cu_q, q_out=None):
    """Split a packed QKV projection, rotate q and k by their tokens' positions, write k and v
    into the pages in place and q to q_out; returns q_out (tokens, n_heads, D).

    qkv: (tokens, (n_heads + 2 * n_kv_heads) * D) with q, k, v heads in that order; cos_table,
    sin_table: (max_pos, D / 2) fp32; the rest as paged_attn_raw (kv_lens counts the tokens
    being written). The rotation is fp32, rounded once.
    """
    _check_cuda(qkv)
    dev = qkv.device
    if torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return qkv_rope_paged_raw(qkv, n_heads, n_kv_heads, cos_table, sin_table, k_pages,
                                      v_pages, page_table, kv_lens, cu_q, q_out)
    heads = n_heads + 2 * n_kv_heads
    if qkv.dim() != 2 or qkv.shape[1] % heads:
        raise AssertionError("qkv must be (tokens, (n_heads + 2 * n_kv_heads) * head_dim)")
    T, F = qkv.shape
    D = F // heads
    B, width, ks, vs = _check_pages(k_pages, v_pages, page_table, kv_lens, cu_q, qkv.dtype, n_kv_heads, D)
    if cos_table.dtype != torch.float32 or sin_table.dtype != torch.float32 \
            or cos_table.shape != sin_table.shape or cos_table.shape[1:] != (D // 2,) \
            or not cos_table.is_contiguous() or not sin_table.is_contiguous():
        raise AssertionError("cos_table and sin_table must be contiguous (max_pos, head_dim / 2) fp32")
    if qkv.stride(1) != 1 or qkv.stride(0) * qkv.element_size() % 16 or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    _check_on(dev.index, cos_table, sin_table, k_pages, v_pages, page_table, kv_lens, cu_q)
    if q_out is None:
        q_out = qkv.new_empty((T, n_heads, D))
    elif q_out.shape != (T, n_heads, D) or q_out.dtype != qkv.dtype or q_out.stride(2) != 1 \
            or q_out.device != dev:
        raise AssertionError("q_out must be (tokens, n_heads, head_dim) in qkv's dtype")
    rc = LIB.bd3_qkv_rope_paged(
        qkv.data_ptr(), qkv.stride(0), T, B, n_heads, n_kv_heads, D, cos_table.data_ptr(),
        sin_table.data_ptr(), cos_table.shape[0], q_out.data_ptr(), k_pages.data_ptr(),
        v_pages.data_ptr(), page_table.data_ptr(), kv_lens.data_ptr(), cu_q.data_ptr(),
        k_pages.shape[0], k_pages.shape[2], width,
        _I64x9(q_out.stride(0), q_out.stride(1), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
               page_table.stride(0)),
        _code(qkv.dtype), _raw_stream(dev))
    if rc:
        check("bd3_qkv_rope_paged", rc)
    return q_out


@torch.library.custom_op("bd3::paged_attn", mutates_args=("workspace",))
def paged_attn_op(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                  page_table: torch.Tensor, kv_lens: torch.Tensor, cu_q: torch.Tensor,
                  max_q_len: int, block_size: int, workspace: torch.Tensor) -> torch.Tensor:
    return paged_attn_raw(q, k_pages, v_pages, page_table, kv_lens, cu_q, max_q_len, block_size,
                          workspace=workspace)


@paged_attn_op.register_fake
def _(q, k_pages, v_pages, page_table, kv_lens, cu_q, max_q_len, block_size, workspace):
    return q.new_empty(tuple(q.shape))


@torch.library.custom_op("bd3::qkv_rope_paged", mutates_args=("k_pages", "v_pages"))
def qkv_rope_paged_op(qkv: torch.Tensor, n_heads: int, n_kv_heads: int, cos_table: torch.Tensor,
                      sin_table: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                      page_table: torch.Tensor, kv_lens: torch.Tensor,
                      cu_q: torch.Tensor) -> torch.Tensor:
    """qkv_rope_paged_raw as a custom op: writes the pages in place, returns q."""
    return qkv_rope_paged_raw(qkv, n_heads, n_kv_heads, cos_table, sin_table, k_pages, v_pages,
                              page_table, kv_lens, cu_q)


@qkv_rope_paged_op.register_fake
def _(qkv, n_heads, n_kv_heads, cos_table, sin_table, k_pages, v_pages, page_table, kv_lens,
      cu_q):
    return qkv.new_empty((qkv.shape[0], n_heads, qkv.shape[1] // (n_heads + 2 * n_kv_heads)))


# ---------------------------------------------------------------------------------------
PROFILE_KERNELS = ("attn_fwd", "attn_prefill", "bwd_prep", "bwd_dq_convert", "bwd_fused",
                   "decode", "decode_combine", "qkv_rope_cache", "subs_sample", "paged_attn",
                   "qkv_rope_paged", "process_logits")


def profile_enable(on: bool = True) -> None:
    """Bracket every library launch with CUDA events on its own stream (see
    bd3_profile_enable)."""
    check("bd3_profile_enable", LIB.bd3_profile_enable(1 if on else 0))


def profile_collect() -> dict:
    """{kernel name: (total ms, launches)} for the launches since the last collect."""
    ms = (ctypes.c_double * 16)()
    cnt = (ctypes.c_int32 * 16)()
    n = LIB.bd3_profile_collect_all(ms, cnt, len(PROFILE_KERNELS))
    if n < 0:
        check("bd3_profile_collect", -n)
    return {PROFILE_KERNELS[i]: (ms[i], cnt[i]) for i in range(len(PROFILE_KERNELS)) if cnt[i]}
