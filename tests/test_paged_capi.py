"""Host-side argument checks of the paged-cache and logits entry points: every pointer is a dummy,
so only calls that are refused before any CUDA call may be made here. And the float64 oracle of
these operators against differently written formulas."""

import math

import pytest
import torch

from oracle import paged as op


def _attn(**over):
    from bd3attn._lib import LIB, i64_array
    a = dict(q=0x1000, o=0x4000, table=0x5000, lens=0x6000, cu=0x7000, B=2, total=32, max_q=16, Hq=4,
             Hkv=2, D=64, pages=8, page=16, width=4, strides=[256, 64] + [2048, 1024, 64] * 2 + [256, 64, 4],
             bs=16, scale=0.125, dtype=0, out=0, ws=0x8000)
    a.update(over)
    return LIB.bd3_paged_attn(a["q"], 0x2000, 0x3000, a["o"], None, a["table"], a["lens"], a["cu"], a["B"],
                              a["total"], a["max_q"], a["Hq"], a["Hkv"], a["D"], a["pages"], a["page"],
                              a["width"], i64_array(a["strides"]), a["bs"], a["scale"], a["dtype"], a["out"],
                              a["ws"], 1 << 30, None)


def test_paged_attention_refusals():
    from bd3attn._lib import (BD3_ERR_INVALID, BD3_ERR_UNSUPPORTED, BD3_ERR_WORKSPACE, BD3_F32, BD3_OK,
                              LIB)
    for over in (dict(B=0), dict(Hkv=0), dict(pages=0), dict(page=0), dict(width=0), dict(Hq=3), dict(Hq=0),
                 dict(table=None), dict(lens=0x6002), dict(cu=None), dict(total=-1), dict(max_q=-1),
                 dict(bs=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
                 dict(out=1), dict(q=None), dict(q=0x1008), dict(o=0x4004),
                 dict(strides=[252, 64] + [2048, 1024, 64] * 2 + [256, 64, 4]),
                 dict(strides=[256, 64] + [2048, 1024, 64] * 2 + [256, 60, 4])):
        assert _attn(**over) == BD3_ERR_INVALID, over
        assert LIB.bd3_last_error()
    for over in (dict(D=128), dict(dtype=BD3_F32, out=BD3_F32), dict(page=12), dict(page=4),
                 dict(pages=1 << 31), dict(width=1 << 28), dict(total=1 << 31, max_q=1 << 31)):
        assert _attn(**over) == BD3_ERR_UNSUPPORTED, over
    assert _attn(ws=None) == BD3_ERR_WORKSPACE
    assert _attn(total=0) == BD3_OK and _attn(max_q=0) == BD3_OK  # no new token: nothing to do


def _write(**over):
    from bd3attn._lib import LIB, i64_array
    a = dict(qkv=0x1000, stride=512, T=32, B=2, Hq=4, Hkv=2, D=64, cos=0x2000, max_pos=64, q=0x3000, k=0x4000,
             table=0x5000, pages=8, page=16, width=4, strides=[256, 64] + [2048, 1024, 64] * 2 + [4], dtype=0)
    a.update(over)
    return LIB.bd3_qkv_rope_paged(a["qkv"], a["stride"], a["T"], a["B"], a["Hq"], a["Hkv"], a["D"], a["cos"],
                                  0x2800, a["max_pos"], a["q"], a["k"], 0x4800, a["table"], 0x6000, 0x7000,
                                  a["pages"], a["page"], a["width"], i64_array(a["strides"]), a["dtype"], None)


def test_paged_write_refusals():
    from bd3attn._lib import BD3_ERR_INVALID, BD3_ERR_UNSUPPORTED, BD3_OK
    for over in (dict(B=0), dict(Hq=0), dict(Hkv=0), dict(T=-1), dict(cos=None), dict(cos=0x2004),
                 dict(max_pos=0), dict(qkv=0x1008), dict(q=None), dict(k=0x4002), dict(stride=508),
                 dict(table=None), dict(strides=[256, 64] + [2048, 1024, 68] * 2 + [4])):
        assert _write(**over) == BD3_ERR_INVALID, over
    for over in (dict(D=24), dict(D=8), dict(dtype=7), dict(D=2048)):
        assert _write(**over) == BD3_ERR_UNSUPPORTED, over
    assert _write(T=0) == BD3_OK


def _logits(**over):
    from bd3attn._lib import LIB, i64_array
    a = dict(x=0x1000, out=0x2000, B=2, S=3, V=100, hist=0x3000, i32=0, cap=8, hlen=0x4000, allowed=0x5000,
             astr=i64_array([4, 0]), dtype=0)
    a.update(over)
    return LIB.bd3_process_logits(a["x"], a["out"], i64_array([300, 100] * 2), a["B"], a["S"], a["V"], a["hist"],
                                  a["i32"], 8, a["cap"], a["hlen"], None, None, None, None, 0, a["allowed"],
                                  a["astr"], a["dtype"], None)


def test_logits_refusals():
    from bd3attn._lib import BD3_ERR_INVALID, BD3_ERR_UNSUPPORTED
    for over in (dict(B=0), dict(S=0), dict(V=0), dict(x=None), dict(out=None), dict(x=0x1001), dict(dtype=2, out=0x2002),
                 dict(hlen=None), dict(cap=-1), dict(hist=0x3004), dict(astr=None)):
        assert _logits(**over) == BD3_ERR_INVALID, over
    for over in (dict(dtype=5), dict(B=70000), dict(V=1 << 31)):
        assert _logits(**over) == BD3_ERR_UNSUPPORTED, over


def test_logits_refuse_misaligned_vectors():
    from bd3attn._lib import BD3_ERR_INVALID, LIB, i64_array
    fine = [0x4000] * 6  # lengths, repetition, presence, frequency, bias, mask
    for i in range(6):
        a = fine[:i] + [0x4000 + 1 + i % 3] + fine[i + 1:]
        assert LIB.bd3_process_logits(0x1000, 0x2000, i64_array([300, 100] * 2), 2, 3, 100, 0x3000, 0, 8, 8,
                                      *a[:5], 0, a[5], i64_array([4, 0]), 0, None) == BD3_ERR_INVALID, i


def test_oracle_attention_on_a_contiguous_cache():
    """Pages in order: the paged oracle equals the block-causal oracle of the contiguous cache."""
    import oracle
    g = torch.Generator().manual_seed(0)
    H, n, m, bs, ps = 2, 20, 70, 16, 8
    k, v = (torch.randn(1, H, 72, 64, generator=g) for _ in "kv")
    q = torch.randn(n, H, 64, generator=g)
    pages = [x[0].unflatten(1, (9, ps)).transpose(0, 1) for x in (k, v)]
    o, lse, mag = op.paged_attention(q, *pages, torch.arange(9)[None].int(), torch.tensor([m]),
                                     torch.tensor([0, n]), bs)
    ref, ref_lse = oracle.attention(q.transpose(0, 1)[None], k[:, :, :m], v[:, :, :m],
                                    oracle.block_causal_mask(n, m, bs))
    assert (o.transpose(0, 1)[None] - ref.double()).abs().max() < 1e-5
    assert (lse.T[None] - ref_lse.double()).abs().max() < 1e-5
    assert (mag >= o.abs() - 1e-12).all()


def test_oracle_rows_without_keys_and_logits():
    q = torch.ones(3, 1, 64)
    pages = torch.ones(1, 1, 8, 64)
    o, lse, _ = op.paged_attention(q, pages, pages, torch.zeros(1, 1).int(), torch.tensor([1]),
                                   torch.tensor([0, 3]), 1)
    assert (o[:2] == 0).all() and (lse[:2] == -math.inf).all()
    assert (o[2] == 1).all() and lse[2, 0] == pytest.approx(8.0)
    x = torch.tensor([[[2.0, -2.0, 1.0, 0.5]]])
    y = op.process_logits(x, torch.tensor([[0, 1, 1, 9]]), torch.tensor([4]), torch.tensor([2.0]),
                          torch.tensor([0.5]), torch.tensor([0.25]), torch.ones(4),
                          torch.tensor([[True, True, True, False]]))
    assert y[0, 0].tolist() == [2 / 2 - 0.25 - 0.5 + 1, -2 * 2 - 0.5 - 0.5 + 1, 2.0, -math.inf]


def test_pack_mask():
    from bd3attn.logits import pack_mask
    g = torch.Generator().manual_seed(1)
    ok = torch.rand(3, 2, 101, generator=g) < 0.5
    words = pack_mask(ok)
    assert words.shape == (3, 2, 4) and words.dtype == torch.int32
    v = torch.arange(101)
    assert torch.equal((words.long()[..., v // 32] >> (v % 32) & 1).bool(), ok)
