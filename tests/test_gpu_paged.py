"""Attention over a paged KV cache and the fused QKV / RoPE page write on the GPU against their
definitions in float64 (oracle/paged.py).

Tolerances. u is the unit roundoff of the type (bf16 2^-8, f16 2^-11): O is rounded once
(u |O|) and the probabilities once before the P V product (u sum p |V|); an f16 probability
below 2^-14 of the largest is off by up to 2^-25 instead (times the keys and max |V|). fp32
accumulation, exponentials and the merge of partial sums add a few 2^-22 of the same sums,
covered by the factor 1.1. The LSE is fp32: a score's error is at most 64 products and sums
of 2^-24 of sum |q k| scale, below 1e-4 for these inputs.
"""

import math

import pytest
import torch

from gpu_util import assert_device_ok
from oracle import paged as op

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LSE_TOL = 1e-4


def make(seed, lens, Hq, Hkv, page_size, dtype, layout="hnd", junk=True, spare=2, width=0):
    """Packed new tokens and a cache of the sequences lens = [(new, positions)], pages handed out
    in no order. With junk, rows past each sequence's end and unused pages hold NaN, and table
    entries past a sequence's pages hold ids outside the cache."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-m // page_size) for _, m in lens]
    width = max(max(need), 1) + width
    order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    pages = [torch.randn(sum(need) + spare, Hkv, page_size, 64, generator=g).to(dtype) for _ in "kv"]
    table = torch.full((len(lens), width), -12345 if junk else 0, dtype=torch.int32)
    used = torch.zeros(sum(need) + spare, page_size, dtype=torch.bool)
    at = 0
    for b, (n, m) in enumerate(lens):
        table[b, :need[b]] = order[at:at + need[b]]
        for j in range(need[b]):
            used[order[at + j].long(), :min(page_size, m - j * page_size)] = True
        at += need[b]
    if junk:
        for x in pages:
            x.masked_fill_(~used[:, None, :, None], math.nan)
    cu = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32)
    q = torch.randn(int(cu[-1]), Hq, 64, generator=g).to(dtype)
    d = dict(q=q, k_pages=pages[0], v_pages=pages[1], page_table=table,
             kv_lens=torch.tensor([m for _, m in lens], dtype=torch.int32), cu_q=cu)
    dev = {k: v.cuda() for k, v in d.items()}
    if layout == "nhd":  # page, row, head, dim in memory
        for k in ("k_pages", "v_pages"):
            dev[k] = dev[k].transpose(1, 2).contiguous().transpose(1, 2)
    return d, dev


def run(dev, lens, block_size, **kw):
    from bd3attn import ops
    return ops.paged_attn_raw(dev["q"], dev["k_pages"], dev["v_pages"], dev["page_table"],
                              dev["kv_lens"], dev["cu_q"], max(n for n, _ in lens), block_size, **kw)


def check(d, out, lse, block_size, scale=None, part=slice(None)):
    dt = d["q"].dtype
    ref, ref_lse, mag = op.paged_attention(d["q"], d["k_pages"], d["v_pages"], d["page_table"],
                                           d["kv_lens"], d["cu_q"], block_size, scale)
    o = out.cpu().double()
    out_u = U[out.dtype]
    tol = 1.1 * (out_u * ref.abs() + U[dt] * mag) + 1e-6
    if dt == torch.float16:
        tol = tol + int(d["kv_lens"].max()) * 2.0 ** -25 * 5
    bad = ((o - ref).abs() > tol)[part]
    assert torch.isfinite(o[part]).all() and not bad.any(), \
        f"{int(bad.sum())} of {bad.numel()} off, worst {(o - ref).abs().max():.3e}"
    if lse is not None:
        got = lse.cpu().double()
        none = ref_lse == -math.inf
        assert torch.equal(none, got == -math.inf)
        assert (o[none] == 0).all()
        err = (got - ref_lse)[~none].abs()
        assert err.numel() == 0 or err.max() <= LSE_TOL, err.max()


CASES = [
    # lens [(new, positions)], q heads, kv heads, page size, block size
    ([(1, 1)], 1, 1, 16, 1),
    ([(16, 16)], 12, 12, 16, 16),
    ([(16, 1056)], 12, 12, 16, 16),
    ([(1, 64), (1, 65), (1, 63), (1, 1), (1, 129)], 4, 4, 64, 1),
    ([(1, 300), (1, 5000), (1, 7)], 8, 2, 16, 1),            # grouped heads, single tokens
    ([(7, 129), (0, 50), (3, 3), (16, 700), (0, 0)], 6, 2, 48, 4),  # empty sequences
    ([(16, 4112)] * 3, 2, 2, 256, 16),
    ([(5, 400), (16, 16), (31, 77)], 3, 1, 8, 4),            # pages of 8, G = 3
    ([(32, 333)], 2, 2, 32, 16), ([(33, 333)], 2, 2, 32, 16),
    ([(64, 64), (64, 1000)], 2, 2, 64, 64),
    ([(100, 1000), (1, 2000), (260, 260), (16, 999)], 4, 2, 48, 4),
    ([(130, 131)], 5, 5, 16, 1), ([(128, 128)], 2, 1, 128, 1), ([(129, 500)], 2, 2, 64, 16),
    ([(300, 2500)], 8, 1, 24, 16),                           # one KV head, 8 query heads
    ([(1, 40000)], 4, 4, 64, 16),                            # few rows, a long axis
    ([(24, 30000), (1, 20)], 2, 1, 128, 8),
    ([(500, 500)] * 5, 2, 2, 64, 500),                       # bidirectional
    ([(4, 10)] * 200, 2, 1, 16, 2),                          # many short sequences
    ([(600, 9000)], 1, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{c[0][0]}h{c[1]}k{c[2]}p{c[3]}b{c[4]}")
def test_matches_definition(case, dtype):
    lens, Hq, Hkv, ps, bs = case
    d, dev = make(len(lens) + ps, lens, Hq, Hkv, ps, dtype)
    o, lse = run(dev, lens, bs, return_lse=True)
    assert_device_ok()
    assert o.dtype == dtype and o.shape == d["q"].shape
    check(d, o, lse, bs)


@pytest.mark.parametrize("lens", [[(3, 1), (2, 0), (40, 7), (4, 50)], [(200, 20), (1, 0)]],
                         ids=["short", "long"])
def test_rows_without_keys(lens):
    """More new tokens than positions: the leading ones see nothing and get O = 0, LSE = -inf."""
    d, dev = make(3, lens, 4, 2, 16, torch.bfloat16)
    o, lse = run(dev, lens, 1, return_lse=True)
    assert_device_ok()
    check(d, o, lse, 1)


@pytest.mark.parametrize("lens", [[(16, 700), (1, 65)], [(150, 700), (1, 65)]], ids=["few", "many"])
def test_layouts_strides_and_output_types(lens):
    """Page-row-head order in memory, q as a slice of a wider projection, fp32 output."""
    d, dev = make(5, lens, 6, 3, 32, torch.bfloat16, layout="nhd")
    wide = torch.randn(len(d["q"]), 10, 64).bfloat16().cuda()
    wide[:, 2:8] = dev["q"]
    dev["q"] = wide[:, 2:8]
    assert not dev["q"].is_contiguous()
    o, lse = run(dev, lens, 4, return_lse=True, out_dtype=torch.float32, scale=0.2)
    assert_device_ok()
    assert o.dtype == torch.float32
    check(d, o, lse, 4, 0.2)
    odd = torch.empty(len(d["q"]) * 6 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:]
    odd.copy_(wide[:, 2:8].reshape(-1))
    dev["q"] = odd.view(-1, 6, 64)  # 2-byte aligned: copied
    o2 = run(dev, lens, 4, out_dtype=torch.float32, scale=0.2)
    assert torch.equal(o, o2)


@pytest.mark.parametrize("rows", [16, 200])
def test_extreme_scores(rows):
    """Scores far apart: a softmax with one survivor, without overflow."""
    lens = [(rows, 1000)]
    d, dev = make(6, lens, 2, 2, 64, torch.bfloat16)
    for x in (d, dev):
        x["q"].mul_(64)
        x["k_pages"].mul_(16)
    o, lse = run(dev, lens, 16, return_lse=True)
    assert_device_ok()
    ref, ref_lse, mag = op.paged_attention(d["q"], d["k_pages"], d["v_pages"], d["page_table"],
                                           d["kv_lens"], d["cu_q"], 16)
    # fp32 scores of this size are off by up to 2^-20 of sum |q k| scale: about 0.01
    assert torch.isfinite(o).all()
    assert ((o.cpu().double() - ref).abs() <= 1.1 * 2.0 ** -8 * (ref.abs() + mag) + 0.05 * mag).all()
    assert ((lse.cpu().double() - ref_lse).abs() <= 1e-5 * ref_lse.abs() + 0.02).all()


def test_workspace_is_left_ready_and_results_repeat():
    """One workspace serves calls of other sizes and both row ranges, in any order; its counts are
    zero after each; the same call gives the same bits."""
    from bd3attn import ops
    ws = ops.paged_workspace("cuda")
    sets = [([(16, 5000), (16, 300)], 16), ([(1, 9000)], 1), ([(300, 3000)], 16), ([(40, 6000)], 4)]
    made = [make(10 + i, lens, 4, 2, 16, torch.bfloat16) for i, (lens, _) in enumerate(sets)]
    first = [run(dev, lens, bs, workspace=ws) for (lens, bs), (_, dev) in zip(sets, made)]
    for _ in range(3):
        for i in (2, 0, 3, 1):
            again = run(made[i][1], *sets[i], workspace=ws)
            assert torch.equal(again, first[i])
    assert torch.equal(run(made[0][1], *sets[0]), first[0])  # a workspace of its own
    assert_device_ok()
    for i, (lens, bs) in enumerate(sets):
        check(made[i][0], first[i], None, bs)


@pytest.mark.parametrize("case", [([(300, 2500)], 8, 1, 24, 16), ([(600, 9000)], 1, 1, 64, 16),
                                  ([(16, 3000)] * 4, 2, 2, 16, 16), ([(1, 40000)], 8, 2, 64, 1)],
                         ids=["300", "600", "16", "1"])
def test_same_bits_in_many_calls(case):
    """Keys that stay in L2 refill the kernels' rings at the highest rate: every call gives the
    first one's bits, whichever CTA merges an item's partials."""
    from bd3attn import ops
    lens, Hq, Hkv, ps, bs = case
    d, dev = make(60, lens, Hq, Hkv, ps, torch.bfloat16)
    ws = ops.paged_workspace("cuda")
    first = run(dev, lens, bs, workspace=ws)
    check(d, first, None, bs)
    same = [torch.equal(run(dev, lens, bs, workspace=ws), first) for _ in range(200)]
    assert_device_ok()
    assert all(same), f"{same.count(False)} of 200 calls differ"


def test_other_stream_and_graph_with_new_lengths():
    """On a side stream, and captured once: a replay reads the lengths and the table anew."""
    from bd3attn import ops
    lens_a, lens_b = [(16, 700), (16, 40), (16, 1500)], [(16, 100), (10, 1600), (16, 16)]
    d, dev = make(20, lens_a, 4, 4, 16, torch.bfloat16, junk=False, spare=4)
    d2, dev2 = make(21, lens_b, 4, 4, 16, torch.bfloat16, junk=False, spare=400)
    side, ws = torch.cuda.Stream(), ops.paged_workspace("cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = run(dev, lens_a, 16, workspace=ws)
    side.synchronize()
    check(d, o, None, 16)
    width = max(d["page_table"].shape[1], d2["page_table"].shape[1])
    n_pages = max(len(d["k_pages"]), len(d2["k_pages"]))
    buf = {"q": torch.zeros(48, 4, 64, dtype=torch.bfloat16, device="cuda"),
           "k_pages": torch.zeros(n_pages, 4, 16, 64, dtype=torch.bfloat16, device="cuda"),
           "page_table": torch.zeros(3, width, dtype=torch.int32, device="cuda"),
           "kv_lens": torch.zeros(3, dtype=torch.int32, device="cuda"),
           "cu_q": torch.zeros(4, dtype=torch.int32, device="cuda")}
    buf["v_pages"] = torch.zeros_like(buf["k_pages"])

    def load(x):
        for k, t in buf.items():
            t.zero_()
            t[tuple(slice(0, n) for n in x[k].shape)].copy_(x[k])

    load(dev)
    run(buf, [(16, 0)], 16, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(buf, [(16, 0)], 16, workspace=ws)
    for x, dd in ((dev, d), (dev2, d2), (dev, d)):
        load(x)
        graph.replay()
        torch.cuda.synchronize()
        check(dd, out[:len(dd["q"])], None, 16)  # rows past cu_q[B] are left alone
    assert_device_ok()


def test_compiled_call_traces():
    from bd3attn import ops
    lens = [(16, 100), (5, 40)]
    d, dev = make(30, lens, 4, 2, 16, torch.bfloat16)
    ws = ops.paged_workspace("cuda")

    @torch.compile(fullgraph=True, backend="eager")
    def f(q, k, v, t, m, cu, w):
        return torch.ops.bd3.paged_attn(q, k, v, t, m, cu, 16, 4, w) * 1.0

    o = f(dev["q"], dev["k_pages"], dev["v_pages"], dev["page_table"], dev["kv_lens"], dev["cu_q"], ws)
    assert_device_ok()
    check(d, o, None, 4)


@pytest.mark.parametrize("rows", [16, 160])
def test_bad_lengths_and_pages_are_cut_and_reported(rows):
    """Lengths, offsets and page ids outside the call's bounds: nothing outside is touched, the
    other sequence's rows are right, and the device status says so."""
    from bd3attn import ops
    lens = [(rows, 400), (rows, 300)]
    d, dev = make(40, lens, 2, 2, 16, torch.bfloat16, junk=False)
    ws = ops.paged_workspace("cuda")
    ref = run(dev, lens, 16, workspace=ws)
    assert_device_ok()
    for name, at, value in (("page_table", (0, 3), 10 ** 6), ("page_table", (0, 3), -5),
                            ("kv_lens", (0,), 10 ** 9), ("kv_lens", (0,), -7)):
        bad = {k: v.clone() for k, v in dev.items()}
        bad[name][at] = value
        o = run(bad, lens, 16, workspace=ws)
        torch.cuda.synchronize()
        assert ops.device_status() == 2, (name, value)
        # (another length of the first sequence moves the borders between the shares: not the
        # same bits)
        check(d, o, None, 16, part=slice(rows, None))
    bad = {k: v.clone() for k, v in dev.items()}
    bad["cu_q"][2] = 10 ** 8
    o = run(bad, lens, 16, workspace=ws)
    torch.cuda.synchronize()
    assert ops.device_status() == 2
    check(d, o, None, 16, part=slice(0, rows))
    assert torch.equal(run(dev, lens, 16, workspace=ws), ref)  # the workspace is as it was


def test_refusals():
    from bd3attn import ops
    from bd3attn._lib import BD3Error
    lens = [(16, 100)]
    _, dev = make(50, lens, 4, 2, 16, torch.bfloat16)

    def refused(kind, block_size=16, lens=lens, **over):
        kw = over.pop("kw", {})
        with pytest.raises(kind):
            run({**dev, **over}, lens, block_size, **kw)

    refused(AssertionError, kv_lens=dev["kv_lens"].long())
    refused(AssertionError, page_table=dev["page_table"][0])
    refused(AssertionError, cu_q=dev["cu_q"][:1])
    refused(AssertionError, k_pages=dev["k_pages"].half())
    refused(AssertionError, q=dev["q"].cpu())
    refused(AssertionError, v_pages=dev["v_pages"][:1])
    refused(TypeError, q=dev["q"].double(), k_pages=dev["k_pages"].double(), v_pages=dev["v_pages"].double())
    refused(BD3Error, q=dev["q"][:, :3])                     # 3 query heads over 2
    refused(BD3Error, block_size=0)
    refused(BD3Error, q=dev["q"].float(), k_pages=dev["k_pages"].float(), v_pages=dev["v_pages"].float())
    refused(BD3Error, k_pages=dev["k_pages"][:, :, :12], v_pages=dev["v_pages"][:, :, :12])  # page of 12
    refused(BD3Error, kw=dict(out_dtype=torch.float16))
    refused(BD3Error, kw=dict(scale=0.0))
    refused(BD3Error, kw=dict(scale=math.inf))
    refused(BD3Error, kw=dict(workspace=torch.zeros(64, dtype=torch.uint8, device="cuda")))
    narrow = torch.zeros(20, 2, 16, 32, dtype=torch.bfloat16, device="cuda")
    refused(BD3Error, q=dev["q"][:, :, :32].contiguous(), k_pages=narrow, v_pages=narrow)  # head_dim 32
    assert_device_ok()


# ---- the fused split, rotation and page write --------------------------------------------------

def rope_case(seed, lens, Hq, Hkv, D, page_size, dtype, layout="hnd"):
    g = torch.Generator().manual_seed(seed)
    need = [-(-m // page_size) for _, m in lens]
    ids = torch.randperm(sum(need) + 2, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), -9, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    cu = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32)
    pages = [torch.randn(sum(need) + 2, Hkv, page_size, D, generator=g).to(dtype) for _ in "kv"]
    angle = torch.rand(max(m for _, m in lens) + 3, D // 2, generator=g) * 6.3
    d = dict(qkv=torch.randn(int(cu[-1]), (Hq + 2 * Hkv) * D, generator=g).to(dtype),
             cos=angle.cos(), sin=angle.sin(), k_pages=pages[0], v_pages=pages[1], page_table=table,
             kv_lens=torch.tensor([m for _, m in lens], dtype=torch.int32), cu_q=cu)
    dev = {k: v.cuda() for k, v in d.items()}
    if layout == "nhd":
        for k in ("k_pages", "v_pages"):
            dev[k] = dev[k].transpose(1, 2).contiguous().transpose(1, 2)
    return d, dev


def write(x, Hq, Hkv, **kw):
    from bd3attn import ops
    return ops.qkv_rope_paged_raw(x["qkv"], Hq, Hkv, x["cos"], x["sin"], x["k_pages"], x["v_pages"],
                                  x["page_table"], x["kv_lens"], x["cu_q"], **kw)


def check_write(d, dev, q, Hq, Hkv):
    """q and k: fp32 products and sums (3 x 2^-24 of |x_1| + |x_2|, here below 2e-6) and one
    rounding; v and every other row of the cache: the same bits."""
    u = U[d["qkv"].dtype]
    rq, rk, rv = op.rope_write(d["qkv"], Hq, Hkv, d["cos"], d["sin"], d["k_pages"], d["v_pages"],
                               d["page_table"], d["kv_lens"], d["cu_q"])
    for name, got, ref in (("q", q, rq), ("k", dev["k_pages"], rk)):
        err = (got.cpu().double() - ref).abs()
        assert (err <= 1.01 * u * ref.abs() + 2e-6).all(), (name, err.max())
    assert torch.equal(dev["v_pages"].cpu().double(), rv)
    touched = (rk != d["k_pages"].double()).flatten(1).any(1)
    assert torch.equal(dev["k_pages"].cpu()[~touched], d["k_pages"][~touched])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32],
                         ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", [
    ([(1, 1)], 1, 1, 64, 16, "hnd"), ([(16, 1056)], 12, 12, 64, 16, "nhd"),
    ([(5, 9), (0, 30), (1, 200), (70, 70), (0, 0), (3, 131)], 6, 2, 64, 48, "hnd"),
    ([(1, k + 1) for k in range(300)], 4, 1, 64, 8, "hnd"),
    ([(33, 50)], 2, 1, 128, 5, "nhd"), ([(9, 20), (9, 9)], 3, 3, 16, 1, "hnd"),
    ([(200, 1000)], 2, 2, 96, 64, "hnd"),
], ids=lambda c: f"{len(c[0])}x{c[0][0]}h{c[1]}k{c[2]}d{c[3]}p{c[4]}{c[5]}")
def test_rope_write_matches_definition(case, dtype):
    lens, Hq, Hkv, D, ps, layout = case
    d, dev = rope_case(7, lens, Hq, Hkv, D, ps, dtype, layout)
    q = write(dev, Hq, Hkv)
    assert_device_ok()
    check_write(d, dev, q, Hq, Hkv)


def test_rope_write_strided_projection_and_padding_tokens():
    """qkv with a wider row, q_out of the caller's, tokens past cu_q[B] left alone."""
    Hq, Hkv = 4, 2
    d, dev = rope_case(8, [(5, 40), (2, 3)], Hq, Hkv, 64, 16, torch.bfloat16)
    wide = torch.zeros(10, 8 * 64 + 64, dtype=torch.bfloat16, device="cuda")
    wide[:7, :512] = dev["qkv"]
    dev["qkv"] = wide[:, :512]
    out = torch.full((10, 2 * Hq, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    q = write(dev, Hq, Hkv, q_out=out[:, :Hq])
    assert_device_ok()
    assert (out[7:] == 7).all() and (out[:, Hq:] == 7).all()
    check_write(d, dev, q[:7], Hq, Hkv)


def test_rope_write_reports_positions_outside():
    """A token past the tables, or on a page that does not exist, writes nothing (status bit 4)."""
    from bd3attn import ops
    d, dev = rope_case(9, [(4, 20), (4, 8)], 2, 1, 64, 16, torch.bfloat16)
    for name, at, value in (("page_table", (0, 1), 10 ** 6), ("page_table", (0, 1), -1),
                            ("kv_lens", (0,), 10 ** 6), ("kv_lens", (0,), 1)):
        bad = {k: v.clone() for k, v in dev.items()}
        bad[name][at] = value
        q = write(bad, 2, 1)
        torch.cuda.synchronize()
        assert ops.device_status() == 4, (name, value)
        good = {k: v.clone() for k, v in dev.items()}
        assert torch.equal(q[4:], write(good, 2, 1)[4:])
    bad = {k: v.clone() for k, v in dev.items()}
    bad["cos"], bad["sin"] = bad["cos"][:19], bad["sin"][:19]  # the last position has no angle
    before = bad["k_pages"].clone()
    write(bad, 2, 1)
    torch.cuda.synchronize()
    assert ops.device_status() == 4
    page = int(d["page_table"][0, 1])
    assert torch.equal(bad["k_pages"][page, :, 3:], before[page, :, 3:])


def test_rope_write_refusals():
    from bd3attn._lib import BD3Error
    _, dev = rope_case(9, [(4, 20)], 2, 1, 64, 16, torch.bfloat16)

    def refused(kind, Hq=2, **over):
        with pytest.raises(kind):
            write({**dev, **over}, Hq, 1)

    refused(AssertionError, Hq=3)
    refused(AssertionError, cos=dev["cos"].double())
    refused(AssertionError, cos=dev["cos"][:, :16])
    refused(AssertionError, k_pages=dev["k_pages"].half())
    refused(AssertionError, cu_q=dev["cu_q"].long())
    refused(BD3Error, k_pages=torch.zeros(4, 1, 16, 68, dtype=torch.bfloat16, device="cuda")[..., :64],
            v_pages=torch.zeros(4, 1, 16, 68, dtype=torch.bfloat16, device="cuda")[..., :64])
    assert_device_ok()


def test_write_then_attend():
    """A prompt written and attended in chunks equals the whole prompt at once."""
    Hq, Hkv, ps, bs, n = 4, 2, 16, 16, 208
    d, dev = rope_case(11, [(n, n)], Hq, Hkv, 64, ps, torch.bfloat16)
    from bd3attn import ops
    ws = ops.paged_workspace("cuda")

    def step(a, e, pages):
        x = {**dev, **pages, "qkv": dev["qkv"][a:e], "kv_lens": torch.tensor([e], dtype=torch.int32, device="cuda"),
             "cu_q": torch.tensor([0, e - a], dtype=torch.int32, device="cuda")}
        q = write(x, Hq, Hkv)
        return ops.paged_attn_raw(q, x["k_pages"], x["v_pages"], x["page_table"], x["kv_lens"], x["cu_q"],
                                  e - a, bs, workspace=ws)

    whole = {k: torch.full_like(dev[k], math.nan) for k in ("k_pages", "v_pages")}
    parts = {k: v.clone() for k, v in whole.items()}
    o = step(0, n, whole)
    cuts = [0, 64, 80, 176, n]
    o2 = torch.cat([step(a, e, parts) for a, e in zip(cuts, cuts[1:])])
    assert_device_ok()
    assert torch.equal(whole["k_pages"].nan_to_num(9), parts["k_pages"].nan_to_num(9))
    assert (o.float() - o2.float()).abs().max() <= 2 * 2.0 ** -8 * 4.5  # two roundings of |O| < 4.5 each

# ---- packed rows that belong to no sequence ----------------------------------------------------

@pytest.mark.parametrize("first", [1, 3, 40, 700])
def test_rope_write_leaves_the_rows_before_the_first_sequence_alone(first):
    """A sub-batch over the whole packed projection: rows before cu_q[0] are in no sequence, though
    the first sequence has earlier positions that they would count back to."""
    Hq, Hkv = 4, 2
    d, dev = rope_case(12, [(5, 800), (0, 30), (2, 3)], Hq, Hkv, 64, 16, torch.bfloat16)
    g = torch.Generator().manual_seed(13)
    before = torch.randn(first, 8 * 64, generator=g).bfloat16()
    d["qkv"] = torch.cat([before, d["qkv"]])
    d["cu_q"] = d["cu_q"] + first
    dev["qkv"], dev["cu_q"] = d["qkv"].cuda(), d["cu_q"].cuda()
    out = torch.full((first + 7, Hq, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    q = write(dev, Hq, Hkv, q_out=out)
    assert_device_ok()
    assert (q[:first] == 7).all()
    rq, rk, rv = op.rope_write(d["qkv"], Hq, Hkv, d["cos"], d["sin"], d["k_pages"], d["v_pages"],
                               d["page_table"], d["kv_lens"], d["cu_q"])
    assert torch.equal(dev["v_pages"].cpu().double(), rv)
    for got, ref in ((q[first:], rq[first:]), (dev["k_pages"], rk)):
        assert ((got.cpu().double() - ref).abs() <= 1.01 * 2.0 ** -8 * ref.abs() + 2e-6).all()
    touched = (rk != d["k_pages"].double()).any(-1).any(1)  # (page, row)
    assert torch.equal(dev["k_pages"].cpu().transpose(1, 2)[~touched], d["k_pages"].transpose(1, 2)[~touched])


def test_offsets_that_run_back_reach_no_other_row():
    """Offsets that run back are outside the contract: the write touches no row but those that the
    offsets name, the attention reports them (status bit 2)."""
    from bd3attn import ops
    d, dev = rope_case(14, [(4, 300), (4, 90)], 4, 2, 64, 16, torch.bfloat16)
    dev["cu_q"] = torch.tensor([6, 8, 4], dtype=torch.int32, device="cuda")
    q = write(dev, 4, 2)
    assert_device_ok()
    k = d["k_pages"].clone()
    page = d["page_table"]
    touched = torch.zeros(k.shape[0], 16, dtype=torch.bool)
    for pos in (298, 299):  # rows 6 and 7 are the first sequence's last positions
        touched[page[0, pos // 16].long(), pos % 16] = True
    assert torch.equal(dev["k_pages"].cpu().transpose(1, 2)[~touched], k.transpose(1, 2)[~touched])
    ops.paged_attn_raw(q, dev["k_pages"], dev["v_pages"], dev["page_table"], dev["kv_lens"], dev["cu_q"], 2, 16)
    torch.cuda.synchronize()
    assert ops.device_status() == 2


@pytest.mark.parametrize("rows", [16, 160])
def test_attention_of_a_sub_batch(rows):
    """cu_q[k:], kv_lens[k:] and page_table[k:] over the whole packed q: the rows of the sequences
    left out, before cu_q[0] and past cu_q[B], belong to no sequence."""
    lens = [(rows, 700), (rows, 90 + rows), (7, 333), (rows, rows)]
    d, dev = make(61, lens, 4, 2, 16, torch.bfloat16)
    for x in (d, dev):
        x.update(cu_q=x["cu_q"][1:4], kv_lens=x["kv_lens"][1:3], page_table=x["page_table"][1:3])
    d["kv_lens"], dev["kv_lens"] = d["kv_lens"].clone(), dev["kv_lens"].clone()
    dev["cu_q"] = dev["cu_q"].clone()
    o, lse = run(dev, lens, 16, return_lse=True)
    assert_device_ok()
    part = slice(rows, 2 * rows + 7)
    ref, ref_lse, mag = op.paged_attention(d["q"], d["k_pages"], d["v_pages"], d["page_table"], d["kv_lens"],
                                           d["cu_q"], 16)
    err = (o.cpu().double() - ref).abs()[part]
    assert (err <= (1.1 * 2.0 ** -8 * (ref.abs() + mag) + 1e-6)[part]).all()
    assert ((lse.cpu().double() - ref_lse).abs()[part] <= LSE_TOL).all()


def test_no_length_for_the_tokens_is_refused():
    """max_q_len 0 (or less) beside tokens would leave the output as it was allocated."""
    from bd3attn import ops
    lens = [(16, 100), (3, 40)]
    _, dev = make(62, lens, 4, 2, 16, torch.bfloat16)
    args = [dev[k] for k in ("q", "k_pages", "v_pages", "page_table", "kv_lens", "cu_q")]
    for n in (0, -1):
        with pytest.raises(AssertionError, match="max_q_len"):
            ops.paged_attn_raw(*args, n, 16)
        with pytest.raises(AssertionError, match="max_q_len"):
            ops.paged_attn_raw(*args, n, 16, return_lse=True, workspace=ops.paged_workspace("cuda"))
    o, lse = ops.paged_attn_raw(args[0][:0], *args[1:5], torch.zeros_like(dev["cu_q"]), 0, 16, return_lse=True)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)  # no tokens: nothing to do
    assert_device_ok()
