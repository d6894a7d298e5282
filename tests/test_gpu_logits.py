"""process_logits on the GPU against its definition in float64 (oracle/paged.py).

Tolerance: the result is rounded once (unit roundoff u of the type) after at most five fp32
operations, each off by 2^-24 of the magnitudes that enter it.
"""

import math

import pytest
import torch

from gpu_util import assert_device_ok
from oracle import paged as op

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def make(seed, B, S, V, dtype, cap, bias=None, allowed=None, lens=None, i32=False):
    g = torch.Generator().manual_seed(seed)
    d = dict(logits=(3 * torch.randn(B, S, V, generator=g)).to(dtype))
    if cap is not None:
        ids = (torch.rand(B, cap, generator=g) ** 2 * (V + 2)).long() - 1  # -1 and V among them
        d["history"] = ids.to(torch.int32) if i32 else ids
        d["history_len"] = torch.tensor(lens, dtype=torch.int32) if lens is not None else \
            torch.randint(0, cap + 1, (B,), generator=g, dtype=torch.int32)
        d["repetition"] = 0.8 + torch.rand(B, generator=g)
        d["presence"] = torch.randn(B, generator=g)
        d["frequency"] = torch.rand(B, generator=g)
    if bias:
        d["bias"] = torch.randn((V,) if bias == "vocab" else (B, V), generator=g)
    if allowed:
        keep = torch.rand((B, V) if allowed == "sequence" else (B, S, V), generator=g)
        d["allowed"] = (keep < 0.4) & (torch.rand((keep.shape[0],) + (1,) * (keep.dim() - 2) + (V // 64 + 1,), generator=g)
                                       .repeat_interleave(64, -1)[..., :V] < 0.6)
    return d


def call(d, **kw):
    from bd3attn.logits import pack_mask, process_logits
    x = {k: v.cuda() for k, v in d.items()}
    if "allowed" in x:
        x["allowed"] = pack_mask(x["allowed"])
    x.update(kw)
    return process_logits(x.pop("logits"), **x)


def check(d, out):
    ref = op.process_logits(**d)
    got = out.cpu().double()
    assert torch.equal(got == -math.inf, ref == -math.inf)
    fine = torch.isfinite(ref)
    big = d["logits"].double().abs() * 2 + 4
    if "frequency" in d:
        big = big + (d["frequency"].double() * d["history"].shape[1] + d["presence"].abs().double())[:, None, None]
    tol = 1.01 * U[out.dtype] * ref.abs() + 5 * 2.0 ** -24 * big
    err = (got - ref).abs()[fine]
    assert torch.equal(torch.isfinite(got), fine) and (err <= tol[fine]).all(), err.max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32],
                         ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", [
    (1, 1, 1, 3, None, None), (1, 1, 7, 5, "vocab", "row"), (2, 3, 8, 0, "vocab", None),
    (3, 2, 1027, 400, "sequence", "row"), (2, 16, 50258, 900, "vocab", "sequence"),
    (5, 1, 4099, 64, None, "row"), (1, 4, 33000, None, "sequence", None),
    (2, 2, 8191, None, None, "sequence"), (40, 1, 2050, 20, "vocab", None),
    (2, 1, 50257, 5000, None, None), (1, 2, 12301, None, None, None),
    # enough sequences for two and four chunks a thread, one slice and several
    (300, 2, 2050, 30, "vocab", "sequence"), (600, 1, 2051, 30, "sequence", "row"),
    (40, 1, 70001, 500, "vocab", "row"), (100, 3, 25000, 100, "vocab", "sequence"),
    # histories long enough for neighbouring CTAs to share their reading
    (3, 5, 50259, 2500, "vocab", "row"), (70, 1, 40961, 2048, None, "sequence"),
    (2, 1, 1500, 9000, "sequence", None),
], ids=lambda c: "x".join(str(v) for v in c))
def test_matches_definition(case, dtype):
    B, S, V, cap, bias, allowed = case
    d = make(B * 100 + S + V, B, S, V, dtype, cap, bias, allowed, i32=V % 2 == 0)
    before = d["logits"].clone()
    out = call(d)
    assert_device_ok()
    assert torch.equal(before, d["logits"]) and out.dtype == dtype
    check(d, out)


def test_history_lengths_are_cut():
    d = make(1, 4, 2, 3001, torch.float32, 50, lens=[0, 50, 1, 7])
    want = call(d)
    check(d, want)
    got = call(d, history_len=torch.tensor([-3, 10 ** 6, 1, 7], dtype=torch.int32, device="cuda"))
    assert torch.equal(got, want)


def test_in_place_views_and_alignments():
    """out is logits, slices of wider buffers at odd offsets, rows of other strides."""
    d = make(2, 3, 5, 2999, torch.bfloat16, 100, "vocab", "row")
    want = call(d)
    check(d, want)
    x = d["logits"].cuda()
    assert call(d, logits=x, out=x).data_ptr() == x.data_ptr()
    assert torch.equal(x, want)
    for off in (1, 3, 8):
        wide = torch.full((3, 6, 3100), 5.0, dtype=torch.bfloat16, device="cuda")
        view = wide[:, 1:, off:off + 2999]
        view.copy_(d["logits"].cuda())
        out = torch.full((5, 3, 3050), 6.0, dtype=torch.bfloat16, device="cuda")
        got = call(d, logits=view, out=out.transpose(0, 1)[..., 2:3001])
        assert torch.equal(got, want)
        assert (out[..., :2] == 6).all() and (out[..., 3001:] == 6).all()
        call(d, logits=view, out=view)
        assert torch.equal(view, want) and (wide[:, 0] == 5).all()
        assert (wide[..., :off] == 5).all() and (wide[:, :, off + 2999:] == 5).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("B", [3, 700])
def test_single_rows_in_views(B, dtype):
    """One row a sequence, of rows at odd offsets, in place and into other strides; what the mask
    forbids may be NaN and the history's tokens may lie at the rows' ends."""
    V = 2600
    d = make(7, B, 1, V, dtype, 80, "sequence", "row")
    d["history"][:, :3] = torch.tensor([0, V - 1, 5], dtype=d["history"].dtype)
    want = call(d)
    check(d, want)
    for off in (1, 2, 7):
        wide = torch.full((B, 2, 2651), math.nan, dtype=dtype, device="cuda")
        view = wide[:, 1:, off:off + V]
        view.copy_(d["logits"].masked_fill(~d["allowed"], math.nan).cuda())
        out = torch.full((B, 2613), 6.0, dtype=dtype, device="cuda")
        got = call(d, logits=view, out=out[:, None, 3:3 + V])
        assert torch.equal(got, want)
        assert (out[:, :3] == 6).all() and (out[:, 3 + V:] == 6).all()
        call(d, logits=view, out=view)
        assert torch.equal(view, want) and wide[:, 0].isnan().all()
        assert wide[..., :off].isnan().all() and wide[..., off + V:].isnan().all()
    assert_device_ok()


def test_infinities_nan_and_empty_masks():
    """NaN and infinities where the mask forbids do not matter; a row with nothing allowed is -inf
    throughout; -inf logits stay -inf through penalties."""
    d = make(3, 2, 3, 1500, torch.float32, 60, "vocab", "row")
    d["allowed"][0, 0] = False
    d["allowed"][1, 2] = True
    d["logits"][~d["allowed"]] = math.nan
    d["logits"][1, 0][~d["allowed"][1, 0]] = math.inf
    d["logits"][1, 2, ::7] = -math.inf
    out = call(d)
    assert_device_ok()
    assert (out[0, 0] == -math.inf).all()
    ref = op.process_logits(**{**d, "logits": d["logits"].nan_to_num(0, math.inf, -math.inf)})
    assert torch.equal(out.cpu() == -math.inf, ref == -math.inf) and not out.isnan().any()


def test_counts_repeat_and_capture():
    """A token repeated 70000 times counts in full; a captured call reads new histories."""
    B, S, V = 1, 2, 600
    d = make(4, B, S, V, torch.float32, 70000, lens=[70000])
    d["history"][:] = 17
    d["frequency"][:] = 0.001
    x = {k: v.cuda() for k, v in d.items()}
    out = call(d)
    check(d, out)
    from bd3attn.logits import process_logits
    buf = torch.empty_like(out)
    process_logits(out=buf, **x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        process_logits(out=buf, **x)
    d["history"][:] = 31
    d["history_len"][:] = 9
    x["history"].copy_(d["history"])
    x["history_len"].copy_(d["history_len"])
    graph.replay()
    torch.cuda.synchronize()
    check(d, buf)


def test_sampler_draws_allowed_tokens_only():
    """Processed logits into the sampler step: every drawn token is one the mask allows."""
    from bd3attn.sampler import subs_sample_step
    B, S, V, mask = 4, 16, 5003, 5002
    for dtype in (torch.bfloat16, torch.float32):
        d = make(5, B, S, V, dtype, 200, "vocab", "row")
        d["allowed"][..., :3] = True
        out = call(d)
        xt = torch.full((B, S), mask, dtype=torch.int64, device="cuda")
        tok = subs_sample_step(out, xt, mask, 1.0, 0.0, generator=torch.Generator().manual_seed(1))
        assert_device_ok()
        assert d["allowed"].gather(-1, tok.cpu()[..., None]).all()


def test_refusals():
    from bd3attn._lib import BD3Error
    d = make(6, 2, 3, 100, torch.float32, 10, "vocab", "row")
    z = torch.zeros(1, device="cuda")
    for kw in (dict(logits=d["logits"]), dict(logits=d["logits"].cuda()[0]), dict(repetition=z),
               dict(repetition=torch.ones(2, device="cuda").double()), dict(bias=z),
               dict(history_len=None), dict(history=d["history"].cuda().float()),
               dict(allowed=torch.zeros(2, 3, 3, dtype=torch.int32, device="cuda")),
               dict(out=torch.zeros(2, 3, 100, device="cuda").half()),
               dict(history_len=d["history_len"].cuda().long())):
        with pytest.raises(AssertionError):
            call(d, **kw)
    with pytest.raises(TypeError):
        call(d, logits=d["logits"].cuda().double())
    with pytest.raises(BD3Error):
        big = torch.zeros(1, 1, 8, device="cuda").expand(70000, 1, 8)
        call(dict(logits=big), out=torch.empty(70000, 1, 8, device="cuda"))
