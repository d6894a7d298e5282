"""Generation over the paged cache (workloads/serving.py) with a small stand-in backbone: the
packed, chunked forward gives the logits of encoding each sequence by itself under the
block-causal mask; grammar masks and penalties reach the drawn tokens; pages come back."""

import pytest
import torch

from gpu_util import assert_device_ok

pytestmark = pytest.mark.gpu

V, BS = 1000, 16
CFG = dict(d_model=128, n_heads=2, n_layers=2, d_ff=256)


@pytest.fixture(scope="module")
def model():
    from workloads.backbone import Backbone
    torch.manual_seed(0)
    return Backbone(V, 256, BS, **CFG).cuda().bfloat16().eval()


def full_logits(model, tokens):
    from workloads import backbone as bb
    bb.use_attention("sdpa")
    n = len(tokens)
    cos, sin = bb.rope_tables(64, n, "cuda")
    idx = torch.arange(n, device="cuda")
    mask = (idx[None, :] // BS) <= (idx[:, None] // BS)
    return model.encode(tokens[None], mask, cos, sin)[0].float()


@pytest.mark.parametrize("page_size", [16, 24, 64])
def test_packed_chunks_match_each_sequence_alone(model, page_size):
    from workloads.serving import PagedGeneration
    g = torch.Generator().manual_seed(1)
    lens = [16, 208, 64, 112]
    seqs = [torch.randint(0, V - 1, (n,), generator=g).cuda() for n in lens]
    gen = PagedGeneration(model, 4, 256, 80, page_size=page_size)
    ids = [gen.cache.add() for _ in lens]
    at, got = [0] * 4, [[] for _ in lens]
    # uneven chunks: blocks of one sequence beside longer chunks of another, one at a time absent
    with torch.no_grad():
        for step in range(20):
            take = {i: min(lens[i] - at[i], BS * (1 + (step + 3 * i) % 5)) for i in range(4)
                    if at[i] < lens[i] and (step + i) % 4}
            if not take:
                continue
            gen.cache.begin({ids[i]: n for i, n in take.items()})
            out = gen.forward(torch.cat([seqs[i][at[i]:at[i] + n] for i, n in take.items()]))
            gen.cache.commit()
            for part, (i, n) in zip(out.split(list(take.values())), take.items()):
                got[i].append(part)
                at[i] += n
        assert at == lens
        assert_device_ok()
        for i, s in enumerate(seqs):
            ref = full_logits(model, s)
            err = (torch.cat(got[i]).float() - ref).abs().max().item()
            assert err <= 0.03 * max(1.0, ref.abs().max().item()), (i, err)


def test_generation_keeps_to_the_grammar_and_returns_its_pages(model):
    from bd3attn.logits import pack_mask
    from workloads.serving import PagedGeneration
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, V - 1, (n,), generator=g).cuda() for n in (32, 0, 160, 48)]
    ok = torch.zeros(4, V, dtype=torch.bool)
    for i in range(4):
        ok[i, 10 * i:10 * i + 400:3] = True
    gen = PagedGeneration(model, 4, 256, 60, page_size=16, steps=4, chunk=64, repetition=1.3,
                          presence=0.2, frequency=0.1, bias=torch.randn(V, generator=g).cuda(), seed=3)
    out = gen.run(prompts, [2, 3, 1, 2], pack_mask(ok).cuda())
    assert_device_ok()
    assert [len(o) for o in out] == [32, 48, 16, 32]
    for i, o in enumerate(out):
        assert ok[i][o.cpu()].all()
    assert gen.cache.free_pages == 60
    assert [len(o) for o in gen.run(prompts[:1], [1])] == [16]  # the cache serves again


def test_penalties_reach_the_draw(model):
    """With a presence penalty beyond every logit, no token of the prompt is drawn; and without
    penalties the prompt's tokens do appear."""
    from workloads.serving import PagedGeneration
    prompt = torch.arange(0, V - 1).repeat_interleave(1)[:240].cuda()
    free = [PagedGeneration(model, 1, 256, 16, steps=4, seed=s).run([prompt], [1])[0] for s in range(4)]
    held = [PagedGeneration(model, 1, 256, 16, steps=4, seed=s, presence=1e4).run([prompt], [1])[0]
            for s in range(4)]
    assert_device_ok()
    assert any((o < 240).any() for o in free) and not any((o < 240).any() for o in held)


def test_the_timing_hooks_count_the_serving_launches():
    """A page write, an attention (each of its kernels) and a logits call under the timing hooks."""
    from bd3attn import ops
    from bd3attn.logits import process_logits
    tab = torch.ones(64, 32, device="cuda")
    kp, vp = (torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pages = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    lens, cu = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([40], [0, 40]))
    qkv = torch.randn(40, 8 * 64, device="cuda").bfloat16()
    ops.profile_enable(True)
    try:
        q = ops.qkv_rope_paged_raw(qkv, 4, 2, tab, tab, kp, vp, pages, lens, cu)
        ops.paged_attn_raw(q, kp, vp, pages, lens, cu // 4, 10, 16)
        ops.paged_attn_raw(q, kp, vp, pages, lens, cu, 40, 16)
        process_logits(torch.randn(2, 3, 100, device="cuda"))
        got = {k: n for k, (ms, n) in ops.profile_collect().items() if ms > 0}
    finally:
        ops.profile_enable(False)
    assert_device_ok()
    assert got == {"qkv_rope_paged": 1, "paged_attn": 2, "process_logits": 1}


def test_a_captured_step_serves_growing_sequences(model):
    """One denoising forward captured in a CUDA graph, replayed block after block as begin()
    advances the lengths and hands out pages."""
    from workloads.serving import PagedGeneration
    g = torch.Generator().manual_seed(4)
    seqs = [torch.randint(0, V - 1, (96,), generator=g).cuda() for _ in range(2)]
    gen = PagedGeneration(model, 2, 128, 20, page_size=16)
    ids = [gen.cache.add() for _ in seqs]
    block = torch.zeros(2 * BS, dtype=torch.int64, device="cuda")
    graph, logits, got = torch.cuda.CUDAGraph(), None, []
    with torch.no_grad():
        for b in range(6):
            gen.cache.begin({i: BS for i in ids})
            block.copy_(torch.cat([s[b * BS:(b + 1) * BS] for s in seqs]))
            if b == 0:
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    gen.forward(block)
                torch.cuda.current_stream().wait_stream(side)
                with torch.cuda.graph(graph):
                    logits = gen.forward(block)
            graph.replay()
            gen.cache.commit()
            got.append(logits.view(2, BS, -1).clone())
        assert_device_ok()
        for i, s in enumerate(seqs):
            ref = full_logits(model, s)
            err = (torch.cat([x[i] for x in got]).float() - ref).abs().max().item()
            assert err <= 0.03 * max(1.0, ref.abs().max().item()), (i, err)


def test_padding_rows_and_a_step_without_new_tokens():
    """More rows than the step has tokens: the rest is in no sequence; a step of no tokens at all
    writes nothing and reports nothing."""
    from bd3attn.paged_cache import PagedKVCache
    cache = PagedKVCache(1, 2, 8, 2, 64, page_size=16)
    a = cache.add()
    tab = torch.ones(64, 32, device="cuda")
    qkv = torch.randn(8, 8 * 64, device="cuda").bfloat16()
    for n in (5, 0):
        cache.begin({a: n})
        before = cache.v[0].clone()
        q = cache.rope_qkv(0, qkv, 4, tab, tab)
        o, lse = cache.attend(0, q, 1, return_lse=True)
        assert o.shape == (8, 4, 64) and torch.isfinite(o[:n]).all() and torch.isfinite(lse[:n]).all()
        assert int((cache.v[0] != before).flatten(1).any(1).sum()) == (n > 0)
        cache.commit()
    assert_device_ok()


def test_a_step_captured_on_a_new_cache_leaves_eager_calls_right():
    """The first attention of a cache may be the one that a graph captures: an eager call before
    the first replay, the replay and a call after it all give the same bits."""
    from bd3attn import ops
    from bd3attn.paged_cache import PagedKVCache

    def new():
        cache = PagedKVCache(1, 2, 128, 1, 2048, page_size=16)
        a = cache.add()
        cache.begin({a: 1984})
        cache.commit()
        cache.begin({a: 16})
        for x in (cache.k[0], cache.v[0]):
            x.normal_(generator=torch.Generator("cuda").manual_seed(5))
        return cache

    q = torch.randn(16, 4, 64, device="cuda").bfloat16()
    new().attend(0, -q, 16)  # the library's own first call
    first, graph = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):  # an earlier graph of the same pool leaves its memory as it used it
        junk = torch.full((1 << 28,), 0xA5, dtype=torch.uint8, device="cuda")
    first.replay()
    del junk
    cache = new()
    with torch.cuda.graph(graph, pool=first.pool()):
        out = cache.attend(0, q, 16)
    eager = cache.attend(0, q, 16).clone()
    graph.replay()
    after = cache.attend(0, q, 16)
    ref = ops.paged_attn_raw(q, cache.k[0], cache.v[0], cache.page_table, cache.kv_lens, cache.cu_q, 16, 16)
    assert_device_ok()
    assert torch.equal(eager, ref) and torch.equal(out, ref) and torch.equal(after, ref)


def test_every_way_out_of_a_run_returns_its_sequences(model):
    """Sequences of no blocks, a request past max_len, a pool that runs out, more prompts than
    sequences, a backbone that fails in mid-step: pages and places are back each time."""
    from workloads.serving import PagedGeneration
    g = torch.Generator().manual_seed(6)
    gen = PagedGeneration(model, 3, 128, 20, page_size=16, steps=2, chunk=32)

    def prompts(*lens):
        return [torch.randint(0, V - 1, (n,), generator=g).cuda() for n in lens]

    def free():
        for s in [gen.cache.add() for _ in range(3)]:
            gen.cache.release(s)
        return gen.cache.free_pages == 20

    assert [len(o) for o in gen.run(prompts(32, 16, 0), [0, 1, 0])] == [0, 16, 0]
    assert free()
    for lens, blocks in (((112, 16), [2, 1]), ((112, 112, 112), [1, 1, 1]), ((16,) * 4, [1] * 4), ((16, 16), [1])):
        with pytest.raises((RuntimeError, IndexError)):
            gen.run(prompts(*lens), blocks)
        assert free(), (lens, blocks)
    forward, calls = gen.forward, []

    def failing(*a, **kw):
        calls.append(1)
        if len(calls) == 3:
            raise ValueError("a step that fails")
        return forward(*a, **kw)

    gen.forward = failing
    with pytest.raises(ValueError, match="a step that fails"):
        gen.run(prompts(32, 16), [2, 2])
    gen.forward = forward
    assert free()
    assert [len(o) for o in gen.run(prompts(96, 16, 0), [1, 2, 3])] == [16, 32, 48]
    assert free()
    assert_device_ok()
