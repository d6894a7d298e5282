"""PagedKVCache's bookkeeping on the CPU: pages taken and given back, provisional and committed
positions, what the device's tables hold, and its refusals."""

import pytest
import torch

from bd3attn.paged_cache import PagedKVCache


def cache(**kw):
    args = dict(n_layers=2, n_kv_heads=3, num_pages=10, max_seqs=3, max_len=64, page_size=16,
                device="cpu")
    return PagedKVCache(**{**args, **kw})


def test_tables_lengths_and_pages():
    c = cache()
    a, b = c.add(), c.add()
    c.begin({a: 17, b: 16})
    assert c.free_pages == 7 and (c.max_new, c.tokens) == (17, 33)
    assert c.cu_q.tolist() == [0, 17, 33, 33] and c.kv_lens.tolist() == [17, 16, 0]
    pages_a, page_b = c.page_table[0, :2].tolist(), c.page_table[1, 0].item()
    assert len({*pages_a, page_b}) == 3
    c.commit()
    assert (c.length(a), c.length(b)) == (17, 16)
    c.begin({b: 1, a: 15})  # another order: a still fits its two pages, b needs a second
    assert c.page_table[1, :2].tolist() == pages_a and c.page_table[0, 0].item() == page_b
    assert c.cu_q.tolist() == [0, 1, 16, 16] and c.kv_lens.tolist() == [17, 32, 0]
    assert c.free_pages == 6
    c.begin({a: 4})  # never committed: starts from the committed 17 again
    assert c.kv_lens.tolist() == [21, 0, 0] and c.length(a) == 17
    c.commit()
    c.release(a)
    assert c.free_pages == 8  # b keeps the page it got for the step that was not committed
    d = c.add()
    c.begin({d: 64, b: 16})
    assert c.free_pages == 4
    used = c.page_table[0].tolist() + c.page_table[1, :2].tolist()
    assert len(set(used)) == 6


def test_a_sequence_may_have_no_new_tokens():
    c = cache()
    a, b = c.add(), c.add()
    c.begin({a: 0, b: 5})
    assert c.cu_q.tolist() == [0, 0, 5, 5] and c.kv_lens.tolist() == [0, 5, 0]
    c.begin({})
    assert c.tokens == c.max_new == 0 and c.cu_q.tolist() == [0] * 4


def test_refusals_change_nothing():
    c = cache()
    a = c.add()
    c.begin({a: 40})
    c.commit()
    with pytest.raises(RuntimeError, match="max_len"):
        c.begin({a: 25})
    b, d = c.add(), c.add()
    with pytest.raises(RuntimeError, match="holds 3"):
        c.add()
    with pytest.raises(RuntimeError, match="pages needed"):
        c.begin({b: 64, d: 64})
    assert c.free_pages == 7 and c.length(b) == 0
    with pytest.raises(ValueError):
        c.begin({a: -1})
    with pytest.raises(KeyError):
        c.begin({99: 1})
    for kw in (dict(page_size=12), dict(num_pages=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            cache(**kw)


def test_no_write_or_attention_outside_a_step():
    """Before the first begin() and after commit() nothing is new: the device still holds the last
    step's lengths, so both calls are refused; so are fewer rows than the step has."""
    c = cache()
    a = c.add()
    qkv, q, tab = torch.zeros(5, 12 * 64), torch.zeros(5, 6, 64), torch.ones(64, 32)

    def refused(kind, match, rows=5):
        with pytest.raises(kind, match=match):
            c.rope_qkv(0, qkv[:rows], 6, tab, tab)
        with pytest.raises(kind, match=match):
            c.attend(0, q[:rows], 1)

    refused(RuntimeError, "begin")
    c.begin({a: 5})
    refused(AssertionError, "5 new tokens", 4)
    c.commit()
    refused(RuntimeError, "begin")
    assert c.length(a) == 5
    with pytest.raises(RuntimeError, match="max_len"):
        c.begin({a: 60})
    refused(RuntimeError, "begin")  # a refused begin() opens nothing
    c.begin({a: 4})
    with pytest.raises(RuntimeError, match="max_len"):
        c.begin({a: 60})
    refused(AssertionError, "4 new tokens", 3)  # and leaves an open step as it is


def test_release_in_a_step_leaves_the_others_in_it():
    """A sequence that ends in mid-step takes its pages and nothing else along: the packed rows stay
    as they are and the others commit."""
    c = cache()
    a, b = c.add(), c.add()
    c.begin({a: 17, b: 20})
    c.release(a)
    assert c.free_pages == 8 and (c.max_new, c.tokens) == (20, 37)
    assert c.cu_q.tolist() == [0, 17, 37, 37]
    with pytest.raises(AssertionError, match="37 new tokens"):
        c.attend(0, torch.zeros(20, 6, 64), 1)
    c.commit()
    assert c.length(b) == 20
    with pytest.raises(KeyError):
        c.length(a)
    c.begin({b: 3})
    c.release(b)
    assert c.free_pages == 10
    c.commit()  # nothing is left in the step
    d = c.add()
    c.begin({d: 16})
    assert c.kv_lens.tolist() == [16, 0, 0] and c.free_pages == 9
