"""Refusals of the paged cache before any CUDA call. Memory that two operands share is refused, and
only that: against a search through all elements.

A call that passes its checks would go on to the GPU: the cases that have to be accepted end in
a later refusal, or are asked of the search alone."""
import ctypes
import itertools
import math
import random
import time

import numpy
import pytest
import torch

from drofell_for_revision_b200 import _capi, paged
from test_paged_cpu import FAKE, INVALID, append, attention, copy, pages, rows, seqs


def message():
    return _capi.lib().w4a16_last_error().decode()


def elements(r, tokens, heads, dim):
    return {r.dev // 2 + t * r.stride_token + h * r.stride_head + d for t in range(tokens) for h in range(heads)
            for d in range(dim)}


def accepts_attention(q, out, tokens, heads):
    """Whether q and out pass: the workspace is checked behind them, and there is none."""
    p = pages(head_dim=8, stride_token=8, stride_head=128, stride_page=256)
    rc = attention(p=p, s=seqs(cu_q_dev=FAKE, tokens=tokens, max_q=1), q=q, out=out, heads=heads)
    assert rc != _capi.W4A16_OK
    return "overlap" not in message()


def test_out_must_not_overlap_q():
    assert attention(out=rows(dev=FAKE + 16)) == INVALID and "overlap" in message()
    assert attention(out=rows(dev=FAKE + 2048)) == INVALID and "overlap" in message()  # the next token's rows
    assert attention(q=rows(dev=2 * FAKE + 1024 * 2), out=rows(dev=2 * FAKE)) == INVALID and "overlap" in message()


def test_views_of_one_buffer_against_a_search():
    """q and out anywhere in a buffer, with the buffer's strides or others: what shares an element is
    refused; what does not is accepted wherever the token strides agree."""
    r = random.Random(5)
    seen = set()
    for _ in range(3000):
        tokens, heads, dim = r.choice([1, 2, 5]), 2 * r.choice([1, 2, 3]), 8
        wide = r.choice([heads, heads + 1, 2 * heads, 3 * heads]) * dim
        q = rows(dev=FAKE + 16 * r.randrange(0, 60), stride_token=wide, stride_head=dim)
        out = rows(dev=FAKE + 16 * r.randrange(0, 60), stride_token=wide, stride_head=dim)
        if r.random() < 0.3:
            q.stride_head = r.choice([0, 8, 16, 8 * tokens])
        if r.random() < 0.2:
            q.stride_token = r.choice([0, 8, wide + 8])
        if r.random() < 0.2:  # heads outside
            out.stride_token, out.stride_head = dim, dim * tokens
            if r.random() < 0.5:
                q.stride_token, q.stride_head = dim, dim * tokens
        meet = bool(elements(q, tokens, heads, dim) & elements(out, tokens, heads, dim))
        ok = accepts_attention(q, out, tokens, heads)
        assert not (meet and ok), (tokens, heads, q.dev, out.dev)
        if tokens == 1 or q.stride_token == out.stride_token:
            assert ok == (not meet)
        seen.add((meet, ok))
    assert seen >= {(True, False), (False, True)}


def test_q_out_must_be_q_or_lie_apart():
    far = dict(k=rows(dev=4 * FAKE, stride_token=256), v=rows(dev=5 * FAKE, stride_token=256))
    p = pages(v_dev=64 * FAKE, k_dev=32 * FAKE)
    for kw in (dict(dev=FAKE + 16), dict(dev=FAKE + 2048), dict(dev=FAKE, stride_token=2048)):
        assert append(p=p, q=rows(), q_out=rows(**kw), **far) == INVALID and "q_out must be q" in message(), kw
    assert append(p=p, q=rows(), q_out=rows(dev=4 * FAKE - 256), **far) == INVALID and "k or v" in message()
    assert append(p=p, q=rows(), q_out=rows(dev=5 * FAKE + 16), **far) == INVALID and "k or v" in message()


def test_k_and_v_pages_must_lie_apart():
    for v in (FAKE, FAKE + 16, FAKE + 128 * 2, FAKE + 4096 * 2, FAKE - 4096 * 2 * 3):
        assert append(p=pages(v_dev=v)) == INVALID and "K and V" in message(), hex(v)


def pages_share(delta, strides, counts, size):
    for x in itertools.product(*(range(1 - n, n) for n in counts)):
        if abs(delta + sum(a * b for a, b in zip(x, strides))) < size:
            return True
    return False


def test_k_and_v_pages_against_a_search():
    """K and V as parts of one tensor in whatever order of its dimensions."""
    r = random.Random(7)
    seen = set()
    for _ in range(2000):
        counts, dim, strides, left = [3, 2, 8], 8, [0, 0, 0], 8 * 2
        for i in r.sample(range(3), 3):  # K and V may lie beside one another at any level
            left *= r.choice([1, 1, 2])
            strides[i] = left
            left *= counts[i]
        delta = 16 * r.randrange(-left // 16 - 2, left // 16 + 2)
        meet = pages_share(delta, strides, counts, dim * 2)
        p = pages(k_dev=FAKE * 16, v_dev=FAKE * 16 + delta, stride_page=strides[0] // 2, stride_head=strides[1] // 2,
                  stride_token=strides[2] // 2, num_pages=3, heads_kv=2, page_size=8, head_dim=8)
        # accepted, the call ends at q_out, which lies on k
        k, q_out = rows(dev=2 * FAKE, stride_head=8), rows(dev=2 * FAKE + 16, stride_head=8)
        assert append(p=p, k=k, v=rows(dev=3 * FAKE), q=rows(dev=4 * FAKE), q_out=q_out) == INVALID
        assert ("K and V" in message()) == meet, (strides, delta)
        seen.add(meet)
    assert seen == {True, False}


def test_copies_of_pages_that_overlap():
    def call(v, stride_layer=1 << 20, layers=2, num=10):
        ids = (ctypes.c_int * 1)(0)
        # accepted, the call ends at a copy of a page onto itself
        return _capi.lib().w4a16_copy_pages(FAKE, v, stride_layer, 4096, layers, num, 4096, ids, ids, 1, 0, None)
    assert copy([1], [2], stride_layer=0) == INVALID and "overlap" in message()
    assert copy([1], [2], stride_layer=4096) == INVALID and "overlap" in message()
    assert copy([1], [2], stride_layer=9 * 4096) == INVALID and "overlap" in message()
    for v, stride, bad in ((FAKE, 40960, False), (FAKE + 16, 40960, True), (FAKE + 4096, 40960, True),
                           (FAKE + 40960, 40960, True), (FAKE + 2 * 40960, 40960, False), (FAKE + 40960, 81920, False),
                           (FAKE - 2 * 40960, 40960, False), (FAKE - 4096, 40960, True)):
        assert call(v, stride) == INVALID
        assert ("K and V" in message()) == bad, (v - FAKE, stride)


@pytest.mark.parametrize("layers,stride_layer,stride_page,bad", [(4, 4096, 4 * 4096, False), (4, 4096, 3 * 4096, True),
                                                                 (4, 2048, 5 * 4096, True), (1, 0, 4096, False)])
def test_layers_inside_pages(layers, stride_layer, stride_page, bad):
    ids = (ctypes.c_int * 1)(0)
    assert _capi.lib().w4a16_copy_pages(FAKE, FAKE, stride_layer, stride_page, layers, 5, 4096, ids, ids, 1, 0, None) == INVALID
    assert ("overlap" in message()) == bad


# ---------------------------------------------------------------- the ids of a copy
def test_copies_cost_what_they_copy():
    """The checks of two copies take no longer, and no more memory, in a cache of 2^31 - 1 pages."""
    best = math.inf
    for _ in range(5):
        start = time.perf_counter()
        assert copy([1, 2], [3, 3], num=(1 << 31) - 1, size=16, stride_page=16, layers=1) == INVALID
        best = min(best, time.perf_counter() - start)
    assert "written twice" in message()
    assert best < 0.005


@pytest.mark.parametrize("num", [10, 1000])  # as many pages as copies, and many more
def test_copies_against_sets(num):
    r = random.Random(11)
    seen = set()
    for _ in range(2000):
        n = r.randrange(1, 7)
        src, dst = [r.randrange(-1, 11) for _ in range(n)], [r.randrange(0, 10) for _ in range(n)]
        if min(src) >= 0 and max(src) < num and len(set(dst)) == n and not set(src) & set(dst):
            continue  # would be launched
        assert copy(src, dst, num=num, stride_page=4096, stride_layer=1 << 30) == INVALID
        want = ("pages" if min(src) < 0 or max(src) >= num else "written twice" if len(set(dst)) < n else "read and written")
        assert want in message()
        seen.add(want)
    assert len(seen) == 3


def test_ids_that_are_not_whole_are_refused():
    """Whatever holds them: none is rounded."""
    k = torch.zeros(3, 6, 2, 16, 64, dtype=torch.float16)
    for bad in ((1.5,), numpy.array([1.5]), (1.0,), numpy.array([2.0], dtype=numpy.float32)):
        for pair in ((bad, [2]), ([2], bad), ((2,), bad)):
            with pytest.raises(RuntimeError, match="whole numbers"):
                paged.copy_pages(k, k.clone(), *pair)
    for good in ((1,), range(1, 2), numpy.array([1]), numpy.array([1], dtype=numpy.uint8), torch.tensor([1])):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            paged.copy_pages(k, k.clone(), good, (2,))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        paged.copy_pages(k, k.clone(), (), [])


@pytest.mark.parametrize("which", ["x", "layernorm"])
def test_the_block_refuses_gradients(which):
    """Its result would carry none, whatever was asked."""
    a = dict(x=torch.zeros(1, 8, dtype=torch.float16), layernorm=torch.ones(8, dtype=torch.float16))
    a[which].requires_grad_()
    k = torch.zeros(2, 1, 8, 8, dtype=torch.float16)
    tables, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)

    def call():
        paged.attention_forward(a["layernorm"], 1e-6, 12345, 12345, 12345, 12345, a["x"], k, k.clone(), tables, lens)
    with pytest.raises(RuntimeError, match=f"{which} requires a gradient"):
        call()
    with torch.no_grad(), pytest.raises(RuntimeError, match="unknown or released"):
        call()
