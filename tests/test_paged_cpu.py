"""The paged cache without a GPU: the books of its pages, and every refusal that comes before a
CUDA call."""
import ctypes
import random

import pytest
import torch

from drofell_for_revision_b200 import _capi, paged

INVALID, UNSUPPORTED, OK = _capi.W4A16_ERR_INVALID, _capi.W4A16_ERR_UNSUPPORTED, _capi.W4A16_OK
FAKE = 0x10000


def pages(**kw):
    d = dict(k_dev=FAKE, v_dev=FAKE, stride_page=4096, stride_head=2048, stride_token=128, num_pages=4, heads_kv=2,
             page_size=16, head_dim=128, dtype=0, device=0)
    d.update(kw)
    return _capi.Pages(**d)


def seqs(**kw):
    d = dict(tables_dev=FAKE, lens_dev=FAKE, cu_q_dev=None, table_stride=4, table_width=4, batch=2, tokens=2, max_q=1)
    d.update(kw)
    return _capi.Seqs(**d)


def rows(**kw):
    d = dict(dev=FAKE, stride_token=1024, stride_head=128)
    d.update(kw)
    return _capi.Rows(**d)


def attention(p=None, s=None, q=None, out=None, heads=4, scale=0.1, window=0, sinks=0, ws=None, n=0):
    ref = lambda x: ctypes.byref(x) if x is not None else None  # noqa: E731
    return _capi.lib().w4a16_paged_attention(ref(p or pages()), ref(s or seqs()), ref(q or rows()),
                                             ref(out or rows(dev=2 * FAKE)), heads, scale, window, sinks, ws, n, None)


def append(p=None, s=None, k=None, v=None, q=None, q_out=None, heads=4, rope=None, positions=0, dim=0, inter=0):
    ref = lambda x: ctypes.byref(x) if x is not None else None  # noqa: E731
    return _capi.lib().w4a16_append_kv(ref(p or pages()), ref(s or seqs()), ref(k or rows()), ref(v or rows()), ref(q),
                                       ref(q_out), heads, rope, positions, dim, inter, None)


@pytest.mark.parametrize("kw,code", [
    (dict(k_dev=None), INVALID), (dict(v_dev=None), INVALID), (dict(dtype=2), INVALID), (dict(k_dev=FAKE + 8), INVALID),
    (dict(page_size=4), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED), (dict(page_size=512), UNSUPPORTED),
    (dict(head_dim=132), UNSUPPORTED), (dict(head_dim=136), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED),
    (dict(stride_token=100), INVALID), (dict(stride_page=-8), INVALID), (dict(num_pages=0), INVALID),
    (dict(heads_kv=0), INVALID), (dict(stride_head=0), INVALID), (dict(stride_token=0), INVALID)])
def test_pages_are_checked(kw, code):
    assert attention(p=pages(**kw)) == code
    assert append(p=pages(**kw)) == code
    assert _capi.lib().w4a16_paged_attention_workspace_size(ctypes.byref(pages(**kw)), ctypes.byref(seqs()), 4, 0, 0) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(tables_dev=None), INVALID), (dict(lens_dev=None), INVALID), (dict(batch=-1), INVALID), (dict(tokens=3), INVALID),
    (dict(table_width=-1), INVALID), (dict(max_q=-1), INVALID), (dict(table_width=1 << 28), UNSUPPORTED),
    (dict(cu_q_dev=FAKE, tokens=1 << 30), UNSUPPORTED)])
def test_sequences_are_checked(kw, code):
    assert attention(s=seqs(**kw)) == code
    assert append(s=seqs(**kw)) == code


def test_attention_arguments_are_checked():
    assert attention(heads=3) == INVALID
    assert attention(heads=0) == INVALID
    assert attention(window=-1) == INVALID
    assert attention(window=4, sinks=-1) == INVALID
    assert attention(sinks=4) == INVALID
    assert b"sinks" in _capi.lib().w4a16_last_error()
    for scale in (float("nan"), float("inf"), 0.0, -0.1):
        assert attention(scale=scale) == INVALID
    assert attention(q=rows(dev=None)) == INVALID
    assert attention(out=rows(stride_head=4)) == INVALID
    assert attention(out=rows(dev=FAKE + 2)) == INVALID
    assert attention(out=rows(dev=FAKE)) == INVALID  # q itself
    assert attention(s=seqs(cu_q_dev=FAKE, max_q=(1 << 31) - 1, tokens=5)) == UNSUPPORTED
    assert _capi.lib().w4a16_paged_error(0, None, None) == INVALID
    # nothing to do: no CUDA call
    assert attention(s=seqs(batch=0, tokens=0)) == OK
    assert attention(s=seqs(cu_q_dev=FAKE, tokens=0)) == OK


def test_append_arguments_are_checked():
    assert append(k=rows(dev=None)) == INVALID
    assert append(v=rows(stride_token=12)) == INVALID
    assert append(q=rows(), q_out=None) == INVALID
    assert append(q=rows(), q_out=rows(), heads=0) == INVALID
    assert append(rope=FAKE, positions=63, dim=128) == INVALID  # tables of 64 tokens
    assert append(rope=FAKE, positions=64, dim=136) == UNSUPPORTED
    assert append(rope=FAKE, positions=64, dim=24) == UNSUPPORTED
    assert append(rope=FAKE, positions=64, dim=20, inter=1) == UNSUPPORTED
    assert append(rope=FAKE + 4, positions=64, dim=128) == INVALID
    assert append(s=seqs(batch=0, tokens=0)) == OK


@pytest.mark.parametrize("kw", [dict(stride_token=0), dict(stride_head=0), dict(stride_token=384), dict(stride_head=64),
                                dict(stride_token=128, stride_head=128)])
def test_rows_that_are_written_must_not_overlap(kw):
    assert attention(out=rows(dev=2 * FAKE, **kw)) == INVALID
    assert append(q=rows(), q_out=rows(**kw)) == INVALID
    assert b"overlap" in _capi.lib().w4a16_last_error()


def test_pages_that_are_written_must_not_overlap():
    for kw in (dict(stride_page=2048), dict(stride_head=1024), dict(stride_token=64)):
        assert append(p=pages(**kw)) == INVALID
        assert b"overlap" in _capi.lib().w4a16_last_error()


def copy(src, dst, k=FAKE, stride_layer=1 << 20, stride_page=4096, layers=2, num=10, size=4096):
    n = len(src)
    arr = lambda x: (ctypes.c_int * n)(*x)  # noqa: E731
    return _capi.lib().w4a16_copy_pages(k, FAKE, stride_layer, stride_page, layers, num, size, arr(src), arr(dst), n, 0,
                                        None)


def test_copy_refuses_what_has_no_order():
    assert copy([1, 2], [3, 3]) == INVALID  # written twice
    assert copy([1, 3], [3, 4]) == INVALID  # written, then read
    assert copy([3, 1], [4, 3]) == INVALID  # read, then written
    assert copy([1], [1]) == INVALID
    assert copy([10], [1]) == INVALID and copy([1], [-1]) == INVALID
    assert copy([1], [2], size=4104) == INVALID
    assert copy([1], [2], size=8192) == INVALID  # pages that overlap
    assert copy([1], [2], k=None) == INVALID
    assert copy([1], [2], layers=40000) == INVALID
    assert copy([], []) == OK


# ---------------------------------------------------------------- the torch entry points
def tensors(heads=4, hkv=2, dim=64, page=16, dtype=torch.float16, batch=2):
    k, v = (torch.zeros(6, hkv, page, dim, dtype=dtype) for _ in range(2))
    return dict(q=torch.zeros(batch, heads, dim, dtype=dtype), k_pages=k, v_pages=v,
                tables=torch.zeros(batch, 3, dtype=torch.int32), lens=torch.zeros(batch, dtype=torch.int32))


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(2, 4, 32, dtype=torch.float16)), "must be"),
    (dict(q=torch.zeros(2, 4, 64)), "type"),
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float16)), "one new token"),
    (dict(v_pages=torch.zeros(6, 2, 8, 64, dtype=torch.float16)), "same strides"),
    (dict(tables=torch.zeros(2, 3, dtype=torch.int64)), "int32"),
    (dict(tables=torch.zeros(3, 2, dtype=torch.int32).T), "contiguous"),
    (dict(lens=torch.zeros(3, dtype=torch.int32)), "sequences"),
    (dict(cu_q=torch.zeros(2, dtype=torch.int32), max_q=2), "offsets"),
    (dict(window=-1), "non-negative"),
    (dict(), "CUDA tensor"),
])
def test_attention_refusals(change, match):
    a = dict(tensors(), **change)
    with pytest.raises(RuntimeError, match=match):
        paged.attention(a.pop("q"), a.pop("k_pages"), a.pop("v_pages"), a.pop("tables"), a.pop("lens"), **a)


def test_gradients_are_refused():
    a = tensors()
    q = a.pop("q").requires_grad_()
    with pytest.raises(RuntimeError, match="requires a gradient"):
        paged.attention(q, **a)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):
        paged.attention(q, **a)


@pytest.mark.parametrize("change,match", [
    (dict(k=torch.zeros(2, 3, 64, dtype=torch.float16)), "k must be"),
    (dict(v=torch.zeros(2, 2, 64, dtype=torch.bfloat16)), "type"),
    (dict(rope=torch.zeros(48, 64, dtype=torch.float64)), "float32"),
    (dict(q_out=torch.zeros(2, 4, 64, dtype=torch.float16)), "without q"),
    (dict(), "CUDA tensor"),
])
def test_append_refusals(change, match):
    a = tensors()
    a.pop("q")
    a.update(k=torch.zeros(2, 2, 64, dtype=torch.float16), v=torch.zeros(2, 2, 64, dtype=torch.float16))
    a.update(change)
    with pytest.raises(RuntimeError, match=match):
        paged.append_kv(**a)


def test_copy_refusals():
    k = torch.zeros(3, 6, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        paged.copy_pages(k, k.clone(), [1], [2])
    with pytest.raises(RuntimeError, match="source pages"):
        paged.copy_pages(k, k.clone(), [1], [2, 3])
    with pytest.raises(RuntimeError, match="one block"):
        paged.copy_pages(k[..., :32], k.clone()[..., :32], [1], [2])
    for big in (torch.tensor([1 << 32]), [1 << 32], [-1], torch.tensor([-1])):
        with pytest.raises(RuntimeError, match="32 bits"):
            paged.copy_pages(k, k.clone(), big, [2])
    with pytest.raises((RuntimeError, TypeError)):
        paged.copy_pages(k, k.clone(), [1.5], [2])
    with pytest.raises(RuntimeError, match="source pages"):
        paged.copy_pages(k, k.clone(), (1, 2), torch.tensor([2]))
    with pytest.raises(RuntimeError, match="whole numbers"):
        paged.copy_pages(k, k.clone(), torch.tensor([1.5]), [2])


# ---------------------------------------------------------------- the books
def test_pool_extends_forks_and_frees():
    pool = paged.PagePool(8, 4)
    assert pool.extend("a", 6) == ([], []) and pool.pages("a") == (0, 1) and pool.length("a") == 6
    pool.fork("a", "b")
    assert pool.free_pages == 6
    assert pool.extend("b", 1) == ([1], [2])  # the shared, partly filled page becomes b's own
    assert pool.pages("b") == (0, 2) and pool.pages("a") == (0, 1)
    assert pool.extend("a", 1) == ([], [])  # nobody shares it any more
    pool.free("a")
    assert pool.free_pages == 6 and pool.pages("b") == (0, 2)
    pool.truncate("b", 4)
    assert pool.pages("b") == (0,) and pool.free_pages == 7
    pool.fork("b", "c")
    assert pool.extend("c", 3) == ([], [])  # a full shared page is not written
    with pytest.raises(RuntimeError, match="pages needed"):
        pool.extend("c", 100)
    assert pool.length("c") == 7
    with pytest.raises(RuntimeError, match="exists"):
        pool.fork("b", "c")
    with pytest.raises(RuntimeError):
        pool.truncate("c", 8)
    tables, lens = pool.tables(["c", "b"], device=torch.device("cpu"))
    assert tables.tolist() == [[0, 1], [0, -1]] and lens.tolist() == [7, 4]
    with pytest.raises(RuntimeError, match="tables of 1"):
        pool.tables(["c"], width=1)
    assert pool.tables([], device=torch.device("cpu"))[0].shape == (0, 0)


def test_pool_against_a_plain_model():
    """Random calls; what each sequence reads through the pages is what a list per sequence holds."""
    for seed in range(30):
        r = random.Random(seed)
        size = r.choice([1, 3, 4])
        pool, store, truth = paged.PagePool(40, size), {}, {}
        names = iter(range(10 ** 6))

        def move(pairs):
            assert len(set(pairs[1])) == len(pairs[1]) and not set(pairs[0]) & set(pairs[1])
            old = dict(store)
            for s, d in zip(*pairs):
                for i in range(size):
                    store[d, i] = old.get((s, i))
        for step in range(200):
            what = r.random()
            if what < 0.5 or not truth:
                name = r.choice(list(truth) + [next(names)])
                n = r.randint(0, 9)
                try:
                    move(pool.extend(name, n))
                except RuntimeError:
                    assert pool.free_pages < n // size + 3
                    continue
                for _ in range(n):
                    at = len(truth.setdefault(name, []))
                    store[pool.pages(name)[at // size], at % size] = step * 100 + at
                    truth[name].append(step * 100 + at)
                truth.setdefault(name, [])
            elif what < 0.65:
                old, new = r.choice(list(truth)), next(names)
                pool.fork(old, new)
                truth[new] = list(truth[old])
            elif what < 0.8:
                name = r.choice(list(truth))
                pool.free(name)
                del truth[name]
            elif what < 0.9:
                name = r.choice(list(truth))
                n = r.randint(0, len(truth[name]))
                pool.truncate(name, n)
                del truth[name][n:]
            else:
                move(pool.compact())
                used = {p for s in truth for p in pool.pages(s)}
                assert used == set(range(len(used)))
            used = {p for s in truth for p in pool.pages(s)}
            assert pool.free_pages == 40 - len(used)
            for name, want in truth.items():
                assert pool.length(name) == len(want)
                assert [store[pool.pages(name)[i // size], i % size] for i in range(len(want))] == want
