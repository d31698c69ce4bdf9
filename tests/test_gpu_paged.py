"""The paged key-value cache on a B200 against plain 64-bit implementations: filling, attention
of single tokens and of prompts (windows, sinks, uneven lengths, empty rows), copying pages.

Tolerances. Outputs are compared element by element with the 64-bit result of the same inputs:
 * the output's rounding is at most half a step, eps / 2 relative;
 * weights enter the value product rounded to the 16-bit type where a kernel says so, at most
   eps / 2 relative each (nothing where it keeps two parts);
 * fp32 sums over n keys, and the fp32 score's error amplified by the exponential, are bounded
   far below that for the sizes here: n 2^-24 and |score| 2^-22.
So |out - exact| <= (eps / 2) |out| + (eps / 2) sum_j p_j |v_j| + 1e-5 max |v| with p the exact
weights: the first and second term are added whole, whatever their signs.
"""
import math

import pytest
import torch

from drofell_for_revision_b200 import paged

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    assert paged.device_error(DEV) == 0


class Batch:
    """Sequences of given (length, new tokens) with pages in random order."""

    def __init__(self, lens, new, heads, heads_kv, dim, page, dtype, seed=0, layout="hsd", extra=3):
        g = torch.Generator(device="cpu").manual_seed(seed)
        self.lens_l, self.new_l, self.page = list(lens), list(new), page
        used = [-(-n // page) for n in lens]
        pages = sum(used) + extra
        order = torch.randperm(pages, generator=g)[:sum(used)].tolist()
        width = max(used + [1])
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.tables = table.to(DEV)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        self.cu_l = cu
        self.cu_q = None if all(n == 1 for n in new) else torch.tensor(cu, dtype=torch.int32, device=DEV)
        self.max_q = max(new + [0])

        def normal(*shape):
            return torch.randn(*shape, generator=g).to(dtype).to(DEV)
        if layout == "hsd":
            self.k, self.v = (normal(pages, heads_kv, page, dim) for _ in range(2))
        else:  # [pages, slot, head, dim] seen as [pages, head, slot, dim]
            self.k, self.v = (normal(pages, page, heads_kv, dim).transpose(1, 2) for _ in range(2))
        self.q = normal(cu[-1], heads, dim)

    def keys(self, b, x):
        """Sequence b's tokens of k or v, [heads_kv, length, dim] in 64 bits."""
        n = self.lens_l[b]
        ids = self.tables[b, :-(-n // self.page)].long()
        return x[ids].transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n].transpose(0, 1).double()


def exact_attention(bt, scale, window, sinks, hide=None):
    """(out, sum_j p_j |v_j|) in 64 bits, every masked key left out by selection."""
    heads, hkv = bt.q.shape[1], bt.k.shape[1]
    out = torch.zeros(bt.q.shape, dtype=torch.float64, device=DEV)
    spread = torch.zeros_like(out)
    for b, (n, m) in enumerate(zip(bt.lens_l, bt.new_l)):
        if m == 0 or n == 0:
            continue
        k, v = bt.keys(b, bt.k), bt.keys(b, bt.v)
        rows = slice(bt.cu_l[b], bt.cu_l[b] + m)
        p = torch.arange(n - m, n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)[None]
        seen = j <= p
        if window:
            seen &= (p - j < window) | (j < sinks)
        if hide is not None:
            seen &= ~hide[b].to(DEV)[None]
        for h in range(heads):
            s = bt.q[rows, h].double() @ k[h * hkv // heads].T * scale
            s = torch.where(seen, s, -math.inf)
            top = s.amax(-1, keepdim=True)
            w = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
            vv = v[h * hkv // heads]
            if torch.isfinite(vv).all():
                out[rows, h] = w @ vv
                spread[rows, h] = w @ vv.abs()
            else:
                prod = torch.where(seen[..., None], w[..., None] * vv[None], 0.0)
                out[rows, h] = prod.sum(1)
                spread[rows, h] = prod.abs().sum(1)
    return out, spread


def check_attention(bt, window=0, sinks=0, scale=None, out=None, hide=None):
    dim = bt.q.shape[2]
    got = paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=bt.max_q, scale=scale,
                          window=window, sinks=sinks, out=out)
    want, spread = exact_attention(bt, 1.0 / math.sqrt(dim) if scale is None else scale, window, sinks, hide)
    half = torch.finfo(got.dtype).eps / 2
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.double()[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)])
    top = max(1.0, float(torch.nan_to_num(bt.v, 0.0, 0.0, 0.0).abs().max()))
    room = half * want.abs() + half * spread + 1e-5 * top
    bad = finite & ((got.double() - want).abs() > room)
    assert not bad.any(), float(((got.double() - want).abs() / room)[finite].max())
    return got


TYPES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,heads_kv,dim,page", [(8, 8, 128, 16), (16, 2, 128, 64), (12, 4, 64, 8), (5, 1, 80, 32),
                                                     (40, 2, 96, 128), (3, 3, 8, 256), (6, 2, 120, 16)])
def test_decode_lengths(dtype, heads, heads_kv, dim, page):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 500, 1000, 4001]
    check_attention(Batch(lens, [1] * len(lens), heads, heads_kv, dim, page, dtype))


@pytest.mark.parametrize("lens", [[1], [7], [64], [128], [129], [3000], [20000], [50001, 3]])
def test_decode_alone(lens):
    check_attention(Batch(lens, [1] * len(lens), 16, 2, 128, 32, torch.bfloat16, seed=3))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (64, 4), (100, 70), (1000, 1), (1 << 30, 5), (4096, 0),
                                          (5, (1 << 31) - 1)])
def test_decode_window(window, sinks):
    lens = [1, 5, 64, 99, 100, 101, 170, 171, 1001, 3333]
    check_attention(Batch(lens, [1] * len(lens), 8, 4, 128, 16, torch.float16, seed=5), window, sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (7, 2), (130, 4)])
def test_few_tokens(dtype, window, sinks):
    check_attention(Batch([9, 300, 2, 1030, 64], [3, 4, 2, 1, 4], 16, 4, 128, 16, dtype, seed=7), window, sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,heads_kv,dim,page", [(4, 4, 128, 16), (16, 2, 128, 128), (14, 2, 64, 8), (6, 2, 96, 64),
                                                     (7, 1, 80, 256), (3, 3, 8, 32), (6, 2, 40, 16), (4, 1, 120, 8)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 3), (300, 200)])
def test_prompts(dtype, heads, heads_kv, dim, page, window, sinks):
    check_attention(Batch([1, 130, 128, 77, 700, 513], [1, 130, 128, 40, 333, 1], heads, heads_kv, dim, page, dtype,
                          seed=11), window, sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (600, 4)])
def test_long_chunk(window, sinks):
    check_attention(Batch([5000, 2049], [1500, 2049], 8, 4, 128, 64, torch.bfloat16, seed=13), window, sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,heads_kv,dim,lens,new,window,sinks", [
    (8, 8, 128, [4099], [65], 0, 0),            # few rows on a long context: keys cut among all SMs
    (16, 1, 64, [9000, 130], [129, 7], 0, 0),
    (5, 1, 128, [3000, 2500], [100, 2500], 0, 0),  # a group that does not divide a row tile
    (4, 2, 128, [6000], [300], 1500, 4),
    (2, 1, 96, [2100], [2100], 700, 0),         # rows that see nothing of a piece
    (32, 8, 64, [33000], [40], 0, 0),
])
def test_chunk_on_a_long_context(dtype, heads, heads_kv, dim, lens, new, window, sinks):
    check_attention(Batch(lens, new, heads, heads_kv, dim, 32, dtype, seed=43), window, sinks)


def test_many_row_tiles():
    """More row pairs than a few rounds of the SMs take, and uneven sequences among them."""
    check_attention(Batch([4100, 1, 900], [4000, 1, 700], 40, 40, 64, 64, torch.float16, seed=47))


def test_many_prompts():
    """More prompts than the threads that count them, some of no new token."""
    g = torch.Generator().manual_seed(2)
    new = torch.randint(0, 40, (300,), generator=g).tolist()
    new[7] = 180
    lens = [n + int(torch.randint(0, 90, (1,), generator=g)) for n in new]
    check_attention(Batch(lens, new, 4, 2, 64, 16, torch.bfloat16, seed=53))


def test_many_sequences():
    """More sequences than a CTA has threads, among them empty ones."""
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 60, (333,), generator=g).tolist()
    check_attention(Batch(lens, [1] * 333, 4, 2, 64, 8, torch.float16, seed=17))


def test_rows_that_see_nothing():
    """Length zero; more new tokens than the length: zeros, exactly."""
    bt = Batch([0, 40, 2], [1, 1, 1], 8, 8, 128, 16, torch.float16)
    got = check_attention(bt)
    assert (got[0] == 0).all()
    for new in (6, 200):
        bt = Batch([40, new], [1, new], 8, 8, 128, 16, torch.float16)
        bt.lens_l[1] = 3
        bt.lens[1] = 3
        got = paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=new)
        assert (got[1:new - 2] == 0).all()  # positions 3 - new .. -1
        assert torch.isfinite(got).all() and (got[new - 2:] != 0).any()


def test_rows_behind_the_last_sequence_stay():
    for new in (2, 150):
        bt = Batch([50, 200], [1, new], 8, 2, 128, 16, torch.bfloat16)
        q = torch.cat((bt.q, torch.full((9, 8, 128), math.nan, dtype=torch.bfloat16, device=DEV)))
        out = torch.full_like(q, 7.0)
        got = paged.attention(q, bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=new, out=out)
        assert got.data_ptr() == out.data_ptr()
        assert (out[new + 1:] == 7.0).all()
        want = paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=new)
        assert torch.equal(out[:new + 1], want)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new", [1, 4, 140])
def test_unwritten_slots_may_hold_anything(value, new):
    """Slots behind the length, pages of nobody, keys outside the window: NaN and infinities
    there change nothing."""
    lens = [200, 143, 333]
    bt = Batch(lens, [new] * 3, 8, 4, 128, 16, torch.float16, seed=19)
    clean = paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=new, window=150, sinks=3)
    k, v = bt.k.clone(), bt.v.clone()
    keep = torch.zeros(k.shape[0], 16, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            if j < 3 or j > n - new - 150:
                keep[int(bt.tables[b, j // 16]), j % 16] = True
    hide = ~keep.to(DEV)[:, None, :, None]
    bt.k.copy_(k.masked_fill(hide, value))
    bt.v.copy_(v.masked_fill(hide, value))
    got = paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=new, window=150, sinks=3)
    assert torch.equal(got, clean)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("new,old,window", [(4, 60, 0), (4, 60, 20), (4, 900, 0), (140, 60, 0), (140, 60, 64),
                                            (140, 2000, 0)])
def test_a_value_reaches_only_the_rows_that_see_it(value, new, old, window):
    bt = Batch([new + old], [new], 4, 2, 128, 16, torch.float16, seed=23)
    for j in (new + old - 3, old + 1, old + new // 2):
        bt.v[int(bt.tables[0, j // 16]), :, j % 16, 5] = value
    check_attention(bt, window)


@pytest.mark.parametrize("heads,dim,seed", [(2, 64, 0), (2, 128, 1), (6, 128, 2)])
def test_row_tiles_without_keys_among_others(heads, dim, seed):
    """Long runs of items in which a row tile, or both, has nothing to do, behind ones whose values
    that are not finite take it long: who has nothing to do must not run ahead."""
    g = torch.Generator().manual_seed(seed)
    kinds = [(200, 200), (50, 50), (0, 40), (30, 100), (160, 1), (0, 200)]
    pick = torch.randint(0, len(kinds), (1000,), generator=g).tolist()
    bt = Batch([kinds[i][0] for i in pick], [kinds[i][1] for i in pick], heads, 2, dim, 16, torch.bfloat16, seed=seed)
    for b, i in enumerate(pick):
        if i == 0:
            bt.v[int(bt.tables[b, 9]), :, 6, 5] = (math.nan, math.inf)[b & 1]
    check_attention(bt)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("what", ["q", "k", "v", "some v"])
@pytest.mark.parametrize("new,old", [(1, 3000), (4, 200), (150, 2000), (700, 0)])
def test_data_that_is_not_finite(value, what, new, old):
    """Results that are not finite by right come out so, and as fast as others within reason (a
    poisoned batch must not look like a hang)."""
    bt = Batch([new + old, 50], [new, 1], 8, 2, 128, 32, torch.bfloat16, seed=59)
    if what == "q":
        bt.q[0, 0] = value
    elif what == "k":
        bt.k.fill_(value)
    elif what == "v":
        bt.v.fill_(value)
    else:
        bt.v[:, 1, :, 3] = value
        bt.v[::2, 0, 5, 7] = -value
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=bt.max_q)
    start.record()
    got = paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=bt.max_q)
    end.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) < 200
    if what in ("q", "k"):
        # scores are then NaN or infinite: no weights to speak of, but rows of other queries stand
        assert torch.isnan(got[0, 0]).all() if value != value else True
        if what == "q":
            assert torch.isfinite(got[:, 1:]).all()
        elif value != value:
            assert torch.isnan(got).all()
    else:
        check_attention(bt)


def test_offsets_that_do_not_ascend():
    """Row offsets of any values: no access out of range, other sequences stand."""
    bt = Batch([60, 90, 40], [3, 5, 4], 4, 2, 64, 16, torch.float16, seed=61)
    kn = torch.randn(12, 2, 64, device=DEV).half()
    for cu in ([0, 9, 2, 12], [-5, 3, 8, 1 << 30], [7, 3, -1, 4], [12, 12, 12, 12], [1 << 30, 5, 5, -(1 << 31)]):
        cu_q = torch.tensor(cu, dtype=torch.int32, device=DEV)
        paged.append_kv(bt.k, bt.v, kn, kn, bt.tables, bt.lens, cu_q=cu_q, q=bt.q)
        for max_q in (5, 40, 300):
            assert paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=cu_q, max_q=max_q).shape == bt.q.shape
    torch.cuda.synchronize()
    check_attention(Batch([60, 90, 40], [3, 5, 4], 4, 2, 64, 16, torch.float16, seed=61))


def test_pages_that_are_no_pages():
    """Tokens of a page id out of range are not seen."""
    for new in (1, 3, 130):
        bt = Batch([500], [new], 8, 2, 128, 16, torch.bfloat16, seed=29)
        hide = torch.zeros(500, dtype=torch.bool)
        tables = bt.tables.clone()
        for at, bad in ((0, -1), (5, bt.k.shape[0]), (9, 2 ** 31 - 1), (10, -2 ** 31)):
            tables[0, at] = bad
            hide[at * 16:at * 16 + 16] = True
        good = bt.tables
        bt.tables = tables
        got = paged.attention(bt.q, bt.k, bt.v, tables, bt.lens, cu_q=bt.cu_q, max_q=new)
        bt.tables = good
        want, spread = exact_attention(bt, 1 / math.sqrt(128), 0, 0, hide=[hide])
        half = torch.finfo(torch.bfloat16).eps / 2
        assert ((got.double() - want).abs() <= half * (want.abs() + spread) + 5e-5).all()


def test_lengths_beyond_the_table_are_held_to_it():
    bt = Batch([64, 30], [1, 1], 8, 8, 128, 16, torch.float16)
    want = paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens)
    got = paged.attention(bt.q, bt.k, bt.v, bt.tables, torch.tensor([2 ** 31 - 1, 30], dtype=torch.int32, device=DEV))
    assert torch.equal(got, want)
    none = paged.attention(bt.q, bt.k, bt.v, bt.tables, torch.tensor([-5, 30], dtype=torch.int32, device=DEV))
    assert (none[0] == 0).all() and torch.equal(none[1], want[1])


def test_layouts_and_strides():
    """Token-major pages, q and out as slices of wider rows."""
    for new in ([1, 1], [130, 70]):
        bt = Batch([300, 77], new, 8, 2, 128, 16, torch.bfloat16, seed=31, layout="shd")
        check_attention(bt, 40, 2)
        wide = torch.randn(bt.q.shape[0], 24, 128, device=DEV).to(torch.bfloat16)
        wide[:, 4:12] = bt.q
        out = torch.zeros_like(wide)
        got = paged.attention(wide[:, 4:12], bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=bt.max_q,
                              out=out[:, 8:16])
        want = paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=bt.max_q)
        assert torch.equal(got, want) and (out[:, :8] == 0).all() and (out[:, 16:] == 0).all()


def test_scale_and_repeats():
    for new in (1, 200):
        bt = Batch([900, 200], [new, new], 8, 2, 128, 32, torch.float16, seed=37)
        one = check_attention(bt, scale=0.3)
        for _ in range(3):
            assert torch.equal(one, paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=new, scale=0.3))


def test_long_cache_offsets_pass_32_bits():
    """A cache of over 2^32 bytes and 2^31 elements a tensor: the last pages are read and written."""
    page, hkv, dim = 256, 8, 128
    pages = (1 << 31) // (page * hkv * dim) + 40
    k = torch.zeros(pages, hkv, page, dim, dtype=torch.float16, device=DEV)
    v = torch.zeros_like(k)
    ids = [pages - 1, 3, pages - 17]
    tables = torch.tensor([ids], dtype=torch.int32, device=DEV)
    n = 700
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    kn, vn = (torch.randn(n, hkv, dim, device=DEV, generator=g).half() for _ in range(2))
    q = torch.randn(n, 16, dim, device=DEV, generator=g).half()
    paged.append_kv(k, v, kn, vn, tables, lens, cu_q=cu)
    small_k, small_v = (torch.zeros(3, hkv, page, dim, dtype=torch.float16, device=DEV) for _ in range(2))
    t2 = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    paged.append_kv(small_k, small_v, kn, vn, t2, lens, cu_q=cu)
    for i, s in zip(ids, (2, 0, 1)):
        assert torch.equal(k[i], small_k[s]) and torch.equal(v[i], small_v[s])
    for rows, c, m in ((q, cu, n), (q[-1:], None, 1)):
        assert torch.equal(paged.attention(rows, k, v, tables, lens, cu_q=c, max_q=m),
                           paged.attention(rows, small_k, small_v, t2, lens, cu_q=c, max_q=m))
    paged.copy_pages(k, v, [pages - 1], [pages - 3])
    assert torch.equal(k[pages - 3], k[pages - 1]) and torch.equal(v[pages - 3], v[pages - 1])


# ---------------------------------------------------------------- filling
def exact_rotation(x, rope, pos, interleaved):
    """64-bit rotation of [tokens, heads, dim]; negative positions pass."""
    r = rope.shape[1]
    out = x.double().clone()
    cos, sin = rope[pos.clamp_min(0)].double()[:, None].chunk(2, -1)
    cos = torch.where(pos[:, None, None] < 0, 1.0, cos)
    sin = torch.where(pos[:, None, None] < 0, 0.0, sin)
    a = torch.arange(0, r, 2, device=DEV) if interleaved else torch.arange(r // 2, device=DEV)
    b = a + (1 if interleaved else r // 2)
    out[..., a] = x[..., a].double() * cos - x[..., b].double() * sin
    out[..., b] = x[..., b].double() * cos + x[..., a].double() * sin
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,heads_kv,dim,rot,page,lens,new", [
    (32, 32, 128, 128, 16, [1, 33, 700, 16, 17], [1, 1, 1, 1, 1]),
    (64, 8, 128, 128, 64, [130, 5, 900], [130, 5, 311]),
    (12, 4, 64, 32, 8, [9, 100, 41], [9, 1, 30]),
    (5, 1, 80, 80, 32, [70, 3], [64, 2]),
    (3, 3, 8, 8, 256, [300], [1]),
    (6, 2, 120, 48, 128, [600, 1], [500, 1]),
])
def test_append(dtype, interleaved, heads, heads_kv, dim, rot, page, lens, new):
    if rot % 16 and not interleaved:
        rot = 0
    bt = Batch(lens, new, heads, heads_kv, dim, page, dtype, seed=41)
    tokens = bt.cu_l[-1]
    g = torch.Generator(device=DEV).manual_seed(5)
    kn, vn = (torch.randn(tokens, heads_kv, dim, device=DEV, generator=g).to(dtype) for _ in range(2))
    rope = paged.rope_table(bt.tables.shape[1] * page, rot) if rot else None
    want_k, want_v = bt.k.clone(), bt.v.clone()
    pos = torch.tensor([n - m + i for n, m in zip(lens, new) for i in range(m)], device=DEV)
    seq = torch.tensor([b for b, m in enumerate(new) for _ in range(m)], device=DEV)
    got = paged.append_kv(bt.k, bt.v, kn, vn, bt.tables, bt.lens, cu_q=bt.cu_q, q=bt.q, rope=rope,
                          interleaved=interleaved)
    page_of = bt.tables[seq, pos // page].long()
    if rope is None:
        assert torch.equal(got, bt.q)
        want_k[page_of, :, pos % page] = kn
    else:
        # one rounding, on top of two products and a sum in fp32
        half = torch.finfo(dtype).eps / 2
        for x, y in ((got, bt.q), (bt.k[page_of, :, pos % page], kn)):
            exact = exact_rotation(y, rope, pos, interleaved)
            room = half * exact.abs() + 2 ** -22 * y.double().abs().amax(-1, keepdim=True) + torch.finfo(dtype).smallest_normal * half
            assert ((x.double() - exact).abs() <= room).all()
        want_k[page_of, :, pos % page] = bt.k[page_of, :, pos % page]
    want_v[page_of, :, pos % page] = vn
    assert torch.equal(bt.k, want_k) and torch.equal(bt.v, want_v)  # every other slot as it was


def test_append_in_place_and_from_one_projection():
    """q, k and v as column ranges of one q/k/v product, q rotated in place; k and v alone."""
    bt = Batch([40, 7], [33, 1], 8, 2, 128, 16, torch.float16)
    rope = paged.rope_table(bt.tables.shape[1] * 16, 128)
    qkv = torch.randn(34, 12, 128, device=DEV).half()
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    k2, v2 = bt.k.clone(), bt.v.clone()
    want = paged.append_kv(k2, v2, k.contiguous(), v.contiguous(), bt.tables, bt.lens, cu_q=bt.cu_q, q=q.contiguous(), rope=rope)
    assert paged.append_kv(bt.k, bt.v, k, v, bt.tables, bt.lens, cu_q=bt.cu_q, rope=rope) is None
    got = paged.append_kv(bt.k, bt.v, k, v, bt.tables, bt.lens, cu_q=bt.cu_q, q=q, rope=rope, q_out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    assert torch.equal(bt.k, k2) and torch.equal(bt.v, v2)


def test_append_leaves_what_is_not_its_own():
    """Rows of no sequence, tokens of negative positions, pages that are no pages."""
    bt = Batch([40, 20], [3, 5], 4, 2, 64, 8, torch.bfloat16)
    bt.lens[1] = 2  # positions -3 .. 1
    tables = bt.tables.clone()
    tables[0, 4] = 10 ** 6  # tokens 32 .. 39 of sequence 0 have no page
    kn, vn = (torch.randn(11, 2, 64, device=DEV).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(11, 4, 64, device=DEV).to(torch.bfloat16)
    out = torch.full_like(q, 5.0)
    k0, v0 = bt.k.clone(), bt.v.clone()
    rope = paged.rope_table(tables.shape[1] * 8, 64)
    paged.append_kv(bt.k, bt.v, kn, vn, tables, bt.lens, cu_q=bt.cu_q, q=q, rope=rope, q_out=out)
    assert (out[8:] == 5.0).all()
    assert torch.equal(out[3:7], q[3:7])  # positions -3 .. 0: nothing to turn
    page = int(tables[1, 0])
    v0[page, :, 0], v0[page, :, 1] = vn[6], vn[7]
    assert torch.equal(bt.v, v0)
    same = torch.ones(bt.k.shape[0], 8, dtype=torch.bool)
    same[page, :2] = False
    assert torch.equal(bt.k.transpose(1, 2)[same.to(DEV)], k0.transpose(1, 2)[same.to(DEV)])


# ---------------------------------------------------------------- copying
@pytest.mark.parametrize("dtype,shape,pairs", [
    (torch.float16, (3, 20, 2, 16, 128), 4), (torch.bfloat16, (1, 1300, 1, 8, 8), 611),
    (torch.float16, (40, 2, 5, 32, 64), 1), (torch.bfloat16, (50, 8, 64, 80), 25)])
def test_copy(dtype, shape, pairs):
    k, v = (torch.randn(shape, device=DEV).to(dtype) for _ in range(2))
    dim = len(shape) - 4
    ids = torch.randperm(shape[dim], generator=torch.Generator().manual_seed(7))
    src, dst = ids[:pairs].tolist(), ids[pairs:2 * pairs].tolist()
    wk, wv = k.clone(), v.clone()
    for w in (wk, wv):
        w.index_copy_(dim, torch.tensor(dst, device=DEV), w.index_select(dim, torch.tensor(src, device=DEV)))
    paged.copy_pages(k, v, src, dst)
    assert torch.equal(k, wk) and torch.equal(v, wv)
    paged.copy_pages(k, v, [], [])
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_copy_layouts():
    """Token-major pages; K and V as halves of one tensor."""
    both = torch.randn(2, 3, 10, 16, 4, 64, device=DEV).half()
    k, v = both[0].transpose(2, 3), both[1].transpose(2, 3)
    want = both.clone()
    want[:, :, 7], want[:, :, 1] = both[:, :, 2], both[:, :, 2]
    paged.copy_pages(k, v, [2, 2], [7, 1])
    assert torch.equal(both, want)
    inter = torch.randn(10, 2, 4, 16, 64, device=DEV).half()  # a page's K and V side by side
    want = inter.clone()
    want[0] = inter[9]
    paged.copy_pages(inter[:, 0], inter[:, 1], [9], [0])
    assert torch.equal(inter, want)
