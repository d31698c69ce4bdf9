"""The paged cache where scores and values are extreme: weights far below the largest, maxima that rise along
the keys, infinities and NaN, empty slots of a padded batch.

Tolerances. As in test_gpu_paged.py an output is off by at most half a step of its own and half a
step of the weights, (eps / 2) (|out| + sum p |v|) together. What comes on top is counted here:
 * fp32 accumulation takes one step, at most 2^-23 relative, for every 16 keys of a product, and
   400 more cover sums inside a tile and the join: (n / 16 + 400) 2^-23 sum p |v|;
 * a score's error is amplified by the exponential: scores of at most 2^9 (base 2) are off by
   2^-23 of that in two roundings, 2^-13 sum p |v|, counted only where scores are that large;
 * fp16 cannot hold a weight below its smallest step: with the weights scaled by 2^7 and the
   running maximum at most 2^8 behind, half a step is 2^-32 of the largest weight (2^-40 where
   they are scaled by 2^15 against the exact maximum): n 2^-32 max |v|.
"""
import math

import pytest
import torch

from drofell_for_revision_b200 import paged
from test_gpu_paged import DEV, Batch, check_attention, exact_attention

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    assert paged.device_error(DEV) == 0


def attend(bt, scale, **kw):
    return paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=bt.cu_q, max_q=bt.max_q, scale=scale, **kw)


def check(bt, scale, n, score_error=0.0, **kw):
    got = attend(bt, scale, **kw)
    want, spread = exact_attention(bt, scale, kw.get("window", 0), kw.get("sinks", 0))
    half = torch.finfo(got.dtype).eps / 2
    room = half * (want.abs() + spread) + ((n / 16 + 400) * 2.0 ** -23 + score_error) * spread
    if got.dtype == torch.float16:
        room = room + n * 2.0 ** -32 * float(bt.v.abs().max()) + 2.0 ** -25  # and half the output's own smallest step
    over = (got.double() - want).abs() / room
    assert float(over.max()) <= 1.0
    return got


# ---------------------------------------------------------------- weights far below the largest
def sinks_first(lens, new, heads, hkv, dim, dtype, low, high):
    """Sequences whose first key lies `low` to `high` nats above the others, its value 0, theirs of
    one sign."""
    bt = Batch(lens, new, heads, hkv, dim, 64, dtype, seed=71)
    g = torch.Generator(device=DEV).manual_seed(71)
    bt.q.mul_(0.01)
    bt.q[..., 0] = 4.0
    bt.k.mul_(0.01)
    gap = low + (high - low) * torch.rand(bt.k.shape[:3], device=DEV, generator=g)
    bt.k[..., 0] = (-gap * math.sqrt(dim) / 4.0).to(dtype)
    bt.v.copy_((bt.v.abs() * 0.5 + 0.5).to(dtype))
    first = bt.tables[:, 0].long()
    bt.k[first, :, 0, 0] = 0.0
    bt.v[first, :, 0] = 0.0
    return bt


# weights of 17.4 nats below the largest round to 0 on fp16's own grid, those of 16.8 to 17.2 to the
# step above
GAPS = [(14.0, 18.0), (17.4, 18.0), (16.8, 17.2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("low,high", GAPS)
@pytest.mark.parametrize("n,new", [(40000, 1), (130001, 1), (33000, 64), (3000, 300)])
def test_one_key_holds_nearly_all_the_weight(dtype, dim, low, high, n, new):
    bt = sinks_first([n], [new], 4, 1, dim, dtype, low, high)
    check(bt, 1.0 / math.sqrt(dim), n)
    # and where all values are 1, so is the result: no weight is counted and not summed
    bt.v.fill_(1.0)
    check(bt, 1.0 / math.sqrt(dim), n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("low,high", GAPS)
@pytest.mark.parametrize("batch,n,new", [(160, 900, 1), (80, 900, 64)])
def test_one_key_holds_nearly_all_the_weight_of_many_sequences(dtype, low, high, batch, n, new):
    """So many that most are not cut into pieces with a maximum of their own."""
    check(sinks_first([n] * batch, [new] * batch, 8, 8, 64, dtype, low, high), 0.125, n)


# ---------------------------------------------------------------- values that are not finite
def far(lens, new, dtype, j_top, seed):
    """Sequences whose key j_top is 256 nats above the others: exp2 of the distance is 0 in fp32."""
    bt = Batch(lens, new, 4, 2, 128, 16, dtype, seed=seed)
    bt.q.mul_(0.1)
    bt.q[..., 0] = 16.0
    bt.k.mul_(0.1)
    bt.k[..., 0] = 0.0
    for b in range(len(lens)):
        bt.k[int(bt.tables[b, j_top // 16]), :, j_top % 16, 0] = 16.0
    return bt


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n,new,j_top", [(5000, 1, 10), (5000, 1, 4990), (5000, 200, 3), (300, 1, 299)])
def test_infinite_values_of_vanishing_weight(dtype, value, n, new, j_top):
    """A weight is never 0, however far its key lies below the largest: an infinity there is one in
    the result, whatever pieces the keys were cut into."""
    bt = far([n, n], [new, new], dtype, j_top, 73)
    for j, d in ((5, 7), (n // 2, 40), (n - new - 1, 100)):
        bt.v[int(bt.tables[0, j // 16]), :, j % 16, d] = value
    want, _ = exact_attention(bt, 1.0, 0, 0)
    got = attend(bt, 1.0).double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    assert not torch.isfinite(want[:new][..., [7, 40, 100]]).any() and torch.isfinite(want[new:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n,new", [(60, 4), (5000, 4), (60, 40), (5000, 200)])
def test_a_row_computed_anew_keeps_what_it_sees(dtype, value, n, new):
    """A row that a value it does not see made not finite is computed anew; an infinity that it does
    see, of vanishing weight, still decides its dimension."""
    bt = far([n], [new], dtype, 1, 79)
    page, slot = int(bt.tables[0, 0]), 0
    bt.v[page, :, slot, 7] = value
    last = n - 1  # seen by the last row alone
    bt.v[int(bt.tables[0, last // 16]), :, last % 16, 90] = math.nan
    want, _ = exact_attention(bt, 1.0, 0, 0)
    got = attend(bt, 1.0).double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])


# ---------------------------------------------------------------- long contexts
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_values_that_are_not_finite_at_the_end_of_a_long_context(dtype, value):
    """The rows just before such a value are computed anew over 200000 keys each while their CTA's other
    warps, with items of other sequences ahead of them, wait: nobody gives up, and nobody else's rows
    change. Other sequences enough that no item is cut."""
    hkv, dim, size, new, n, others = 8, 128, 64, 2048, 200064, 9
    g = torch.Generator(device=DEV).manual_seed(97)
    used, few = n // size, 2048 // size
    k, v = (torch.randn(used + others * few, hkv, size, dim, device=DEV, generator=g, dtype=torch.float32).to(dtype)
            for _ in range(2))
    tables = torch.zeros(others + 1, used, dtype=torch.int32, device=DEV)
    tables[0] = torch.arange(used, device=DEV)
    tables[1:, :few] = used + torch.arange(others * few, device=DEV).view(others, few)
    lens = torch.tensor([n] + [2048] * others, dtype=torch.int32, device=DEV)
    cu = torch.arange(0, (others + 1) * new + 1, new, dtype=torch.int32, device=DEV)
    q = torch.randn((others + 1) * new, hkv, dim, device=DEV, generator=g).to(dtype)
    clean = paged.attention(q, k, v, tables, lens, cu_q=cu, max_q=new)
    at = n - 60  # in the last tile of 128 keys, which begins at n - 128
    keep = v[at // size, :, at % size].clone()
    v[at // size, :, at % size] = value
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    got = paged.attention(q, k, v, tables, lens, cu_q=cu, max_q=new)
    end.record()
    assert paged.device_error(DEV) == 0
    assert start.elapsed_time(end) < 10000
    first, row = new - 128, at - (n - new)  # rows of the tile, the first that sees the value
    assert (torch.isnan(got[row:new]) if value != value else got[row:new] == value).all()
    assert torch.equal(got[:first], clean[:first]) and torch.equal(got[new:], clean[new:])
    v[at // size, :, at % size] = keep
    half = torch.finfo(dtype).eps / 2
    for h in (0, 5):
        kk, vv = (x[:used, h].reshape(-1, dim)[:at].double() for x in (k, v))
        s = q[first:row, h].double() @ kk.T / math.sqrt(dim)
        s.masked_fill_(torch.arange(at, device=DEV)[None] > torch.arange(n - 128, at, device=DEV)[:, None], -math.inf)
        w = torch.softmax(s, -1)
        want, spread = w @ vv, w @ vv.abs()
        room = half * (want.abs() + spread) + (n / 16 + 400) * 2.0 ** -23 * spread
        assert ((got[first:row, h].double() - want).abs() <= room).all()


def test_many_items_with_rows_to_settle():
    """More items a CTA than bits to note them by, a few of them with rows to settle."""
    bt = Batch([60 + i % 50 for i in range(700)], [40] * 700, 8, 8, 64, 16, torch.float16, seed=101)
    for b in range(0, 700, 9):
        bt.v[int(bt.tables[b, 2]), :, b % 16, b % 64] = (math.nan, math.inf, -math.inf)[b % 3]
    check_attention(bt)


# ---------------------------------------------------------------- sequences without a key
def graph_time(call, calls=20):
    """Microseconds a call, of several in one graph."""
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(calls):
            call()
    best = math.inf
    for _ in range(4):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        graph.replay()
        end.record()
        torch.cuda.synchronize()
        best = min(best, start.elapsed_time(end) * 1000 / calls)
    return best


@pytest.mark.parametrize("heads,hkv,dim,new", [(64, 8, 128, 1), (32, 32, 80, 1), (64, 8, 128, 2), (32, 32, 64, 30)])
@pytest.mark.parametrize("batch", [16, 300])
def test_empty_slots_of_a_padded_batch(heads, hkv, dim, new, batch):
    """A fixed batch in which some slots hold no sequence: their rows are 0, the others right, and the
    call takes no longer than with sequences there, within a factor of two (and 20 us) for noise."""
    bt = Batch([500] * batch if batch < 100 else [60] * batch, [new] * batch, heads, hkv, dim, 16, torch.float16, seed=103)
    full = attend(bt, 0.1)
    base = graph_time(lambda: attend(bt, 0.1, out=full))
    empty = torch.zeros(batch, dtype=torch.bool)
    empty[[0, 3, 4, batch - 1]] = True
    bt.lens.masked_fill_(empty.to(DEV), 0)
    out = torch.full_like(full, math.nan)
    attend(bt, 0.1, out=out)
    assert (out[empty.repeat_interleave(new).to(DEV)] == 0).all()
    bt.lens_l = [0 if e else n for n, e in zip(bt.lens_l, empty.tolist())]
    check(bt, 0.1, 500, out=out)
    took = graph_time(lambda: attend(bt, 0.1, out=out))
    assert took < 2 * base + 20, (took, base)


# ---------------------------------------------------------------- rows computed anew
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,hkv,dim", [(4, 4, 128), (8, 1, 64), (6, 2, 128), (10, 2, 80), (4, 4, 120), (12, 4, 8)])
@pytest.mark.parametrize("n,new,window,sinks", [(2600, 260, 0, 0), (700, 700, 0, 0), (2600, 300, 500, 4), (300, 130, 33, 70)])
def test_rows_computed_anew(dtype, heads, hkv, dim, n, new, window, sinks):
    """Values that are not finite all along the new tokens and at the edges of what windows show: most
    rows have some in their tiles that they do not see, and compute everything else anew. Some
    pages are no pages."""
    bt = Batch([n, 40], [new, 20], heads, hkv, dim, 16, dtype, seed=107)
    hide = [torch.zeros(n, dtype=torch.bool), torch.zeros(40, dtype=torch.bool)]
    for j in range(max(0, n - new - 3), n, 37):
        bt.v[int(bt.tables[0, j // 16]), :, j % 16, j % dim] = (math.nan, math.inf, -math.inf)[j % 3]
    for j in range(5, max(6, n - new - window), 97):
        bt.v[int(bt.tables[0, j // 16]), :, j % 16, (j // 7) % dim] = math.inf
    good, bt.tables = bt.tables, bt.tables.clone()
    bt.tables[0, 3], bt.tables[0, (n - new) // 16] = -1, bt.k.shape[0]
    for at in (3, (n - new) // 16):
        hide[0][at * 16:at * 16 + 16] = True
    got = attend(bt, 1 / math.sqrt(dim), window=window, sinks=sinks)
    bt.tables = good
    want, spread = exact_attention(bt, 1 / math.sqrt(dim), window, sinks, hide)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    finite = torch.isfinite(want)
    assert torch.equal(got[torch.isinf(want)].double(), want[torch.isinf(want)])
    room = torch.finfo(dtype).eps / 2 * (want.abs() + spread) + (n / 16 + 400) * 2.0 ** -23 * spread + n * 2.0 ** -32 * 8 + 2.0 ** -25
    assert ((got.double() - want).abs() <= room)[finite].all()
    assert finite.any() and not finite.all()


# ---------------------------------------------------------------- arguments left out
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2], [40, 7, 0], [300, 1, 150]])
def test_max_q_may_be_left_out(new):
    """With row offsets and no max_q every row of a sequence gets its result."""
    bt = Batch([n + 50 for n in new], new, 8, 2, 64, 16, torch.float16, seed=109)
    cu = torch.tensor(bt.cu_l, dtype=torch.int32, device=DEV)
    out = torch.full_like(bt.q, math.nan)
    paged.attention(bt.q, bt.k, bt.v, bt.tables, bt.lens, cu_q=cu, out=out)
    want, spread = exact_attention(bt, 0.125, 0, 0)
    assert ((out.double() - want).abs() <= 2.0 ** -11 * (want.abs() + spread) + 1e-5 * float(bt.v.abs().max())).all()


def test_append_with_a_q_of_no_heads():
    """k and v are stored whatever q holds."""
    bt = Batch([40, 7], [1, 1], 4, 2, 64, 16, torch.float16, seed=113)
    kn, vn = (torch.randn(2, 2, 64, device=DEV).half() for _ in range(2))
    k, v = bt.k.clone(), bt.v.clone()
    paged.append_kv(k, v, kn, vn, bt.tables, bt.lens)
    got = paged.append_kv(bt.k, bt.v, kn, vn, bt.tables, bt.lens, q=torch.empty(2, 0, 64, dtype=torch.float16, device=DEV))
    assert got.shape == (2, 0, 64)
    assert torch.equal(bt.k, k) and torch.equal(bt.v, v)


# ---------------------------------------------------------------- scores that are not finite
def by_selection(bt, scale, window=0):
    """The rule in 64 bits, rows by heads: 'nan' where a visible score is NaN or +inf (softmax of an
    infinity), 0 where every visible one is -inf, else the result without the keys at -inf."""
    heads, hkv = bt.q.shape[1], bt.k.shape[1]
    out = torch.zeros(bt.q.shape, dtype=torch.float64, device=DEV)
    spread = torch.zeros_like(out)
    for b, (n, m) in enumerate(zip(bt.lens_l, bt.new_l)):
        k, v = bt.keys(b, bt.k), bt.keys(b, bt.v)
        rows = slice(bt.cu_l[b], bt.cu_l[b] + m)
        p = torch.arange(n - m, n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)[None]
        seen = (j <= p) & ((p - j < window) if window else True)
        for h in range(heads):
            q = bt.q[rows, h].double()
            prod = q[:, None] * k[h * hkv // heads][None]
            s = prod.sum(-1) * scale
            s = torch.where(seen, s, -math.inf)
            bad = (torch.isnan(s) | (s == math.inf)).any(-1)
            top = s.nan_to_num(0.0, 0.0, -math.inf).amax(-1, keepdim=True)
            w = torch.exp(torch.where(s == -math.inf, -math.inf, s.nan_to_num(0.0, 0.0)) - top.nan_to_num(0.0, 0.0, 0.0))
            w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
            vv = v[h * hkv // heads]
            out[rows, h] = torch.where(bad[:, None], math.nan, w @ vv)
            spread[rows, h] = w @ vv.abs()
    return out, spread


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("what", ["k", "every k", "q", "q to -inf"])
@pytest.mark.parametrize("n,new", [(40, 1), (1500, 1), (90, 6), (200, 150), (1500, 140)])
def test_scores_that_are_not_finite(dtype, value, what, n, new):
    bt = Batch([n, 30], [new, 1], 4, 2, 128, 16, dtype, seed=83)
    if what == "k":  # one key, one dimension: +inf for queries of one sign, -inf for the others
        j = n // 2
        bt.k[int(bt.tables[0, j // 16]), 0, j % 16, 7] = value
    elif what == "every k":
        bt.k[bt.tables[0].long().clamp_min(0), 1, :, 7] = value
    elif what == "q":
        bt.q[0, 1, 7] = value
    else:  # every score of the row -inf
        bt.k[..., 7] = -bt.k[..., 7].abs() - 0.5
        bt.q[0, 1, 7] = value
    want, spread = by_selection(bt, 1 / math.sqrt(128))
    got = attend(bt, 1 / math.sqrt(128))
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    half = torch.finfo(dtype).eps / 2
    ok = ~torch.isnan(want)
    room = half * (want.abs() + spread) + (n / 16 + 400) * 2.0 ** -23 * spread + n * 2.0 ** -32 * float(bt.v.abs().max())
    assert ((got.double() - want).abs() <= room + 2.0 ** -25)[ok].all()
    if what == "q to -inf" and value == math.inf:
        assert (got[0, 1] == 0).all()


# ---------------------------------------------------------------- maxima that rise along the keys
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,hkv,dim", [(4, 4, 128), (8, 1, 64), (6, 2, 128)])
@pytest.mark.parametrize("n,new,window,sinks", [(2600, 260, 0, 0), (700, 700, 0, 0), (2600, 1, 0, 0), (2600, 5, 0, 0),
                                                (2600, 300, 500, 4), (5000, 40, 0, 0)])
def test_maxima_that_rise(dtype, heads, hkv, dim, n, new, window, sinks):
    """Each tile of 128 keys raises the maximum of a row by its own factor: not at all, by just less
    and just more than what is tolerated without rescaling (2^8), by far more, or it falls. Rows
    of all kinds lie side by side in a warp; under the window the first tiles show some of them
    nothing."""
    bt = Batch([n], [new], heads, hkv, dim, 64, dtype, seed=89)
    bt.q.mul_(0.02)
    bt.k.mul_(0.5)
    factors = torch.tensor([0.0, 7.875, 8.125, 20.0, -3.0, 0.5, 16.0], device=DEV)
    rows = torch.arange(new * heads, device=DEV).view(new, heads)
    bt.q[..., 0] = factors[rows % 7].to(dtype)
    used = -(-n // 64)
    for i in range(used):
        bt.k[int(bt.tables[0, i]), :, :, 0] = float(i // 2 % 16)  # and starts again behind 2048 keys
    check(bt, math.log(2), n, score_error=2.0 ** -13, window=window, sinks=sinks)


# ---------------------------------------------------------------- long contexts of ordinary data
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,new", [([60001, 5], [1, 1]), ([20000], [4]), ([40000], [150]), ([9000, 9000, 100], [200, 1, 100])])
def test_long_contexts_without_an_absolute_term(dtype, lens, new):
    """Outputs of a long context are small: a bound in terms of sum p |v| and the type alone."""
    bt = Batch(lens, new, 8, 2, 128, 64, dtype, seed=127)
    check(bt, 1 / math.sqrt(128), max(lens))


# ---------------------------------------------------------------- values near the type's end
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,new", [([900], [1]), ([50000], [1]), ([700, 20], [4, 2]), ([6000], [200]), ([400, 30], [400, 30]),
                                      ([900] * 80, [64] * 80), ([500] * 200, [1] * 200)])
def test_values_near_the_types_end(dtype, lens, new):
    """A mean of values is no larger than they are, though the sum that it is made of may pass fp32's
    range (bf16 has fp32's exponents)."""
    bt = Batch(lens, new, 8, 4, 64, 16, dtype, seed=131)
    g = torch.Generator(device=DEV).manual_seed(131)
    top = float(torch.finfo(dtype).max)
    bt.v.copy_((top * (0.5 + 0.4 * torch.rand(bt.v.shape, device=DEV, generator=g))).to(dtype))
    bt.v[..., 3] *= -1
    want, spread = exact_attention(bt, 0.125, 0, 0)
    got = attend(bt, 0.125)
    room = torch.finfo(dtype).eps / 2 * (want.abs() + spread) + (max(lens) / 16 + 400) * 2.0 ** -23 * spread
    if dtype == torch.float16:
        room = room + max(lens) * 2.0 ** -32 * top
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= room).all()


# ---------------------------------------------------------------- scores of any size
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,new", [([900], [1]), ([1000], [4]), ([1000], [30]), ([900], [200]), ([1000], [1000]),
                                      ([700] * 120, [20] * 120)])
def test_scores_of_any_size(dtype, lens, new):
    """Scores from 1 to 2^30 in size, the largest of them far above or far below 0: where they are that
    large one key takes all the weight, and no rounding of a maximum may reach the weights."""
    bt = Batch(lens, new, 8, 4, 64, 16, dtype, seed=137)
    n = max(lens)
    g = torch.Generator().manual_seed(137)
    steps = 128 if dtype == torch.bfloat16 else 1024  # numbers between 2^15 and 2^16
    rows = torch.arange(bt.q.shape[0] * 8).view(-1, 8)
    bt.q.zero_()
    bt.q[..., 0] = ((2.0 ** (rows % 15)) * (1 - 2 * (rows % 2))).to(dtype).to(DEV)
    for b, length in enumerate(lens):
        k = 2.0 ** 15 * (1 + torch.randperm(n, generator=g)[:length] % steps / steps)
        k = (k * (1 - 2 * (torch.arange(length) // 300 % 2)) if b % 3 == 0 else k if b % 3 == 1 else -k).to(dtype).to(DEV)
        at = torch.arange(length, device=DEV)
        bt.k[bt.tables[b].long()[at // 16], :, at % 16, 0] = k[:, None]
    bt.k[..., 1:] = 0
    check(bt, 1.0, n)
