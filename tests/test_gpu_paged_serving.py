"""The paged cache's operators as a serving loop uses them: together, captured, on several streams.

Tolerances as in test_gpu_paged.py: an output is off by its own rounding and by the rounding of
the weights, half a step each (of the output and of sum p |v|). Where k, v or q went through a
rotation first, the reference takes the stored, rounded values."""
import ctypes
import math
import threading

import pytest
import torch

from drofell_for_revision_b200 import _capi, exllama, paged, real_quant, synthetic

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    assert paged.device_error(DEV) == 0


def plain(q, k, v, window=0, sinks=0):
    """64-bit attention of the last len(q) tokens of one sequence: (out, sum p |v|)."""
    m, n, group = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    k, v = (x.double().repeat_interleave(group, 1) for x in (k, v))
    s = torch.einsum("ihd,jhd->hij", q.double(), k) / math.sqrt(q.shape[2])
    p = torch.arange(n - m, n, device=q.device)[:, None]
    j = torch.arange(n, device=q.device)[None]
    seen = j <= p
    if window:
        seen &= (p - j < window) | (j < sinks)
    w = s.masked_fill(~seen, -math.inf).softmax(-1)
    return torch.einsum("hij,jhd->ihd", w, v), torch.einsum("hij,jhd->ihd", w, v.abs())


def close(got, want, spread, more=0.0):
    half = torch.finfo(got.dtype).eps / 2
    assert ((got.double() - want).abs() <= half * (want.abs() + spread) + 1e-5 * max(1.0, float(spread.max())) + more).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_a_serving_loop(dtype, window, sinks):
    """Prompts, decode steps, forks that diverge, freed sequences, compaction: after every step
    each sequence attends to exactly its own history."""
    heads, hkv, dim, size, layers = 8, 2, 64, 16, 2
    g = torch.Generator(device=DEV).manual_seed(1)
    pool = paged.PagePool(64, size)
    kp, vp = (torch.full((layers, 64, hkv, size, dim), math.nan, dtype=dtype, device=DEV) for _ in range(2))
    history = {}  # name -> per layer (k, v)

    def step(new):
        """new: {name: tokens}. One call of each operator per layer for the whole batch."""
        src, dst = [], []
        for name, n in new.items():
            s, d = pool.extend(name, n)
            src += s
            dst += d
        paged.copy_pages(kp, vp, src, dst)
        tables, lens = pool.tables(new, device=torch.device(DEV))
        first = [0]
        for n in new.values():
            first.append(first[-1] + n)
        cu = torch.tensor(first, dtype=torch.int32, device=DEV)
        single = all(n == 1 for n in new.values())
        for layer in range(layers):
            q = torch.randn(first[-1], heads, dim, device=DEV, generator=g).to(dtype)
            k, v = (torch.randn(first[-1], hkv, dim, device=DEV, generator=g).to(dtype) for _ in range(2))
            for i, name in enumerate(new):
                rows = slice(first[i], first[i + 1])
                old = history.setdefault(name, {}).get(layer)
                mine = (k[rows], v[rows])
                history[name][layer] = mine if old is None else tuple(torch.cat(x) for x in zip(old, mine))
            kw = {} if single else dict(cu_q=cu)
            assert paged.append_kv(kp[layer], vp[layer], k, v, tables, lens, q=None, **kw) is None
            if not single:
                kw["max_q"] = max(new.values())
            out = paged.attention(q, kp[layer], vp[layer], tables, lens, window=window, sinks=sinks, **kw)
            for i, name in enumerate(new):
                rows = slice(first[i], first[i + 1])
                close(out[rows], *plain(q[rows], *history[name][layer], window, sinks))

    step({"a": 150, "b": 5, "c": 33})
    for _ in range(3):
        step({"a": 1, "b": 1, "c": 1})
    for new, old in (("a2", "a"), ("a3", "a"), ("b2", "b")):
        pool.fork(old, new)
        history[new] = dict(history[old])
    step({"a": 1, "a2": 1, "a3": 1, "b": 1, "b2": 1, "c": 1})  # the forks diverge
    step({"a2": 7, "b2": 20, "c": 1})
    for name in ("a", "c"):
        pool.free(name)
        del history[name]
    src, dst = pool.compact()
    assert src
    paged.copy_pages(kp, vp, src, dst)
    step({"a2": 1, "a3": 1, "b": 1, "b2": 1})
    pool.truncate("a2", 20)
    history["a2"] = {i: tuple(x[:20] for x in kv) for i, kv in history["a2"].items()}
    step({"a2": 3, "d": 90, "b": 1})


def test_a_layer_of_the_framework():
    """attention_forward on quantized projections, prompt and decode steps, against the dense
    weights in 64 bits; then the MLP block behind it.

    The chain rounds at every stage (r, q, k, v, rotated q and k, attention, o: eight roundings to
    fp16, 2^-11 each, in products of hidden terms): bound as the framework's other fused blocks,
    1e-2 of the largest value."""
    hidden, heads, hkv, dim, size, inter = 512, 8, 2, 64, 16, 768
    dev = torch.device(DEV)
    lin = {}
    for i, (name, n_in, n_out) in enumerate((("q", hidden, heads * dim), ("k", hidden, hkv * dim), ("v", hidden, hkv * dim),
                                             ("o", heads * dim, hidden), ("gate", hidden, inter), ("up", hidden, inter),
                                             ("down", inter, hidden))):
        layer = synthetic.make_layer(n_in, n_out, 128, act_order=False, seed=i)
        m = real_quant.QuantLinear(128, n_in, n_out, False, False)
        m.qweight.copy_(layer.qweight)
        m.qzeros.copy_(layer.qzeros)
        m.scales.copy_(layer.scales * 0.1)
        m = m.to(dev)
        m.post_init(exllama.TuningParams(), exllama.CacheV2(dev))
        lin[name] = m
    q4 = {n: m.q4_matrix.cuda_q4 for n, m in lin.items()}
    w = {n: m.q4_matrix.dense(torch.float16).double() for n, m in lin.items()}
    g = torch.Generator(device=DEV).manual_seed(3)
    norm = (1 + 0.1 * torch.randn(hidden, device=DEV, generator=g)).half()
    kp, vp = (torch.zeros(40, hkv, size, dim, dtype=torch.float16, device=DEV) for _ in range(2))
    pool = paged.PagePool(40, size)
    rope = paged.rope_table(40 * size, dim, device=dev)
    seen = {}

    def turn(x, pos):
        c, s = rope[pos].double()[:, None].chunk(2, -1)
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    for new in ({"x": 70, "y": 200}, {"x": 1, "y": 1}, {"x": 1, "y": 1}, {"x": 3, "y": 1}):
        for name, n in new.items():
            pool.extend(name, n)
        tables, lens = pool.tables(new, width=40, device=dev)
        rows = sum(new.values())
        x = torch.randn(rows, hidden, device=DEV, generator=g).half()
        first = [0]
        for n in new.values():
            first.append(first[-1] + n)
        cu = torch.tensor(first, dtype=torch.int32, device=DEV)
        got = paged.attention_forward(norm, 1e-6, q4["q"], q4["k"], q4["v"], q4["o"], x, kp, vp, tables, lens, rope=rope,
                                      cu_q=cu, max_q=max(new.values()))
        d = x.double()
        r = d * norm.double() * torch.rsqrt((d * d).mean(-1, keepdim=True) + 1e-6)
        want = []
        for i, (name, n) in enumerate(new.items()):
            mine = r[first[i]:first[i + 1]]
            pos = torch.arange(pool.length(name) - n, pool.length(name), device=DEV)
            q = turn((mine @ w["q"]).view(n, heads, dim), pos)
            k = turn((mine @ w["k"]).view(n, hkv, dim), pos)
            v = (mine @ w["v"]).view(n, hkv, dim)
            old = seen.get(name)
            seen[name] = (k, v) if old is None else (torch.cat((old[0], k)), torch.cat((old[1], v)))
            want.append(plain(q, *seen[name])[0].reshape(n, -1) @ w["o"])
        want = torch.cat(want)
        assert float((got.double() - want).abs().max() / want.abs().max()) < 1e-2
        h = (x + got).contiguous()
        bufs = [torch.empty(rows, n, dtype=torch.float16, device=DEV) for n in (hidden, inter, inter, hidden)]
        exllama.mlp_forward_v2(norm, 1e-6, q4["gate"], q4["up"], q4["down"], *bufs[:3], None, h, bufs[3])
        assert torch.isfinite(bufs[3]).all()


def make(lens, new, heads=8, hkv=2, dim=128, size=16, dtype=torch.float16, seed=0, width=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    used = [-(-n // size) for n in lens]
    order = torch.randperm(sum(used), device=DEV, generator=g).int()
    tables = torch.full((len(lens), width or max(used)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(used):
        tables[b, :n] = order[at:at + n]
        at += n
    k, v = (torch.randn(sum(used), hkv, size, dim, device=DEV, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(sum(new), heads, dim, device=DEV, generator=g).to(dtype)
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    return dict(q=q, k_pages=k, v_pages=v, tables=tables, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                cu_q=cu, max_q=max(new))


@pytest.mark.parametrize("new", [1, 3, 40, 300])
def test_captured_and_replayed_with_other_lengths(new):
    """A graph replays with what lengths and tables hold then, and every replay gives what a plain
    call gives, bit for bit."""
    a = make([2000, 900, 1500], [new] * 3, width=200)
    out = torch.empty_like(a["q"])
    paged.attention(**a, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attention(**a, out=out)
    for lens in ([2000, 900, 1500], [1, 899, 0], [333, 17, 1500], [1024, 1, 640]):
        a["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        a["tables"].copy_(a["tables"].flip(0))
        out.fill_(math.nan)
        graph.replay()
        assert torch.equal(out, paged.attention(**a))


@pytest.mark.parametrize("new", [1, 200])
def test_two_graphs_and_streams_do_not_share_a_workspace(new):
    """Two captured calls replayed at once on two streams, and plain calls on two streams."""
    a, b = make([3000, 700], [new] * 2, seed=1), make([2500, 1100], [new] * 2, seed=2)
    want = [paged.attention(**x) for x in (a, b)]
    outs = [torch.empty_like(x["q"]) for x in (a, b)]
    graphs, streams = [], [torch.cuda.Stream(DEV) for _ in range(2)]
    for x, o in zip((a, b), outs):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            paged.attention(**x, out=o)
        graphs.append(gr)
    torch.cuda.synchronize()
    for _ in range(20):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs, want))
    got = [[], []]
    for _ in range(20):
        for i, (x, st) in enumerate(zip((a, b), streams)):
            with torch.cuda.stream(st):
                got[i].append(paged.attention(**x))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_append_and_copy_captured():
    a = make([40, 90], [1, 1])
    kn, vn = (torch.randn(2, 2, 128, device=DEV).half() for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    kp, vp = a["k_pages"], a["v_pages"]
    with torch.cuda.graph(graph):
        paged.append_kv(kp, vp, kn, vn, a["tables"], a["lens"])
        paged.copy_pages(kp, vp, [0], [1])
    for lens in ([40, 90], [7, 33]):
        a["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        kn.normal_()
        wk, wv = kp.clone(), vp.clone()
        for b, n in enumerate(lens):
            page, slot = int(a["tables"][b, (n - 1) // 16]), (n - 1) % 16
            wk[page, :, slot], wv[page, :, slot] = kn[b], vn[b]
        wk[1], wv[1] = wk[0].clone(), wv[0].clone()
        graph.replay()
        assert torch.equal(kp, wk) and torch.equal(vp, wv)


def test_from_a_thread_that_never_used_cuda():
    """The tensor maps of the prompt kernel need a current context."""
    a = make([500, 260], [150, 150])
    want = paged.attention(**a)
    got = []

    def work():
        got.append(paged.attention(**a))
        torch.cuda.synchronize()
    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert torch.equal(got[0], want)


def test_refusals_with_tensors_on_the_gpu():
    a = make([50, 60], [1, 1])
    call = dict(a, cu_q=None)
    for name in ("tables", "lens", "q"):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            paged.attention(**dict(call, **{name: call[name].cpu()}))
    with pytest.raises(RuntimeError, match="query heads"):
        paged.attention(**dict(call, q=torch.zeros(2, 7, 128, dtype=torch.float16, device=DEV)))
    with pytest.raises(RuntimeError, match="sinks"):
        paged.attention(**call, sinks=3)
    with pytest.raises(RuntimeError, match="scale"):
        paged.attention(**call, scale=-1.0)
    with pytest.raises(RuntimeError, match="page size"):
        paged.attention(**dict(call, k_pages=call["k_pages"][:, :, :12], v_pages=call["v_pages"][:, :, :12]))
    odd = torch.zeros(2, 8, 132, dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError, match="aligned|multiples"):
        paged.attention(**dict(call, q=odd[:, :, 2:130]))
    with pytest.raises(RuntimeError, match="rope table"):
        paged.append_kv(call["k_pages"], call["v_pages"], call["q"][:, :2], call["q"][:, :2], call["tables"], call["lens"],
                        rope=paged.rope_table(8, 128))
    with pytest.raises(RuntimeError, match="written twice"):
        paged.copy_pages(call["k_pages"], call["v_pages"], [0, 1], [2, 2])
    q4 = 12345
    with pytest.raises(RuntimeError, match="unknown or released"):
        paged.attention_forward(torch.ones(8), 1e-6, q4, q4, q4, q4, call["q"], call["k_pages"], call["v_pages"],
                                call["tables"], call["lens"])


def test_c_abi_checks_its_workspace():
    for new in (1, 100):
        a = make([4000, 700], [new] * 2)
        lib, ref = _capi.lib(), ctypes.byref
        k = a["k_pages"]
        pages = _capi.Pages(k.data_ptr(), a["v_pages"].data_ptr(), k.stride(0), k.stride(1), k.stride(2), k.shape[0],
                            k.shape[1], k.shape[2], k.shape[3], _capi.DTYPE_FP16, 0)
        seqs = _capi.Seqs(a["tables"].data_ptr(), a["lens"].data_ptr(), a["cu_q"].data_ptr(), a["tables"].stride(0),
                          a["tables"].shape[1], 2, 2 * new, new)
        need = lib.w4a16_paged_attention_workspace_size(ref(pages), ref(seqs), 8, 0, 0)
        assert need > 0
        out = torch.zeros_like(a["q"])
        qr, outr = (_capi.Rows(t.data_ptr(), t.stride(0), t.stride(1)) for t in (a["q"], out))
        ws = torch.empty(need + 64, dtype=torch.uint8, device=DEV)
        scale = 1 / math.sqrt(128)

        def call(ptr, size):
            return lib.w4a16_paged_attention(ref(pages), ref(seqs), ref(qr), ref(outr), 8, scale, 0, 0, ptr, size,
                                             _capi.stream_ptr(0))
        assert call(ws.data_ptr(), need - 1) == _capi.W4A16_ERR_WORKSPACE
        assert call(None, need) == _capi.W4A16_ERR_WORKSPACE
        assert call(ws.data_ptr() + 16, need) == _capi.W4A16_ERR_INVALID
        assert call(ws.data_ptr(), need) == _capi.W4A16_OK
        assert torch.equal(out, paged.attention(**a))
        # the workspace's bytes are within what was asked for
        ws.fill_(0xA5)
        assert call(ws.data_ptr(), need) == _capi.W4A16_OK
        assert (ws[need:] == 0xA5).all()
