"""Cases of the paged key-value cache: filling it (rotary embedding fused), attention of single tokens over it,
attention of a prompt's or chunk's tokens with a sliding window and sinks, and copying its pages.

Head counts and widths are those of the Llama-2 7B, 13B and 70B layers that ``bench.py`` runs (32/32, 40/40 and
64/8 heads of 128), others in the drawn cases. ``run`` is one call a serving program makes for one layer; copying
moves the pages of every layer that the cache holds.
"""
import math
import random

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decode step of 8 sequences: the smallest write of a serving loop
        dict(name="append_decode_8", op="append", heads=32, heads_kv=32, dim=128, page=16, dtype="fp16", batch=8,
             new=1, longest=1500, ragged=True, interleaved=False),
        # a prompt batch of ragged lengths
        dict(name="append_prompts", op="append", heads=64, heads_kv=8, dim=128, page=64, dtype="bf16", batch=5,
             new=2111, longest=4096, ragged=True, interleaved=False),
        # a single user's next token: latency counts
        dict(name="decode_one", op="attend", heads=32, heads_kv=32, dim=128, page=16, dtype="fp16", batch=1, new=1,
             longest=777, ragged=False, window=0, sinks=0),
        # a serving batch of uneven lengths, heads shared by 8
        dict(name="decode_batch_ragged", op="attend", heads=64, heads_kv=8, dim=128, page=64, dtype="bf16", batch=48,
             new=1, longest=8191, ragged=True, window=0, sinks=0),
        # two very long contexts: all the parallelism is along the cache
        dict(name="decode_long", op="attend", heads=64, heads_kv=8, dim=128, page=32, dtype="fp16", batch=2, new=1,
             longest=130001, ragged=False, window=0, sinks=0),
        # streaming generation: a window and the first tokens
        dict(name="decode_window", op="attend", heads=40, heads_kv=40, dim=128, page=32, dtype="bf16", batch=24,
             new=1, longest=12000, ragged=True, window=1024, sinks=4),
        # short prompts of uneven lengths, among them single tokens
        dict(name="prompt_short_ragged", op="attend", heads=32, heads_kv=32, dim=128, page=16, dtype="fp16", batch=7,
             new=300, longest=300, ragged=True, window=0, sinks=0),
        # one long prompt
        dict(name="prompt_long", op="attend", heads=32, heads_kv=32, dim=128, page=64, dtype="bf16", batch=1,
             new=8192, longest=8192, ragged=False, window=0, sinks=0),
        # prompts with shared heads
        dict(name="prompt_grouped", op="attend", heads=64, heads_kv=8, dim=128, page=128, dtype="bf16", batch=3,
             new=2048, longest=2048, ragged=False, window=0, sinks=0),
        # a chunk of a long prompt under a window with sinks
        dict(name="chunk_window_sinks", op="attend", heads=40, heads_kv=40, dim=128, page=32, dtype="fp16", batch=1,
             new=2047, longest=12287, ragged=False, window=2048, sinks=4),
        # eight beams fork: one partly filled page each, every layer
        dict(name="copy_fork_8", op="copy", layers=32, heads_kv=32, dim=128, page=16, dtype="fp16", pages=64, pairs=8),
        # compaction of a cache
        dict(name="copy_compact", op="copy", layers=16, heads_kv=8, dim=128, page=64, dtype="bf16", pages=1200,
             pairs=511),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "prompt", "prompt", "copy"])
    heads, heads_kv = rng.choice([(32, 32), (40, 40), (64, 8), (32, 8), (16, 1), (12, 4), (14, 2)])
    c = dict(heads=heads, heads_kv=heads_kv, dim=rng.choice([128, 128, 128, 64, 80, 96]),
             page=rng.choice([8, 16, 32, 64, 128]), dtype=rng.choice(["fp16", "bf16"]))
    if op == "copy":
        del c["heads"]
        layers = _log(rng, 1, 16)
        per = layers * heads_kv * c["dim"] * c["page"] * 4
        pairs = _log(rng, 1, max(2, min(511, int(5e8 / per))))
        c.update(op="copy", layers=layers, pairs=pairs, pages=2 * pairs + rng.randint(0, 50))
        return c
    c.update(ragged=rng.random() < 0.6)
    if op == "append":
        if rng.random() < 0.5:
            c.update(op="append", batch=_log(rng, 1, 128), new=1, longest=_log(rng, 1, 2000))
        else:
            new = _log(rng, 2, 2000)
            c.update(op="append", batch=rng.randint(1, 4), new=new, longest=new + rng.randint(0, 500))
        c["interleaved"] = rng.random() < 0.3
        return c
    windowed = rng.random() < 0.5
    c.update(op="attend", window=_log(rng, 1, 3000) if windowed else 0, sinks=rng.choice([0, 1, 4, 70]) if windowed else 0)
    if op == "attend":
        batch = _log(rng, 1, 64)
        most = max(2, int(4e8 / (batch * heads_kv * c["dim"] * 4)))
        c.update(batch=batch, new=1 if rng.random() < 0.8 else rng.randint(2, 4), longest=_log(rng, 4, min(60000, most)))
    else:
        batch = rng.randint(1, 5)
        new = _log(rng, 5, int(3500 / math.sqrt(batch)))
        c.update(batch=batch, new=new, longest=new + (_log(rng, 1, 3000) if rng.random() < 0.5 else 0))
    return c


def _lengths(case):
    """(lengths after the new tokens, new tokens of each sequence): part of the case, whatever the seed."""
    r = random.Random(case["batch"] * 1000003 + case["longest"] * 101 + case["new"])
    lens, new = [], []
    for b in range(case["batch"]):
        n = case["new"]
        old = case["longest"] - n
        if case["ragged"] and b:  # the first one is the longest
            n = n if n == 1 else _log(r, 1, n)
            old = _log(r, 1, old + 1) - 1
        lens.append(old + n)
        new.append(n)
    return lens, new


def _draw_normal(shape, dtype, gen, scale=1.0):
    """Normal values of `dtype`, made in pieces so that a large cache needs no copy in 32 bits."""
    x = torch.empty(shape, dtype=dtype, device="cuda")
    flat = x.view(-1)
    step = 1 << 28
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, device="cuda", dtype=torch.float32, generator=gen).mul_(scale)
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    r = random.Random(seed)
    dtype, hkv, dim, size = TYPES[case["dtype"]], case["heads_kv"], case["dim"], case["page"]
    s = dict(case=case)
    if case["op"] == "copy":
        shape = (case["layers"], case["pages"], hkv, size, dim)
        s["k"], s["v"] = (_draw_normal(shape, dtype, gen) for _ in range(2))
        ids = r.sample(range(case["pages"]), 2 * case["pairs"])
        s["src"], s["dst"] = ids[:case["pairs"]], ids[case["pairs"]:]
        s["src_dev"], s["dst_dev"] = (torch.tensor(x, device="cuda") for x in (s["src"], s["dst"]))
        return s
    lens, new = _lengths(case)
    used = [-(-n // size) for n in lens]
    pages, width = sum(used) + 3, max(used)
    ids = r.sample(range(pages), sum(used))
    table = torch.zeros(case["batch"], width, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    tokens = sum(new)
    first = [0]
    for n in new:
        first.append(first[-1] + n)
    s["k_pages"], s["v_pages"] = (_draw_normal((pages, hkv, size, dim), dtype, gen) for _ in range(2))
    s["tables"] = table.cuda()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["cu_q"] = None if max(new) == 1 else torch.tensor(first, dtype=torch.int32, device="cuda")
    s["max_q"] = max(new)
    # of each new token: its sequence, its place among the sequence's new tokens, its position in the sequence
    s["seq"] = torch.tensor([b for b, n in enumerate(new) for _ in range(n)], device="cuda")
    s["place"] = torch.tensor([i for n in new for i in range(n)], device="cuda")
    s["pos"] = torch.tensor([lens[b] - n + i for b, n in enumerate(new) for i in range(n)], device="cuda")
    s["q"] = _draw_normal((tokens, case["heads"], dim), dtype, gen)
    if case["op"] == "append":
        s["k_new"], s["v_new"] = (_draw_normal((tokens, hkv, dim), dtype, gen) for _ in range(2))
        rate = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
        angle = torch.arange(width * size, dtype=torch.float64, device="cuda")[:, None] * rate
        s["rope"] = torch.cat((angle.cos(), angle.sin()), 1).float()
    return s


def _rotated(x, cos, sin, interleaved):
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)
    lo, hi = a * cos - b * sin, b * cos + a * sin
    return torch.stack((lo, hi), -1).flatten(-2) if interleaved else torch.cat((lo, hi), -1)


def _plain_append(s):
    size, dtype = s["case"]["page"], s["q"].dtype
    cos, sin = s["rope"][s["pos"]][:, None].chunk(2, -1)
    page = s["tables"][s["seq"], s["pos"] // size].long()
    slot = s["pos"] % size
    s["k_pages"][page, :, slot] = _rotated(s["k_new"].float(), cos, sin, s["case"]["interleaved"]).to(dtype)
    s["v_pages"][page, :, slot] = s["v_new"]
    return dict(q=_rotated(s["q"].float(), cos, sin, s["case"]["interleaved"]).to(dtype), k=s["k_pages"], v=s["v_pages"])


def _plain_attend(s):
    c = s["case"]
    batch, hkv, dim, group = c["batch"], c["heads_kv"], c["dim"], c["heads"] // c["heads_kv"]
    k, v = (x[s["tables"].long()].transpose(2, 3).reshape(batch, -1, hkv, dim).permute(0, 2, 1, 3).float()
            for x in (s["k_pages"], s["v_pages"]))  # [batch, heads_kv, tokens, dim]
    length = k.shape[2]
    q = torch.zeros(batch, s["max_q"], hkv, group, dim, device="cuda")
    q[s["seq"], s["place"]] = s["q"].view(-1, hkv, group, dim).float()
    q = q.permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, dim)
    score = (q @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(dim)).view(batch, hkv, s["max_q"], group, length)
    pos = torch.full((batch, s["max_q"]), -1, dtype=torch.long, device="cuda")
    pos[s["seq"], s["place"]] = s["pos"]
    j = torch.arange(length, device="cuda")
    seen = j <= pos[..., None]
    if c["window"]:
        seen &= (pos[..., None] - j < c["window"]) | (j < c["sinks"])
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True).clamp_min(1e-30)
    # keys that nobody may see hold whatever the pages held before: their product is no part of the sum
    v = v.masked_fill(~seen.any(1)[:, None, :, None], 0.0)
    o = (p.view(batch, hkv, -1, length) @ v).view(batch, hkv, s["max_q"], group, dim) / total
    o = o.permute(0, 2, 1, 3, 4)[s["seq"], s["place"]]
    return o.reshape(-1, c["heads"], dim).to(s["q"].dtype)


def _plain_copy(s):
    s["k"][:, s["dst_dev"]] = s["k"][:, s["src_dev"]]
    s["v"][:, s["dst_dev"]] = s["v"][:, s["src_dev"]]
    return s["k"], s["v"]


def run(s):
    c = s["case"]
    if own:
        from drofell_for_revision_b200 import paged
        if c["op"] == "append":
            q = paged.append_kv(s["k_pages"], s["v_pages"], s["k_new"], s["v_new"], s["tables"], s["lens"],
                                cu_q=s["cu_q"], q=s["q"], rope=s["rope"], interleaved=c["interleaved"])
            return dict(q=q, k=s["k_pages"], v=s["v_pages"])
        if c["op"] == "attend":
            return paged.attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], cu_q=s["cu_q"],
                                   max_q=s["max_q"], window=c["window"], sinks=c["sinks"])
        paged.copy_pages(s["k"], s["v"], s["src"], s["dst"])
        return s["k"], s["v"]
    return {"append": _plain_append, "attend": _plain_attend, "copy": _plain_copy}[c["op"]](s)


def _seen(case, p):
    """How many keys the query at position p sees, and the lowest of its window."""
    if not case["window"]:
        return p + 1, 0
    low = max(0, p + 1 - case["window"])
    return p + 1 - low + min(case["sinks"], low), low


def work(case):
    dim, hkv, size = case["dim"], case["heads_kv"], 2
    if case["op"] == "copy":
        return dict(bytes=2 * 2 * case["layers"] * case["pairs"] * hkv * case["page"] * dim * size, flops=0)
    lens, new = _lengths(case)
    tokens = sum(new)
    if case["op"] == "append":
        rows = tokens * (case["heads"] + 2 * hkv)
        return dict(bytes=2 * rows * dim * size + tokens * dim * 4, flops=3 * tokens * (case["heads"] + hkv) * dim)
    pairs = keys = 0
    for n, m in zip(lens, new):
        pairs += sum(_seen(case, p)[0] for p in range(n - m, n))
        low = _seen(case, n - m)[1]  # the keys that any of the queries sees, each read once
        keys += n - low + min(case["sinks"], low)
    return dict(bytes=2 * keys * hkv * dim * size + 2 * tokens * case["heads"] * dim * size,
                flops=4 * dim * case["heads"] * pairs)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        for x in (s["k"], s["v"]):
            for a, b in zip(s["src"], s["dst"]):
                x[:, b] = x[:, a]
        return s["k"], s["v"]
    lens, new = _lengths(case)
    table, size, dim = s["tables"].tolist(), case["page"], case["dim"]
    if case["op"] == "append":
        half = dim // 2
        q, k = s["q"].double(), s["k_new"].double()
        out_k, out_v = s["k_pages"].double(), s["v_pages"].double()
        # (x_a + i x_b)(cos + i sin) for each pair (a, b)
        angle = torch.complex(s["rope"][:, :half].double(), s["rope"][:, half:].double())[s["pos"]].unsqueeze(1)
        a = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
        b = a + (1 if case["interleaved"] else half)
        for x in (q, k):
            z = torch.complex(x[..., a], x[..., b]) * angle
            x[..., a], x[..., b] = z.real, z.imag
        t = 0
        for i, (n, m) in enumerate(zip(lens, new)):
            for p in range(n - m, n):
                out_k[table[i][p // size], :, p % size] = k[t]
                out_v[table[i][p // size], :, p % size] = s["v_new"][t].double()
                t += 1
        return dict(q=q, k=out_k, v=out_v)
    group = case["heads"] // case["heads_kv"]
    if 4 * dim * case["heads"] * sum(n * m for n, m in zip(lens, new)) > 2e13:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        pages = s["tables"][i, :-(-n // size)].long()
        p = torch.arange(n - m, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        hidden = j > p
        if case["window"]:
            hidden |= (j >= case["sinks"]) & (j <= p - case["window"])
        for h in range(case["heads_kv"]):
            k, v = (x[pages, h].reshape(-1, dim)[:n].double() for x in (s["k_pages"], s["v_pages"]))
            for g in range(h * group, (h + 1) * group):
                logit = s["q"][first:first + m, g].double() @ k.T / math.sqrt(dim)
                out[first:first + m, g] = torch.softmax(logit.masked_fill(hidden, -math.inf), -1) @ v
        first += m
    return out
