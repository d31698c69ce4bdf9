"""Paged key-value cache for serving: filling it, attention over it, its pages.

What lies between the q/k/v stage of a decoder layer
(``exllama.attention_forward_qkv_stage_v2``) and its output projection. The reference
serves these from its vLLM fork (After-Revision-DROFELL/cuda_extends/vllm_cache.py,
vllm_attention.py); here they are kernels of this library (``w4a16_append_kv``,
``w4a16_paged_attention``, ``w4a16_copy_pages``).

A layer's K and V are two tensors [pages, key-value heads, page size, head dim], fp16 or
bf16, of any strides they share (last dimension contiguous, the others multiples of 8
elements). A sequence is a row of ``tables`` (int32 page ids) and its length in ``lens``
(int32, the new tokens counted). Its new tokens are the rows ``cu_q[b]`` to ``cu_q[b + 1]``
of q, k and v; without ``cu_q`` every sequence has one, row b. Tables, lengths and offsets
stay on the device: calls do not synchronise, and one captured in a CUDA graph replays with
whatever they then hold. Calls run on the current stream. Nothing here has a gradient.

``PagePool`` keeps the books on the host: which pages are free, who shares which.
"""
from __future__ import annotations

import ctypes
import heapq
import math
from typing import Dict, Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import _capi, exllama

PageIds = Union[Sequence[int], torch.Tensor]


def _ext():
    ext = _capi.torch_fast_path()
    if ext is None:
        raise RuntimeError("the torch extension is not built; run `python -m drofell_for_revision_b200.build`")
    return ext


def append_kv(k_pages: torch.Tensor, v_pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor, tables: torch.Tensor,
              lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
              rope: Optional[torch.Tensor] = None, interleaved: bool = False,
              q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Store the new tokens' k and v [tokens, key-value heads, head dim] into their pages and
    return q [tokens, heads, head dim] rotated (in ``q_out``, which may be q and must not overlap
    it, k or v otherwise; None without q).

    ``rope`` is a float32 table [positions, rope dim]: a position's cosines, then its sines
    (``rope_table``); q and k are rotated by it, dimension i with i + rope dim / 2, or 2 i
    with 2 i + 1 when ``interleaved``. It must cover the tables' width times the page size.
    Pages written here must belong to one sequence only. Rows of no sequence are left as
    they were (undefined in a q that this call makes)."""
    return _ext().append_kv(k_pages, v_pages, k, v, tables, lens, cu_q, q, rope, interleaved, q_out)


def attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor,
              cu_q: Optional[torch.Tensor] = None, max_q: Optional[int] = None, scale: Optional[float] = None, window: int = 0,
              sinks: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v of every new token over its sequence's tokens up to itself;
    with ``window`` over the last ``window`` of them (itself counted) and the sequence's first
    ``sinks``. q [tokens, heads, head dim], heads a multiple of the key-value heads; scale
    (positive) 1 / sqrt(head dim) unless given. ``max_q`` is at least the most new tokens of a
    sequence: rows beyond it get no result. Left out, it is the number of rows (1 without
    ``cu_q``); given, it lets the call choose its kernel and cut its work by what is there. Rows
    that see nothing are 0 (also where every score is -inf); rows of no sequence are left as they
    were (undefined in an output that this call makes). ``out`` must not overlap q or hold an
    element twice.

    Scores, softmax statistics and sums are fp32. The weights enter the value product in two
    16-bit parts where a sequence has few new rows, and rounded once to the inputs' type where it
    has more (over 32 of new tokens x heads of a key-value head, over 16 on tables of 1024 tokens and
    more): there the error is up to 1.45 times that of an fp32 product."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if max_q is None:
        max_q = 1 if cu_q is None else q.shape[0]
    return _ext().paged_attention(q, k_pages, v_pages, tables, lens, cu_q, max_q, scale, window, sinks, out)


def device_error(device: Optional[torch.device] = None) -> int:
    """Nonzero if a bounded wait inside an attention kernel on this device gave up since the
    last call (outputs since then may be missing). Synchronises the current stream."""
    index = torch.device(device or "cuda").index
    index = torch.cuda.current_device() if index is None else index
    v = ctypes.c_int(0)
    _capi.check(_capi.lib().w4a16_paged_error(index, _capi.stream_ptr(index), ctypes.byref(v)))
    return v.value


def attention_forward(layernorm: torch.Tensor, norm_epsilon: float, q_proj: int, k_proj: int, v_proj: int, o_proj: int,
                      x: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
                      lens: torch.Tensor, rope: Optional[torch.Tensor] = None, cu_q: Optional[torch.Tensor] = None,
                      max_q: Optional[int] = None, window: int = 0, sinks: int = 0, interleaved: bool = False,
                      output: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The attention block of a decoder layer, beside ``exllama.mlp_forward_v2``: RMSNorm and the
    q, k, v projections (``attention_forward_qkv_stage_v2``), k and v into the pages, attention
    over them, the o projection. x [rows, hidden] fp16, one row per new token; the projections
    are q4 handles (``q4_matrix.cuda_q4``). Returns [rows, hidden] without the residual."""
    for t, name in ((x, "x"), (layernorm, "layernorm")):
        if torch.is_grad_enabled() and t.requires_grad:
            raise RuntimeError(f"{name} requires a gradient: the paged cache is for serving and has none (use torch.no_grad())")
    hq, hk, hv, ho = (exllama._handle(h) for h in (q_proj, k_proj, v_proj, o_proj))
    if x.dim() != 2 or x.shape[1] != hq.K:
        raise RuntimeError(f"x must be [rows, {hq.K}]")
    dim, rows = k_pages.shape[-1], x.shape[0]
    heads, heads_kv = hq.N // dim, hk.N // dim
    if hq.N % dim or hk.N % dim or hv.N != hk.N or ho.K != hq.N:
        raise RuntimeError(f"projections of {hq.N}, {hk.N}, {hv.N} columns and {ho.K} rows for heads of {dim}")
    rms = torch.empty_like(x)
    q, k, v = (torch.empty((rows, h.N), dtype=x.dtype, device=x.device) for h in (hq, hk, hv))
    _capi.qkv_forward(hq, hk, hv, layernorm, norm_epsilon, x, rms, q, k, v)
    q = q.view(rows, heads, dim)
    append_kv(k_pages, v_pages, k.view(rows, heads_kv, dim), v.view(rows, heads_kv, dim), tables, lens, cu_q=cu_q, q=q,
              rope=rope, interleaved=interleaved, q_out=q)
    mixed = attention(q, k_pages, v_pages, tables, lens, cu_q=cu_q, max_q=max_q, window=window, sinks=sinks)
    if output is None:
        output = torch.empty((rows, ho.N), dtype=x.dtype, device=x.device)
    return ho.gemm(mixed.view(rows, ho.K), output)


def _ids(x: PageIds) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        x = torch.as_tensor(x) if len(x) else torch.empty(0, dtype=torch.int64)
    if x.is_floating_point() or x.is_complex() or x.dtype == torch.bool:
        raise RuntimeError("page ids must be whole numbers")
    if x.is_cuda:
        raise RuntimeError("src and dst must be lists of page ids on the host")
    if x.numel() and (int(x.min()) < 0 or int(x.max()) >= 1 << 31):
        raise RuntimeError("page ids must fit 32 bits")
    return x.to(torch.int32).contiguous()


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: PageIds, dst: PageIds) -> None:
    """Copy pages src[i] to dst[i] of K and V [(layers,) pages, heads, page size, head dim], of
    all layers. The ids are host lists, read before the call returns; no page may be written
    twice, or both read and written."""
    if type(src) is list and type(dst) is list:
        _ext().copy_page_lists(k_pages, v_pages, src, dst)
    else:
        _ext().copy_pages(k_pages, v_pages, _ids(src), _ids(dst))


def rope_table(positions: int, dim: int, base: float = 10000.0, device: Optional[torch.device] = None) -> torch.Tensor:
    """The float32 angles of ``append_kv``: cosines and sines of p base^(-2 i / dim), taken in 64 bits."""
    rate = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * rate
    return torch.cat((angle.cos(), angle.sin()), 1).float().to(device or "cuda")


class PagePool:
    """The books of a cache's pages, on the host. A sequence (any hashable name) owns a list of
    pages; forked sequences share them until one has to write.

    The methods that move data return (src, dst) page lists for ``copy_pages``; nothing here
    touches the device, so the copies can be queued where the caller's stream wants them,
    before the pages are next written."""

    def __init__(self, num_pages: int, page_size: int) -> None:
        if num_pages <= 0 or page_size <= 0:
            raise RuntimeError(f"a pool of {num_pages} pages of {page_size} tokens")
        self.num_pages, self.page_size = num_pages, page_size
        self._free = list(range(num_pages))  # a heap: the lowest page is taken first
        self._refs = [0] * num_pages
        self._pages: Dict[object, List[int]] = {}
        self._lens: Dict[object, int] = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: object) -> int:
        return self._lens[seq]

    def pages(self, seq: object) -> Tuple[int, ...]:
        return tuple(self._pages[seq])

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free, page)

    def extend(self, seq: object, tokens: int) -> Tuple[List[int], List[int]]:
        """Room for ``tokens`` more tokens of ``seq`` (a new sequence if the name is new). A last
        page that is shared and about to be written is replaced by a page of its own: returned
        as the copy to make before the tokens are stored. RuntimeError, and nothing changed,
        when the pages do not suffice."""
        if tokens < 0:
            raise RuntimeError(f"extend by {tokens} tokens")
        pages = self._pages.get(seq, [])
        length = self._lens.get(seq, 0)
        need = -(-(length + tokens) // self.page_size) - len(pages)
        split = tokens > 0 and length % self.page_size != 0 and self._refs[pages[-1]] > 1
        if need + split > len(self._free):
            raise RuntimeError(f"{need + split} pages needed, {len(self._free)} free")
        src: List[int] = []
        dst: List[int] = []
        if split:
            old, new = pages[-1], self._take()
            self._drop(old)
            src.append(old)
            dst.append(new)
            pages[-1] = new
        pages.extend(self._take() for _ in range(need))
        self._pages[seq] = pages
        self._lens[seq] = length + tokens
        return src, dst

    def fork(self, seq: object, new: object) -> None:
        """``new`` becomes a copy of ``seq`` that shares its pages (no data moves until one of
        them is extended into a shared page)."""
        if new in self._pages:
            raise RuntimeError(f"sequence {new!r} exists")
        pages = self._pages[seq]
        for p in pages:
            self._refs[p] += 1
        self._pages[new] = list(pages)
        self._lens[new] = self._lens[seq]

    def truncate(self, seq: object, length: int) -> None:
        """Forget the tokens of ``seq`` from ``length`` on and free the pages that held only those."""
        if not 0 <= length <= self._lens[seq]:
            raise RuntimeError(f"truncate {self._lens[seq]} tokens to {length}")
        pages = self._pages[seq]
        keep = -(-length // self.page_size)
        for p in pages[keep:]:
            self._drop(p)
        del pages[keep:]
        self._lens[seq] = length

    def free(self, seq: object) -> None:
        """Forget ``seq``; pages that nobody shares become free."""
        for p in self._pages.pop(seq):
            self._drop(p)
        del self._lens[seq]

    def compact(self) -> Tuple[List[int], List[int]]:
        """Move the used pages into the lowest page numbers, the fewest that have to: returned as
        the copy to make before anything else is stored. Tables made before are stale."""
        used = self.num_pages - len(self._free)
        src = [p for p in range(used, self.num_pages) if self._refs[p]]
        dst = sorted(p for p in self._free if p < used)
        to = dict(zip(src, dst))
        for s, d in to.items():
            self._refs[d], self._refs[s] = self._refs[s], 0
        for pages in self._pages.values():
            pages[:] = [to.get(p, p) for p in pages]
        self._free = list(range(used, self.num_pages))
        return src, dst

    def tables(self, seqs: Iterable[object], width: Optional[int] = None,
               device: Optional[torch.device] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(tables, lens) of ``seqs`` in that order, int32 on ``device``; rows are filled up with
        -1, which no kernel reads as a page."""
        names = list(seqs)
        most = max((len(self._pages[s]) for s in names), default=0)
        width = most if width is None else width
        if width < most:
            raise RuntimeError(f"tables of {width} pages for a sequence of {most}")
        rows = [self._pages[s] + [-1] * (width - len(self._pages[s])) for s in names]
        tables = torch.tensor(rows, dtype=torch.int32).reshape(len(names), width)
        lens = torch.tensor([self._lens[s] for s in names], dtype=torch.int32)
        device = device or torch.device("cuda")
        return tables.to(device), lens.to(device)
